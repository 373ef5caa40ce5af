"""ops.kv_fork and ops.kv_compact on the GPU, bit for bit against dense indexing of the slabs."""
import numpy as np
import pytest
import torch

from flyai_amd import kvlayout, ops
from flyai_amd._lib import ContextOverflow, FlyaiError

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _pools(layers, n, seed):
    """Random bits, NaN and infinities among them: a move keeps every bit."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return [torch.randint(-32768, 32768, (layers, n), device=DEV, generator=g, dtype=torch.int32).to(torch.int16)
            .view(torch.bfloat16) for _ in range(2)]


def _bits(t):
    return t.view(torch.int16)


def _moved(pool, kind, heads, src, dst, src_slab, dst_slab, src_pool=None):
    """The pool with positions src of one slab copied to dst of another, through kvlayout's offsets."""
    out = pool.clone()
    (sb, sc), (db, dc) = src_slab, dst_slab
    fn = kvlayout.k_offsets if kind == "k" else kvlayout.v_offsets
    so = fn(torch.as_tensor(src, device=DEV)).reshape(-1)
    do = fn(torch.as_tensor(dst, device=DEV)).reshape(-1)
    for h in range(heads):
        out[:, db + h * dc * 64 + do] = (pool if src_pool is None else src_pool)[:, sb + h * sc * 64 + so]
    return out


@pytest.mark.parametrize("lo,hi", [(0, 1), (0, 64), (0, 77), (5, 6), (63, 65), (3, 200), (64, 128), (128, 320), (9, 9), (0, 0)])
@pytest.mark.parametrize("copies", [1, 3])
def test_fork(lo, hi, copies):
    layers, heads = 3, 2
    caps = [320, 384, 320, 1024][:copies + 1]
    bases = np.cumsum([0] + [heads * c * 64 + 8 * i for i, c in enumerate(caps)]).tolist()
    slabs = list(zip(bases, caps))
    k, v = _pools(layers, bases[-1] + 8, lo + hi)
    wk, wv = k.clone(), v.clone()
    pos = np.arange(lo, hi)
    for d in slabs[1:]:
        wk = _moved(wk, "k", heads, pos, pos, slabs[0], d)
        wv = _moved(wv, "v", heads, pos, pos, slabs[0], d)
    ops.kv_fork(k, v, heads, slabs[0], slabs[1:], lo, hi)
    assert torch.equal(_bits(k), _bits(wk)) and torch.equal(_bits(v), _bits(wv))


def test_fork_to_many_and_from_other_pools():
    """More destinations than one launch takes, from another workspace's pools."""
    layers, heads, cap = 2, 1, 64
    k, v = _pools(layers, 70 * cap * 64, 1)
    sk, sv = _pools(layers, 2 * 128 * 64, 2)
    slabs = [(i * cap * 64, cap) for i in range(70)]
    src, pos = (128 * 64, 128), np.arange(0, 50)
    wk, wv = k.clone(), v.clone()
    for d in slabs:
        wk = _moved(wk, "k", heads, pos, pos, src, d, sk)
        wv = _moved(wv, "v", heads, pos, pos, src, d, sv)
    ops.kv_fork(k, v, heads, src, slabs, 0, 50, src_k=sk, src_v=sv)
    assert torch.equal(_bits(k), _bits(wk)) and torch.equal(_bits(v), _bits(wv))
    before = k.clone()
    ops.kv_fork(k, v, heads, slabs[0], [], 0, 50)
    assert torch.equal(_bits(k), _bits(before))


def _keep_cases():
    rng = np.random.RandomState(0)
    return {
        "one": (100, [7]), "none": (100, []), "stays": (0, [0, 1, 2, 3]), "path": (61, [0, 3, 8, 13, 17]),
        "by_one": (0, list(range(1, 300))), "by_64": (0, list(range(64, 300))), "by_8": (40, list(range(8, 200))),
        "ends": (0, list(range(4)) + list(range(250, 1000))), "sparse": (3, sorted(rng.choice(1000, 333, replace=False).tolist())),
        "long": (0, sorted(rng.choice(1020, 900, replace=False).tolist())), "full_704": (5, list(range(300, 1004))),
        "by_5_all": (5, list(range(5, 1019))), "alternate": (1, list(range(0, 1020, 2))), "last": (1023, [0]),
        "runs": (9, [i for i in range(1000) if i % 20 < 11]),
    }


@pytest.mark.parametrize("name", list(_keep_cases()))
def test_compact(name):
    start, keep = _keep_cases()[name]
    layers, heads, cap = 2, 2, 1024
    base = 16
    k, v = _pools(layers, base + heads * cap * 64 + 24, 3)
    src, dst = start + np.asarray(keep, dtype=np.int64), start + np.arange(len(keep))
    wk = _moved(k, "k", heads, src, dst, (base, cap), (base, cap))
    wv = _moved(v, "v", heads, src, dst, (base, cap), (base, cap))
    ops.kv_compact(k, v, heads, [(base, cap, start, keep)])
    assert torch.equal(_bits(k), _bits(wk)) and torch.equal(_bits(v), _bits(wv))


@pytest.mark.parametrize("rows,span", [(1, 9000), (40, 9000), (255, 4000), (600, 9000), (1100, 9000), (2100, 9000), (4600, 9000),
                                       (257, 300), (9, 600)])
@pytest.mark.parametrize("start", [0, 45])
def test_compact_by_density(rows, span, start):
    """From a few positions of a long context to half of them, and all of them in one stretch of it."""
    heads, cap = 2, 9088
    rng = np.random.RandomState(rows)
    k, v = _pools(2, heads * cap * 64, 6)
    for shift in (0, 9000 - span):
        keep = shift + np.sort(rng.choice(span, rows, replace=False))
        src, dst = start + keep, start + np.arange(rows)
        wk, wv = _moved(k, "k", heads, src, dst, (0, cap), (0, cap)), _moved(v, "v", heads, src, dst, (0, cap), (0, cap))
        gk, gv = k.clone(), v.clone()
        ops.kv_compact(gk, gv, heads, [(0, cap, start, keep)])
        assert torch.equal(_bits(gk), _bits(wk)) and torch.equal(_bits(gv), _bits(wv))


def test_compact_past_one_launch():
    """More positions than one launch's words: pieces of a long slab, beside a short one."""
    heads, cap = 1, 60032
    rng = np.random.RandomState(5)
    k, v = _pools(1, heads * (cap + 128) * 64, 5)
    keep = np.sort(rng.choice(60000, 41000, replace=False))
    slabs = [(0, 128), (128 * heads * 64, cap)]
    moves = [(*slabs[0], 1, [2, 70, 100]), (*slabs[1], 30, keep)]
    wk, wv = k, v
    for (b, c, start, kp) in moves:
        src, dst = start + np.asarray(kp), start + np.arange(len(kp))
        wk, wv = (_moved(wk, "k", heads, src, dst, (b, c), (b, c)), _moved(wv, "v", heads, src, dst, (b, c), (b, c)))
    ops.kv_compact(k, v, heads, moves)
    assert torch.equal(_bits(k), _bits(wk)) and torch.equal(_bits(v), _bits(wv))


def test_compact_many_slabs():
    """More slabs, and more rows in all, than one launch takes; numpy and tensor lists; one layer's pool."""
    heads, cap, n = 1, 128, 30
    rng = np.random.RandomState(4)
    k, v = _pools(1, n * heads * cap * 64, 4)
    k, v = k[0], v[0]
    wk, wv, moves = k[None].clone(), v[None].clone(), []
    for i in range(n):
        m = int(rng.randint(1, 90))
        start = int(rng.randint(0, 30))
        keep = np.sort(rng.choice(cap - start, m, replace=False)).astype(np.int32)
        slab = (i * heads * cap * 64, cap)
        wk = _moved(wk, "k", heads, start + keep, start + np.arange(m), slab, slab)
        wv = _moved(wv, "v", heads, start + keep, start + np.arange(m), slab, slab)
        moves.append((*slab, start, torch.from_numpy(keep) if i % 2 else keep))
    ops.kv_compact(k, v, heads, moves)
    assert torch.equal(_bits(k), _bits(wk[0])) and torch.equal(_bits(v), _bits(wv[0]))


def test_offsets_past_32_bits():
    """A slab whose elements lie past 2^31 in its pool, and one past 2^31 within a layer stride."""
    heads, cap = 8, 64
    far = (2 ** 31 // (heads * cap * 64) + 3) * heads * cap * 64
    n = far + heads * cap * 64
    k = torch.zeros(1, n, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros(1, n, dtype=torch.bfloat16, device=DEV)
    near = heads * cap * 64
    sk, sv = _pools(1, near, 5)
    k[:, :near], v[:, :near] = sk, sv
    ops.kv_fork(k, v, heads, (0, cap), [(far, cap)], 0, 64)
    assert torch.equal(_bits(k[:, far:]), _bits(sk)) and torch.equal(_bits(v[:, far:]), _bits(sv))
    ops.kv_compact(k, v, heads, [(far, cap, 2, [9, 30, 50])])
    pos = np.array([11, 32, 52])
    assert torch.equal(_bits(k[:, far:]), _bits(_moved(sk, "k", heads, pos, np.array([2, 3, 4]), (0, cap), (0, cap))))
    assert torch.equal(_bits(v[:, far:]), _bits(_moved(sv, "v", heads, pos, np.array([2, 3, 4]), (0, cap), (0, cap))))
    assert not bool(k[:, near:far].any())


def test_captured():
    """A captured fork and compaction replay with the plan they were captured with, on what the pools hold then."""
    heads, cap = 2, 128
    slab = heads * cap * 64
    k, v = _pools(2, 2 * slab, 6)
    plan = lambda a, b: (ops.kv_fork(a, b, heads, (0, cap), [(slab, cap)], 0, 100), ops.kv_compact(a, b, heads, [(slab, cap, 10, [3, 40, 41])]))
    plan(k.clone(), v.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan(k, v)
    for i in range(3):
        nk, nv = _pools(2, 2 * slab, 7 + i)
        k.copy_(nk)
        v.copy_(nv)
        graph.replay()
        torch.cuda.synchronize()
        plan(nk, nv)
        assert torch.equal(_bits(k), _bits(nk)) and torch.equal(_bits(v), _bits(nv))


def test_refusals_leave_the_pools_alone():
    heads, cap = 2, 128
    slab = heads * cap * 64
    k, v = _pools(2, 2 * slab, 12)
    before = k.clone(), v.clone()
    with pytest.raises(ContextOverflow):
        ops.kv_fork(k, v, heads, (0, cap), [(slab, cap)], 0, cap + 1)
    with pytest.raises(ContextOverflow):
        ops.kv_compact(k, v, heads, [(slab, cap, 100, [0, 28])])
    with pytest.raises(FlyaiError):
        ops.kv_fork(k, v, heads, (0, cap), [(64, cap)], 0, 10)
    with pytest.raises(ValueError):
        ops.kv_compact(k, v, heads, [(0, cap, 0, [-1])])
    with pytest.raises(ValueError):
        ops.kv_compact(k, v, heads, [(0, cap, 0, [0.5])])
    for keep in ([3, 2], [2, 2]):
        with pytest.raises(FlyaiError, match="ascending"):
            ops.kv_compact(k, v, heads, [(0, cap, 0, keep)])
    with pytest.raises(ValueError):
        ops.kv_fork(k, v[:1], heads, (0, cap), [(slab, cap)], 0, 10)
    with pytest.raises(TypeError):
        ops.kv_fork(k.float(), v.float(), heads, (0, cap), [(slab, cap)], 0, 10)
    torch.cuda.synchronize()
    assert torch.equal(_bits(k), _bits(before[0])) and torch.equal(_bits(v), _bits(before[1]))


def test_positions_past_32_bits_are_refused():
    heads, cap = 2, 128
    slab = heads * cap * 64
    k, v = _pools(2, 2 * slab, 12)
    before = k.clone()
    with pytest.raises(ContextOverflow):
        ops.kv_fork(k, v, heads, (0, cap), [(slab, cap)], 0, 2 ** 32 + 5)
    with pytest.raises(FlyaiError):
        ops.kv_fork(k, v, heads, (0, cap), [(slab, cap)], 2 ** 32, 5)
    with pytest.raises(FlyaiError):
        ops.kv_fork(k, v, heads, (0, cap), [(slab, cap)], -2 ** 32, 5)
    with pytest.raises(TypeError):
        ops.kv_fork(k, v, heads, (0, cap), [(slab, cap)], 0, 5.5)
    for n_heads in (2 ** 32 + 2, -2 ** 32 + 2):
        with pytest.raises(FlyaiError):
            ops.kv_fork(k, v, n_heads, (0, cap), [(slab, cap)], 0, 5)
        with pytest.raises(FlyaiError):
            ops.kv_compact(k, v, n_heads, [(0, cap, 0, [1])])
    with pytest.raises(ValueError):
        ops.kv_compact(k, v, heads, [(0, cap, 2 ** 32, [1])])
    with pytest.raises(ValueError):
        ops.kv_compact(k, v, heads, [(0, cap, 0, [2 ** 32 + 1])])
    torch.cuda.synchronize()
    assert torch.equal(_bits(k), _bits(before))


# ---- through the workspace ---------------------------------------------------------------------------

def _workspace(layers=2, slots=3, caps=(100, 200, 100), heads=2, seed=20):
    from flyai_amd.runtime import KVWorkspace
    kv = KVWorkspace(layers, slots, 0, heads, 64, DEV, caps=list(caps))
    k, v = _pools(layers, kv.k_pools.shape[1], seed)
    kv.k_pools.copy_(k)
    kv.v_pools.copy_(v)
    return kv


def _dense(kv):
    return [[(_bits(kv.k_dense(l, s)), _bits(kv.v_dense(l, s))) for s in range(kv.n_slots)] for l in range(kv.n_layers)]


def test_workspace_fork_and_compact():
    kv = _workspace()
    before = _dense(kv)
    kv.fork(1, [0, 2], 77)
    kv.compact([1, 2], [10, 0], [[3, 8, 20], list(range(4)) + list(range(50, 120))])
    after = _dense(kv)
    for l in range(kv.n_layers):
        for t in range(2):
            b, a = [x[t] for x in before[l]], [x[t] for x in after[l]]
            assert torch.equal(a[0][:, :77], b[1][:, :77]) and torch.equal(a[0][:, 77:], b[0][:, 77:])
            want = b[1].clone()
            want[:, 10:13] = b[1][:, [13, 18, 30]]
            assert torch.equal(a[1], want)
            forked = b[2].clone()
            forked[:, :77] = b[1][:, :77]
            want = forked.clone()
            want[:, 4:74] = forked[:, 50:120]
            assert torch.equal(a[2], want)
    with pytest.raises(ContextOverflow):
        kv.fork(1, [0], 129)
    with pytest.raises(ValueError):
        kv.fork(3, [0], 10)
    with pytest.raises(ValueError):
        kv.compact([0], [1, 2], [[1]])


def test_copy_slot_between_workspaces():
    kv, other = _workspace(), _workspace(layers=3, slots=1, caps=(200,), seed=21)
    kv.copy_slot(1, other, 0)
    for l in range(2):
        assert torch.equal(_bits(kv.k_dense(l, 1)), _bits(other.k_dense(l, 0)))
        assert torch.equal(_bits(kv.v_dense(l, 1)), _bits(other.v_dense(l, 0)))
    before = _dense(kv)
    kv.copy_slot(0, kv, 2)
    kv.copy_slot(1, kv, 1)
    after = _dense(kv)
    for l in range(2):
        assert torch.equal(after[l][0][0], before[l][2][0]) and torch.equal(after[l][1][1], before[l][1][1])
    with pytest.raises(ValueError):
        kv.copy_slot(0, other, 0)


def test_workspace_pools_are_the_layers():
    kv = _workspace()
    assert kv.k[1].data_ptr() == kv.k_pools[1].data_ptr() and kv.v[0].data_ptr() == kv.v_pools.data_ptr()
    kv.zero()
    assert not bool(kv.k_pools.any()) and not bool(kv.v_pools.any())
