"""What pack_shared, rope_kv_append_at, attn_shared, spec_verify and a stage's prefixes refuse on the host, before any launch: every call
here names addresses that are never read."""
import ctypes as C
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from flyai_amd import _lib, ops
from flyai_amd._lib import ContextOverflow, FlyaiError
from flyai_amd.runtime import KVWorkspace, RaggedStage
from flyai_amd.sampling import Sampler

FAKE = 0x100000


def _each(fn, good, bads):
    """Every change of the good arguments is refused, by name."""
    assert len(good) == len(getattr(_lib.lib(), fn).argtypes)
    for i, v, text in bads:
        args = list(good)
        args[i] = v
        assert getattr(_lib.lib(), fn)(*args) == _lib.FLYAI_EINVAL, (fn, i, v)
        assert text in _lib.lib().flyai_last_error().decode(), (fn, i, v)


def test_pack_shared():
    #       q     starts base  cap   of    len   S  n  D   max  cu ...
    good = [FAKE] * 6 + [4, 2, 64, 32] + [FAKE] * 7 + [None]
    nulls = [(i, None, "null") for i in (*range(6), *range(10, 17))]
    _each("flyai_pack_shared", good, nulls + [(6, 0, "n_seqs"), (6, 8193, "n_seqs"), (6, -1, "n_seqs"), (7, -1, "n_prefixes"), (8, 0, "head_dim"),
                                              (9, -1, "max_tokens"), (9, 2 ** 24 + 1, "max_tokens")])


def test_attn_shared():
    good = [FAKE] * 8 + [4, 2, 8, 0, 32, 1 << 20, FAKE, None]
    nulls = [(i, None, "null") for i in (*range(8), 14)]
    _each("flyai_attn_shared_plan", good, nulls + [(8, 4097, ""), (8, -1, ""), (9, 1025, ""), (9, -1, ""), (10, 0, ""), (10, 65, ""), (11, -1, "window"),
                                                   (12, 65537, ""), (12, -1, ""), (13, -1, "pool_elems"), (14, FAKE + 8, "align")])
    good = [FAKE] * 4 + [64, 8, 64, 32, 4, 2] + [FAKE] * 3 + [None]
    nulls = [(i, None, "null") for i in (0, 1, 2, 3, 10, 11, 12)]
    _each("flyai_attn_shared", good, nulls + [(4, 32, ""), (4, 65, ""), (5, 4, ""), (6, 128, ""), (6, 32, ""), (7, 65537, ""), (8, 4097, ""), (9, 1025, ""),
                                              *((i, FAKE + 8, "align") for i in (0, 1, 2, 10, 11, 12))])
    size = _lib.lib().flyai_attn_shared_plan_bytes
    assert size(32, 4, 2) > 0 and not any((size(-1, 4, 2), size(65537, 4, 2), size(32, 4097, 2), size(32, 4, 1025)))
    size = _lib.lib().flyai_attn_shared_workspace_bytes
    assert size(32, 8) > 0 and not any((size(-1, 8), size(65537, 8), size(32, 0), size(32, 65)))


def test_sizes_grow_with_the_batch():
    """A stage keeps the largest step's plan and workspace: no smaller step needs more."""
    plan, ws = _lib.lib().flyai_attn_shared_plan_bytes, _lib.lib().flyai_attn_shared_workspace_bytes
    sizes = (0, 1, 15, 16, 17, 64, 100, 1000, 4096)
    for a, b in zip(sizes, sizes[1:]):
        assert plan(a, 7, 3) <= plan(b, 7, 3) and plan(100, a, 3) <= plan(100, b, 3) and ws(a, 8) <= ws(b, 8)
        assert plan(100, 7, min(a, 1024)) <= plan(100, 7, min(b, 1024))


def test_spec_verify():
    #       logits R  V     cu   S  draft u  u_draw temps ks ps   t  k  p    probs n  row   out ...       ws    stream
    good = [FAKE, 8, 1000, FAKE, 2, FAKE, FAKE, FAKE, None, None, None, 1.0, 0, 1.0, FAKE, 8, None, FAKE, FAKE, FAKE, FAKE, None]
    nulls = [(i, None, "null") for i in (0, 3, 5, 6, 7, 17, 18, 19, 20)]
    _each("flyai_spec_verify", good, nulls + [(1, -1, "R"), (2, 0, "V"), (2, 2 ** 22 + 1, "V"), (4, -1, "S"), (4, 65536, "n_streams"), (12, -1, "top_k"),
                                              (15, -1, "n_probs"), (15, 7, "probs_row"), (20, FAKE + 4, "align")])
    size = _lib.lib().flyai_spec_verify_workspace_bytes
    assert size(8, 1000, 2) > 0 and not any((size(-1, 1000, 2), size(8, 0, 2), size(8, 2 ** 22 + 1, 2), size(8, 1000, -1)))


def test_arguments_of_the_ops():
    """Wrong types, shapes, devices and strides: refused before the library is reached."""
    i32, i64 = (lambda *s: torch.zeros(*s, dtype=torch.int32)), (lambda *s: torch.zeros(*s, dtype=torch.int64))
    good = dict(q_lens=i32(3), starts=i32(3), kv_base=i64(3), kv_cap=i32(3), prefix_of=i32(3), prefix_len=i32(2))
    for name in good:
        for bad in (good[name].float(), i32(4) if name != "prefix_len" else i64(2), torch.zeros(6, dtype=good[name].dtype)[::2]):
            with pytest.raises((ValueError, TypeError)):
                ops.pack_shared(**{**good, name: bad}, head_dim=64, max_tokens=8)
    with pytest.raises((ValueError, TypeError)):
        ops.pack_shared(**good, head_dim=64, max_tokens=8.5)
    more = dict(prefix_base=i64(2), prefix_cap=i32(2), n_kv_heads=1, window=0, n_tokens=8, pool_elems=4096)
    for name, bad in (("prefix_base", i32(2)), ("prefix_cap", i32(3)), ("n_tokens", 1.5), ("window", None), ("pool_elems", "1")):
        with pytest.raises((ValueError, TypeError)):
            ops.attn_shared_plan(**good, **{**more, name: bad})
    f = lambda d, *s: torch.zeros(*s, dtype=d)  # noqa: E731
    good = dict(logits=f(torch.bfloat16, 4, 100), cu_rows=i32(3), draft=i32(4), u=f(torch.float64, 4), u_draw=f(torch.float64, 2), temp=1.0)
    for change in (dict(logits=f(torch.float32, 4, 100)), dict(logits=f(torch.bfloat16, 4, 200)[:, ::2]), dict(cu_rows=i64(3)), dict(cu_rows=i32(0)),
                   dict(draft=i32(5)), dict(u=f(torch.float32, 4)), dict(u_draw=f(torch.float64, 3)), dict(temp=f(torch.float64, 2)),
                   dict(temp=f(torch.float32, 3)), dict(top_k=f(torch.float32, 2)), dict(top_p=f(torch.float32, 1)), dict(probs_row=i32(4)),
                   dict(draft_probs=f(torch.float32, 3, 100)), dict(draft_probs=f(torch.float32, 4, 99)), dict(draft_probs=f(torch.float64, 4, 100)),
                   dict(draft_probs=f(torch.float32, 2, 100), probs_row=i32(3))):
        with pytest.raises((ValueError, TypeError)):
            ops.spec_verify(**{**good, **change})
    plan = ops.AttnSharedPlan(torch.zeros(64, dtype=torch.int32), 8, 3, 2, 1, 0, 4096)
    q, pool = f(torch.bfloat16, 8, 8, 64), f(torch.bfloat16, 4096)
    for change in (dict(q=q[:7]), dict(q=q.float()), dict(k_pool=pool[:4000]), dict(v_pool=pool[:100]), dict(sinks=f(torch.float32, 7)), dict(out=q[:4])):
        args = dict(q=q, k_pool=pool, v_pool=pool, sinks=f(torch.float32, 8), plan=plan, out=None)
        with pytest.raises((ValueError, TypeError)):
            ops.attn_shared(**{**args, **change})


HIDDEN = 64


@pytest.fixture
def stage(monkeypatch):
    """A RaggedStage of one layer with room for prefixes, and no workspace: a call that passes every check stops there."""
    lib = _lib.lib()
    cfg = _lib.StageConfig(n_layers=1, hidden=HIDDEN, n_q_heads=8, n_kv_heads=1, head_dim=64, n_experts=4, top_k=2, intermediate=64,
                           window=128, max_tokens=64, max_seqs=4, max_attn_items=64, rope_positions=4096, attn_split_keys=1024,
                           rms_eps=1e-5, attn_prefill_min=32)
    h = C.c_void_p()
    assert lib.flyai_stage_create(C.byref(cfg), C.byref(h)) == 0
    kv = KVWorkspace(1, 5, 128, 1, 64, "cpu")
    names = ("ln1", "ln2", "wqkv", "bqkv", "wo", "bo", "sinks", "router_w", "router_b", "w13_packed", "b13", "w2_packed", "b2", "k_pool", "v_pool")
    d = _lib.LayerDesc(**{f: FAKE for f in names}, sliding=0, pad=0, kv_pool_elems=kv.k[0].numel())
    assert lib.flyai_stage_set_layer(h, 0, C.byref(d)) == 0
    st = object.__new__(RaggedStage)
    st.__dict__.update(_h=h, _destroy=lib.flyai_stage_destroy, _sync=lambda d: None, device=torch.device("cpu"), kv=kv, _shared_ws=None,
                       shape=SimpleNamespace(hidden=HIDDEN))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: SimpleNamespace(cuda_stream=None))
    return st


def _step(st, starts=(100, 100), slots=(1, 2), prefixes=((0, 100), (0, 100)), q=(1, 1)):
    return st.forward(torch.zeros(sum(q), HIDDEN, dtype=torch.bfloat16), list(q), list(starts), list(slots), prefixes=list(prefixes))


def test_stage_prefixes(stage):
    with pytest.raises(ValueError, match="set_prefixes"):
        _step(stage)
    stage.set_prefixes()
    for good in ({}, dict(starts=(227, 100)), dict(prefixes=((0, 100), None)), dict(slots=(1, 0), prefixes=((0, 100), None)),
                 dict(prefixes=((3, 0), (4, 128)), starts=(0, 128)), dict(prefixes=((0, 64), (0, 100)))):
        with pytest.raises(FlyaiError, match="workspace not set"):
            _step(stage, **good)
    for bad, error in ((dict(starts=(99, 100)), "before its prefix"), (dict(starts=(-1, 100)), "start"), (dict(slots=(0, 2)), "appends"),
                       (dict(slots=(1, 0), starts=(100, 99), prefixes=((0, 100), None)), "appends"),
                       (dict(slots=(1, 0), starts=(100, 64), prefixes=((0, 100), (3, 64))), "appends")):
        with pytest.raises(FlyaiError, match=error):
            _step(stage, **bad)
    for bad in (dict(starts=(228, 100)), dict(starts=(2 ** 32 + 100, 100)), dict(slots=(1, 0), starts=(100, 128), prefixes=((0, 100), None))):
        with pytest.raises(ContextOverflow):
            _step(stage, **bad)
    for bad in (dict(prefixes=((0, 100),)), dict(prefixes=((5, 10), None)), dict(prefixes=((-1, 10), None)), dict(prefixes=((0, 129), None)),
                dict(prefixes=((0, -1), None)), dict(prefixes=((0, 2 ** 32 + 1), None))):
        with pytest.raises(ValueError):
            _step(stage, **bad)


def test_stage_prefixes_at_the_c_entry(stage):
    lib, kv = _lib.lib(), stage.kv
    stage.set_prefixes()
    i32, i64 = (lambda *v: np.array(v, dtype=np.int32)), (lambda *v: np.array(v, dtype=np.int64))

    def call(of=(0, 0), length=(100,), base=(0,), cap=(128,), n=1, at=(1, 2), drop=None):
        arrays = [i32(1, 1), i32(100, 100), i64(*(kv.base(s) for s in at)), i32(128, 128), i32(*of), i32(*length), i64(*base), i32(*cap)]
        p = [C.c_void_p(a.ctypes.data) for a in arrays]
        if drop is not None:
            p[drop] = None
        rc = lib.flyai_stage_forward_shared(stage._h, *p[:4], None, 2, *p[4:], n, FAKE, None)
        return rc, lib.flyai_last_error().decode()

    assert "workspace not set" in call()[1]
    for i in range(8):
        assert call(drop=i) [0] == _lib.FLYAI_EINVAL and "null" in call(drop=i)[1]
    for kw in (dict(of=(1, 0)), dict(of=(-2, 0)), dict(n=-1), dict(cap=(64,)), dict(cap=(100,)), dict(base=(4,)), dict(base=(-8,)), dict(length=(-1,)),
               dict(base=(64 * 64,)), dict(n=5, of=(0, 4), length=(1,) * 5, base=(0,) * 5, cap=(128,) * 5)):
        rc, text = call(**kw)
        assert rc == _lib.FLYAI_EINVAL and "workspace not set" not in text, (kw, rc, text)
    rc, text = call(cap=(1024,))
    assert rc == _lib.FLYAI_ERANGE
    size = int(lib.flyai_stage_shared_workspace_bytes(stage._h))
    for p, n in ((FAKE + 128, size), (FAKE, size - 1)):
        assert lib.flyai_stage_set_shared(stage._h, p, n) == _lib.FLYAI_EINVAL
    assert "workspace not set" in call()[1]  # what was bound is still there
    stage.set_prefixes(False)
    assert "flyai_stage_set_shared" in call()[1]


def test_accept_batch_wants_a_distribution_for_each_draft():
    """A row fewer, a row for each row of logits, another vocabulary: refused before the generator is asked."""
    sm = Sampler(temp=1.0, seed=3, device="cpu")
    before = sm.gen.bit_generator.state
    logits, drafts = torch.zeros(6, 50, dtype=torch.bfloat16), [[1, 2], [], [3]]
    for shape in ((2, 50), (6, 50), (4, 50), (0, 50), (3, 49), (3,), (1, 3, 50)):
        with pytest.raises(ValueError, match="probs must have shape"):
            sm.accept_batch(logits, drafts, probs=torch.zeros(shape))
    with pytest.raises(ValueError, match="probs must have shape"):
        sm.accept_batch(logits[:0], [], probs=torch.zeros(1, 50))
    assert sm.gen.bit_generator.state == before


@pytest.mark.parametrize("base", [2 ** 63 - 8, 2 ** 63 - 128 * 64, 2 ** 62, 2 ** 40])
def test_slabs_whose_end_passes_64_bits(stage, base):
    """The slab of a prefix and of a sequence, with prefixes in the step and without: past the pools, though the sum wraps round."""
    lib, kv = _lib.lib(), stage.kv
    stage.set_prefixes()
    i32, i64 = (lambda *v: np.array(v, dtype=np.int32)), (lambda *v: np.array(v, dtype=np.int64))

    def call(own, prefix):
        arrays = [i32(1, 1), i32(100, 100), i64(kv.base(1), own), i32(128, 128), i32(0, 0), i32(100), i64(prefix), i32(128)]
        p = [C.c_void_p(a.ctypes.data) for a in arrays]
        return (lib.flyai_stage_forward_shared(stage._h, *p[:4], None, 2, *p[4:], 1, FAKE, None), lib.flyai_last_error().decode(),
                lib.flyai_stage_forward(stage._h, *p[:4], 2, FAKE, None), lib.flyai_last_error().decode())

    rc, text, _, _ = call(kv.base(2), base)
    assert rc == _lib.FLYAI_ERANGE and "prefix 0" in text and "past the pools" in text
    rc, text, plain, plain_text = call(base, kv.base(0))
    assert rc == plain == _lib.FLYAI_ERANGE and all("sequence 1" in t and "past the pools" in t for t in (text, plain_text))
    root = i32(-1), i32(0)
    assert lib.flyai_stage_forward_tree(stage._h, 5, 1, *(C.c_void_p(a.ctypes.data) for a in root), base, 128, FAKE, None) == _lib.FLYAI_ERANGE


def test_slabs_without_positions(stage):
    """What the plan on the GPU refuses, a step refuses before any launch: its rows would be zeros, and no error."""
    lib, kv = _lib.lib(), stage.kv
    stage.set_prefixes()
    i32, i64 = (lambda *v: np.array(v, dtype=np.int32)), (lambda *v: np.array(v, dtype=np.int64))
    for length, cap in ((0, 0), (0, -64), (0, 2 ** 30 + 64)):
        arrays = [i32(1), i32(0), i64(kv.base(1)), i32(128), i32(0), i32(length), i64(kv.base(0)), i32(cap)]
        p = [C.c_void_p(a.ctypes.data) for a in arrays]
        rc = lib.flyai_stage_forward_shared(stage._h, *p[:4], None, 1, *p[4:], 1, FAKE, None)
        assert rc == _lib.FLYAI_EINVAL and "prefix 0 needs" in lib.flyai_last_error().decode(), (length, cap)


def test_spec_verify_rows_of_a_launch():
    #       logits R    V  cu   S  draft u   u_draw temps ks   ps    t    k  p    probs n row   out ...       ws    stream
    good = [FAKE, 0, 16, FAKE, 2, FAKE, FAKE, FAKE, None, None, None, 1.0, 0, 1.0, None, 0, None, FAKE, FAKE, FAKE, FAKE, None]
    _each("flyai_spec_verify", good, [(1, 2 ** 22, "rows"), (1, 2 ** 31 - 1, "rows")])
