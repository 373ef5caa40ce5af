"""Adapters through the stage: RaggedStage.forward with an AdapterBank, bit for bit against a layer put together from the
single operators (each of them held to its own oracle elsewhere), and its batches, graphs, trees and refusals."""
import pytest
import torch

from flyai_amd import ops
from flyai_amd._lib import FlyaiError
from flyai_amd.lora import AdapterBank
from flyai_amd.runtime import KVWorkspace, RaggedStage

import gpu_harness as gh

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def _adapter(shape, n_layers, r, seed, projections="qkvo", scale=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    t = lambda *s: (torch.randn(*s, device=DEV, generator=g) * 0.03 * scale).to(BF16)
    H, nq, nkv = shape.hidden, shape.n_q_heads * shape.head_dim, shape.n_kv_heads * shape.head_dim
    size = {"q": (H, nq), "k": (H, nkv), "v": (H, nkv), "o": (nq, H)}
    return [{p: (t(r, size[p][0]), t(size[p][1], r)) for p in projections} for _ in range(n_layers)]


def _bank(shape, n_layers, max_rank=32):
    bank = AdapterBank(shape, n_layers, 4, max_rank, DEV)
    bank.load(0, _adapter(shape, n_layers, 16, 1), 2.0)
    bank.load(1, _adapter(shape, n_layers, max_rank, 2), 0.5)
    bank.load(3, _adapter(shape, n_layers, 5, 3, "qv"), 1.5)
    return bank                                                     # slot 2 is empty


def _composed(case, bank, adapters):
    """The stage's one layer by single operators on the case's own KV -> hidden.  (Between layers the stage takes the next
    input norm's sum in another order, with the experts' combine.)"""
    sh, kv, q_lens, starts = case["shape"], case["kv"], case["q_lens"], case["starts"]
    T, S, D = case["T"], len(q_lens), sh.head_dim
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    base = torch.tensor([kv.base(s) for s in case["slots"]], dtype=torch.int64, device=DEV)
    cap = i32([kv.slot_cap(s) for s in case["slots"]])
    packed = ops.pack_ragged(i32(q_lens), i32(starts), base, cap, D, max(T, 64))
    pos, sid = packed["positions"], packed["seq_id"]
    row_seq, ad = sid[:T].contiguous(), i32(adapters)
    h = case["hidden"].clone()
    for l, lw in enumerate(case["layers"][:1]):
        window = sh.window if lw.sliding else 0
        xn = ops.rmsnorm(h, lw.ln1, sh.rms_eps)
        qkv = ops.linear_lora(xn, lw.wqkv, lw.bqkv, bank.qkv_a[l], bank.qkv_b[l], bank.scale, bank.ranks, ad,
                              segments=bank.segments, row_seq=row_seq)
        q = ops.rope_kv_append(qkv, pos, sid, case["rot"].cos, case["rot"].sin, sh.n_q_heads, sh.n_kv_heads, D, base, cap,
                               kv.k[l], kv.v[l])
        items, groups, small, pitems = ops.attn_plan_prefill(q_lens, starts, sh.n_kv_heads, window, 1024, 32)
        out = torch.empty_like(q)
        if items.shape[0]:
            out = ops.attn_ragged(q, kv.k[l], kv.v[l], base, cap, lw.sinks, window, items, groups, small, sh.n_kv_heads)
        if pitems.shape[0]:
            ops.attn_prefill(q, kv.k[l], kv.v[l], base, cap, lw.sinks, window, pitems, sh.n_kv_heads, out)
        ops.linear_lora(out.view(T, -1), lw.wo, lw.bo, bank.o_a[l], bank.o_b[l], bank.scale, bank.ranks, ad, row_seq=row_seq,
                        residual=h)
        xn = ops.rmsnorm(h, lw.ln2, sh.rms_eps)
        _, wts, _, off, perm, inv = ops.moe_route_permute(xn, lw.router_w, lw.router_b, sh.top_k)
        g = ops.moe_gate_up(xn, perm, off, sh.top_k, lw.w13_packed, lw.b13, sh.n_experts, sh.intermediate)
        y = ops.moe_down(g, off, lw.w2_packed, lw.b2, sh.n_experts, sh.hidden)
        h = ops.moe_combine(y, inv, wts, residual=h)
    return h


def _copy(kv):
    return kv.k_pools.clone(), kv.v_pools.clone()


def _restore(kv, saved):
    kv.k_pools.copy_(saved[0])
    kv.v_pools.copy_(saved[1])


BATCHES = {"decode": ((1, 1, 4, 7, 16), (300, 5, 1000, 0, 130), (0, -1, 1, 3, 2)),
           "verify": ((5,) * 20, tuple(range(10, 1010, 50)), tuple(i % 5 - 1 for i in range(20))),
           "prompts": ((200, 1, 90, 3), (0, 700, 64, 20), (1, 0, -1, 3)),
           "one_prompt": ((260,), (37,), (1,)),
           "long_prompt": ((1, 992, 3, 4), (5, 60, 700, 0), (2, 1, -1, 3)),
           "longer_prompt": ((3, 1, 1500, 2), (0, 900, 17, 64), (0, 1, 1, 3))}


@pytest.mark.parametrize("name", list(BATCHES))
def test_stage_is_its_operators(name):
    q_lens, starts, adapters = BATCHES[name]
    case = gh.small_stage_case(n_layers=1, n_experts=8, seed=21, q_lens=q_lens, starts=starts)
    bank = _bank(case["shape"], 1)
    kv, saved = case["kv"], _copy(case["kv"])
    want = _composed(case, bank, adapters)
    after = _copy(kv)
    _restore(kv, saved)
    st = RaggedStage(case["shape"], case["layers"], case["rot"], kv, max_tokens=max(64, case["T"]), max_seqs=len(q_lens), lora=bank)
    got = st.forward(case["hidden"].clone(), q_lens, starts, case["slots"], adapters)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    assert torch.equal(kv.k_pools, after[0]) and torch.equal(kv.v_pools, after[1])
    # without adapters: the bits of a stage that has no bank
    _restore(kv, saved)
    none = st.forward(case["hidden"].clone(), q_lens, starts, case["slots"], [None] * len(q_lens))
    _restore(kv, saved)
    plain = RaggedStage(case["shape"], case["layers"], case["rot"], kv, max_tokens=max(64, case["T"]), max_seqs=len(q_lens))
    ref = plain.forward(case["hidden"].clone(), q_lens, starts, case["slots"])
    assert torch.equal(none, ref) and not torch.equal(got, ref)


@pytest.mark.parametrize("graphs", [False, True])
def test_a_sequence_depends_on_its_own_adapter_alone(graphs):
    """Each sequence of a mixed batch alone, and with other adapters beside it: the same bits; replayed graphs included."""
    q_lens, starts, adapters = BATCHES["decode"]
    case = gh.small_stage_case(n_layers=2, n_experts=8, seed=22, q_lens=q_lens, starts=starts)
    bank = _bank(case["shape"], 2)
    kv, saved = case["kv"], _copy(case["kv"])
    st = RaggedStage(case["shape"], case["layers"], case["rot"], kv, max_tokens=64, max_seqs=5, lora=bank, use_graphs=graphs)

    def step(which, ads):
        _restore(kv, saved)
        rows = torch.cat([case["hidden"][sum(q_lens[:b]):sum(q_lens[:b + 1])] for b in which])
        out = st.forward(rows.clone(), [q_lens[b] for b in which], [starts[b] for b in which], which, ads).clone()
        torch.cuda.synchronize()
        return out

    whole = step([0, 1, 2, 3, 4], adapters)
    for turn in range(2):
        for b in range(5):
            lo, hi = sum(q_lens[:b]), sum(q_lens[:b + 1])
            assert torch.equal(step([b], [adapters[b]]), whole[lo:hi]), (turn, b)
            others = [(a + turn) % 4 if i != b else adapters[b] for i, a in enumerate(adapters)]
            assert torch.equal(step([0, 1, 2, 3, 4], others)[lo:hi], whole[lo:hi]), (turn, b)
    # an emptied slot: as without; refilled: as before (graphs read the bank in place)
    bank.unload(0)
    gone = step([0], [0])
    assert torch.equal(gone, step([0], [-1])) and not torch.equal(gone, whole[:1])
    bank.load(0, _adapter(case["shape"], 2, 16, 1), 2.0)
    assert torch.equal(step([0, 1, 2, 3, 4], adapters), whole)


@pytest.mark.parametrize("M", [9, 300])
def test_tree_with_an_adapter(M):
    """A tree that is a chain is a verify step, with an adapter as without."""
    case = gh.small_stage_case(n_layers=2, n_experts=8, seed=23, q_lens=(M,), starts=(200,))
    bank = _bank(case["shape"], 2)
    kv, saved = case["kv"], _copy(case["kv"])
    st = RaggedStage(case["shape"], case["layers"], case["rot"], kv, max_tokens=max(64, M), max_seqs=1, lora=bank, prefill_min=0)
    want = st.forward(case["hidden"].clone(), [M], [200], [0], [1])
    after = _copy(kv)
    _restore(kv, saved)
    got = st.forward_tree(case["hidden"].clone(), 200, list(range(-1, M - 1)), list(range(M)), 0, adapter=1)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(kv.k_pools, after[0]) and torch.equal(kv.v_pools, after[1])


def test_fork_decode_compact_with_adapters():
    """The operators as they serve together: a prompt with one adapter, its cache forked to two samples, both decoded with it in
    one batch (the same bits as one), and a drafted chain compacted to its accepted part."""
    case = gh.small_stage_case(n_layers=2, n_experts=8, seed=24, q_lens=(40,), starts=(0,))
    shape = case["shape"]
    kv = KVWorkspace(2, 3, 256, shape.n_kv_heads, shape.head_dim, DEV)
    bank = _bank(shape, 2)
    st = RaggedStage(shape, case["layers"], case["rot"], kv, max_tokens=64, max_seqs=3, lora=bank)
    st.forward(case["hidden"].clone(), [40], [0], [0], [1])
    kv.fork(0, [1, 2], 40)
    rows = case["hidden"][:3].contiguous()
    alone = st.forward(rows.clone(), [3], [40], [0], [1])
    both = st.forward(torch.cat([rows, rows]), [3, 3], [40, 40], [1, 2], [1, 1])
    assert torch.equal(both[:3], alone) and torch.equal(both[3:], alone)
    want = [kv.k_dense(l, 1)[:, [40, 42]] for l in range(2)]
    kv.compact([1], [40], [[0, 2]])
    torch.cuda.synchronize()
    for l in range(2):
        assert torch.equal(kv.k_dense(l, 1)[:, 40:42], want[l])
        assert torch.equal(kv.k_dense(l, 2)[:, :43], kv.k_dense(l, 0)[:, :43])


def test_refusals():
    case = gh.small_stage_case(n_layers=2, n_experts=8, seed=25, q_lens=(1, 1), starts=(3, 4))
    shape, slots = case["shape"], case["slots"]
    st = RaggedStage(shape, case["layers"], case["rot"], case["kv"], max_tokens=64, max_seqs=2)
    step = lambda ads: st.forward(case["hidden"].clone(), [1, 1], [3, 4], slots, ads)
    with pytest.raises(FlyaiError, match="has none"):
        step([0, -1])
    with pytest.raises(ValueError):
        step([-1])
    with pytest.raises(ValueError):
        st.set_lora(AdapterBank(shape, 1, 2, 16, DEV))
    bank = _bank(shape, 2)
    st.set_lora(bank)
    for bad in (4, -2):
        with pytest.raises(FlyaiError, match="outside"):
            step([0, bad])
    with pytest.raises(FlyaiError, match="outside"):
        st.forward_tree(case["hidden"].clone(), 3, [-1, 0], [0, 1], 0, adapter=7)
    good = _adapter(shape, 2, 16, 1)
    before = bank.qkv_a.clone()
    for bad in (good[:1], [good[0], {"q": (good[0]["q"][0], good[0]["k"][1])}], [good[0], {"gate": good[0]["q"]}],
                _adapter(shape, 2, 33, 1)):
        with pytest.raises(ValueError):
            bank.load(0, bad, 1.0)
    with pytest.raises(ValueError):
        bank.load(4, good, 1.0)
    assert torch.equal(bank.qkv_a, before) and bank.ranks.tolist() == [16, 32, 0, 5]
    with pytest.raises(ValueError):
        AdapterBank(shape, 2, 2, 129, DEV)
    st.set_lora(None)
    with pytest.raises(FlyaiError, match="has none"):
        step([0, -1])
    step([None, -1])
