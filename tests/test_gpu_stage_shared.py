"""Sequences behind shared prefixes through the stage: RaggedStage.forward(prefixes=), bit for bit against a layer put together from the
single operators, and against the same batch on copies of its prefixes."""
import pytest
import torch

from flyai_amd import ops
from flyai_amd._lib import ContextOverflow, FlyaiError
from flyai_amd.runtime import KVWorkspace, RaggedStage

import gpu_harness as gh

pytestmark = pytest.mark.gpu
DEV = "cuda"

# slots: 0 and 1 hold the prompts of 700 and 130 positions, 2 a sequence of its own, the rest what follows a prompt; the last sequence
# is the second prompt's own, which goes on behind it
PROMPTS = [(0, 700), (1, 130)]
CASES = {"decode": ((1,) * 6, (700, 705, 130, 40, 900, 150), (3, 4, 5, 2, 6, 1), (0, 0, 1, None, 0, None)),
         "drafts": ((4, 1, 3, 5, 2, 7), (763, 700, 131, 0, 890, 130), (3, 4, 5, 2, 6, 1), (0, 0, 1, None, 0, None)),
         "questions": ((90, 70, 40, 60, 1, 2), (700, 700, 130, 3, 701, 130), (3, 4, 5, 2, 6, 1), (0, 0, 1, None, 0, None))}


def _case(name, n_layers=1, seed=0):
    q_lens, starts, slots, of = CASES[name]
    case = gh.small_stage_case(n_layers, seed=seed, q_lens=q_lens, starts=starts, maxlen=1024)
    case["kv"] = KVWorkspace(n_layers, 7, 1024, case["shape"].n_kv_heads, 64, DEV, caps=[700, 1024, 300, 300, 200, 300, 300])
    gh.fill_kv_random(case["kv"], seed + 7)
    case.update(slots=list(slots), prefixes=[None if p is None else PROMPTS[p] for p in of], of=[-1 if p is None else p for p in of])
    return case


def _stage(case, **kw):
    st = RaggedStage(case["shape"], case["layers"], case["rot"], case["kv"], max_tokens=max(64, case["T"]), max_seqs=8, **kw)
    st.set_prefixes()
    return st


def _forward(st, case, hidden=None, **kw):
    h = case["hidden"].clone() if hidden is None else hidden
    return st.forward(h, case["q_lens"], case["starts"], case["slots"], prefixes=case["prefixes"], **kw)


def _pools(kv):
    return kv.k_pools.clone(), kv.v_pools.clone()


def _restore(kv, saved):
    kv.k_pools.copy_(saved[0])
    kv.v_pools.copy_(saved[1])


def _composed(case):
    sh, kv, T, D = case["shape"], case["kv"], case["T"], 64
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    i64 = lambda v: torch.tensor(v, dtype=torch.int64, device=DEV)  # noqa: E731
    lengths = dict(q_lens=i32(case["q_lens"]), starts=i32(case["starts"]), kv_base=i64([kv.base(s) for s in case["slots"]]),
                   kv_cap=i32([kv.slot_cap(s) for s in case["slots"]]), prefix_of=i32(case["of"]), prefix_len=i32([n for _, n in PROMPTS]))
    pk = ops.pack_shared(**lengths, head_dim=D, max_tokens=T)
    lw, h = case["layers"][0], case["hidden"].clone()
    qkv = ops.linear(ops.rmsnorm(h, lw.ln1, sh.rms_eps), lw.wqkv, lw.bqkv)
    q = ops.rope_kv_append(qkv, pk["positions"], pk["seq_id"], case["rot"].cos, case["rot"].sin, sh.n_q_heads, sh.n_kv_heads, D,
                           lengths["kv_base"], lengths["kv_cap"], kv.k[0], kv.v[0], kv_pos=pk["kv_pos"])
    plan = ops.attn_shared_plan(**lengths, prefix_base=i64([kv.base(s) for s, _ in PROMPTS]), prefix_cap=i32([kv.slot_cap(s) for s, _ in PROMPTS]),
                                n_kv_heads=sh.n_kv_heads, window=sh.window if lw.sliding else 0, n_tokens=T, pool_elems=kv.k[0].numel())
    out = ops.attn_shared(q, kv.k[0], kv.v[0], lw.sinks, plan)
    assert int(pk["status"]) == 0 and int(plan.status) == 0
    ops.linear(out.view(T, -1), lw.wo, lw.bo, residual=h)
    xn = ops.rmsnorm(h, lw.ln2, sh.rms_eps)
    _, wts, _, off, perm, inv = ops.moe_route_permute(xn, lw.router_w, lw.router_b, sh.top_k)
    g = ops.moe_gate_up(xn, perm, off, sh.top_k, lw.w13_packed, lw.b13, sh.n_experts, sh.intermediate)
    return ops.moe_combine(ops.moe_down(g, off, lw.w2_packed, lw.b2, sh.n_experts, sh.hidden), inv, wts, residual=h)


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("sliding", [True, False])
def test_a_layer_is_the_operators(name, sliding):
    case = _case(name)
    case["layers"][0].sliding = sliding
    saved = _pools(case["kv"])
    got = _forward(_stage(case), case)
    after = _pools(case["kv"])
    _restore(case["kv"], saved)
    assert got.equal(_composed(case))
    assert after[0].equal(case["kv"].k_pools) and after[1].equal(case["kv"].v_pools)


@pytest.mark.parametrize("name", CASES)
def test_as_on_copies_of_the_prefixes(name):
    """A layer against forward on slots that hold copies of the prompts: K and V bit for bit, attention within both sides'
    roundings."""
    case = _case(name, n_layers=1, seed=3)
    kv, n = case["kv"], len(case["q_lens"])
    flat = KVWorkspace(1, n, 1024, kv.n_kv_heads, 64, DEV)
    for b, (slot, p, start) in enumerate(zip(case["slots"], case["prefixes"], case["starts"])):
        P = p[1] if p else 0
        if p:
            flat.set_dense(0, b, *(f(0, p[0], torch.arange(P, device=DEV)) for f in (kv.k_dense, kv.v_dense)), torch.arange(P, device=DEV))
        own = torch.arange(start - P, device=DEV)
        if len(own):
            flat.set_dense(0, b, *(f(0, slot, own) for f in (kv.k_dense, kv.v_dense)), own + P)
    stage = _stage(case)
    _forward(stage, case)
    st = RaggedStage(case["shape"], case["layers"], case["rot"], flat, max_tokens=max(64, case["T"]), max_seqs=8)
    st.forward(case["hidden"].clone(), case["q_lens"], case["starts"], list(range(n)))
    for b, (slot, p, start, q) in enumerate(zip(case["slots"], case["prefixes"], case["starts"], case["q_lens"])):
        new = torch.arange(start, start + q, device=DEV)
        for f in ("k_dense", "v_dense"):
            assert getattr(kv, f)(0, slot, new - (p[1] if p else 0)).equal(getattr(flat, f)(0, b, new))
    # Attention's rows: either one is off by 2^-8 (sum p |v| + 2 |out|) at most (P to bf16 in the products and the row sum, the result to
    # bf16) and by 2^-12 of sum p |v| for its sums in fp32, and both sums are at most the largest |v| that the row sees.  (The layer's
    # rows are not compared: an expert that is chosen by less than that changes them by any amount.)
    largest = float(max(case["kv"].v_pools.abs().max(), flat.v_pools.abs().max()))
    a, b = (x.debug_buffer(3, torch.bfloat16, (case["T"], 4096)).float() for x in (stage, st))
    assert float((a - b).abs().max()) <= 2 * largest * (3 * 2.0 ** -8 + 2.0 ** -12)
    assert not a.equal(torch.zeros_like(a))


def test_graphs_and_other_lengths():
    """Captured steps: replayed with other starts, prefixes and slots, bit for bit the eager ones; plain steps between them."""
    case = _case("drafts", n_layers=2, seed=5)
    eager, graphs = _stage(case), _stage(case, use_graphs=True)
    saved = _pools(case["kv"])
    for i in range(4):
        step = dict(case, starts=[s + (i if s >= 700 else 0) for s in case["starts"]])
        if i == 3:
            step["prefixes"] = [None if p is None else (p[0], p[1] - 64) for p in case["prefixes"]]
            step["starts"] = [s - 64 if p else s for s, p in zip(step["starts"], case["prefixes"])]
        _restore(case["kv"], saved)
        want = _forward(eager, step)
        plain = eager.forward(case["hidden"].clone()[:1], [1], [10], [2])
        _restore(case["kv"], saved)
        got = _forward(graphs, step)
        assert graphs.forward(case["hidden"].clone()[:1], [1], [10], [2]).equal(plain)
        assert got.equal(want), i
    assert graphs.graphs_captured == 2


def test_none_is_the_plain_step():
    case = _case("decode")
    st = _stage(case)
    args = [1, 2], [5, 100], [2, 3]
    h = case["hidden"][:3]
    want = st.forward(h.clone(), *args)
    for prefixes in (None, [None, None]):
        assert st.forward(h.clone(), *args, prefixes=prefixes).equal(want)


def test_refusals():
    """Before any launch: the pools stay as they were."""
    case = _case("drafts")
    st = RaggedStage(case["shape"], case["layers"], case["rot"], case["kv"], max_tokens=64, max_seqs=8)
    saved = _pools(case["kv"])
    h = case["hidden"]

    def step(q=(1, 1), starts=(700, 130), slots=(3, 5), prefixes=((0, 700), (1, 130))):
        return st.forward(h[:sum(q)].clone(), list(q), list(starts), list(slots), prefixes=list(prefixes))

    with pytest.raises(ValueError, match="set_prefixes"):
        step()
    st.set_prefixes()
    step()
    _restore(case["kv"], saved)
    for error, kw in ((ValueError, dict(prefixes=((0, 700),))), (ValueError, dict(prefixes=((0, 701), None))), (ValueError, dict(prefixes=((7, 1), None))),
                      (ValueError, dict(prefixes=((0, -1), None))), (FlyaiError, dict(starts=(699, 130))),
                      (ContextOverflow, dict(starts=(1000, 130))), (ContextOverflow, dict(starts=(700, 130 + 300))),
                      (FlyaiError, dict(slots=(0, 5))),                              # appends to the slot that it reads
                      (FlyaiError, dict(slots=(1, 5))),                              # ... to another's
                      (FlyaiError, dict(slots=(3, 1), starts=(700, 129), prefixes=((1, 130), None))),  # the owner, before what is read
                      (ContextOverflow, dict(slots=(3, 0), starts=(700, 700), prefixes=((0, 700), None)))):
        with pytest.raises(error):
            step(**kw)
    torch.cuda.synchronize()
    assert case["kv"].k_pools.equal(saved[0]) and case["kv"].v_pools.equal(saved[1])
    st.set_prefixes(False)
    with pytest.raises(ValueError, match="set_prefixes"):
        step()


def test_a_served_model_behind_one_prompt():
    """GptOssModel.step(prefixes=): requests behind one prompt's slot, continued greedily together, commit what each commits alone."""
    from test_gpu_request_edges import _served
    m = _served(False)
    m.stage.set_prefixes()
    prompt = [(7 * i + 3) % 1024 for i in range(60)]
    m.step([prompt], [0], [0], [False])
    own = [[3, 1, 4, 1, 5], [9, 2, 6], [5]]

    def serve(which, steps=5):
        chunks, starts, out = [own[i] for i in which], [60] * len(which), [[] for _ in which]
        for _ in range(steps):
            toks = m.step(chunks, starts, [1 + i for i in which], [True] * len(which), prefixes=[(0, 60)] * len(which))
            starts = [s + len(c) for s, c in zip(starts, chunks)]
            chunks = [[t] for t in toks]
            for o, t in zip(out, toks):
                o.append(t)
        return out

    together = serve([0, 1, 2])
    for i in range(3):
        assert serve([i]) == [together[i]], i
    assert len(set(map(tuple, together))) == 3


@pytest.mark.parametrize("name", ["drafts", "questions"])
def test_adapters_behind_prefixes(name):
    """Adapters of sequences behind prefixes: K and V as on copies of the prompts, bit for bit, and not those without adapters."""
    from test_gpu_stage_lora import _bank
    case = _case(name, seed=9)
    kv, n, ads = case["kv"], len(case["q_lens"]), [0, None, 1, 3, -1, 1]
    bank = _bank(case["shape"], 1)
    flat = KVWorkspace(1, n, 1024, kv.n_kv_heads, 64, DEV)
    st = RaggedStage(case["shape"], case["layers"], case["rot"], flat, max_tokens=max(64, case["T"]), max_seqs=8, lora=bank)
    st.forward(case["hidden"].clone(), case["q_lens"], case["starts"], list(range(n)), adapters=ads)
    saved = _pools(kv)
    _forward(_stage(case), case)
    without = _pools(kv)
    _restore(kv, saved)
    for graphs in (False, True):
        _restore(kv, saved)
        _forward(_stage(case, lora=bank, use_graphs=graphs), case, adapters=ads)
        for b, (slot, p, start, q) in enumerate(zip(case["slots"], case["prefixes"], case["starts"], case["q_lens"])):
            new = torch.arange(start, start + q, device=DEV)
            for f in ("k_dense", "v_dense"):
                assert getattr(kv, f)(0, slot, new - (p[1] if p else 0)).equal(getattr(flat, f)(0, b, new)), (b, f)
        assert not kv.k_pools.equal(without[0])
