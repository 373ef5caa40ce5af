"""ops.pack_shared, rope_kv_append(kv_pos=), attn_shared_plan, attn_shared and spec_verify together: steps of drafted tokens behind shared
prompts, each step's lengths made by the last one on the GPU."""
import numpy as np
import pytest
import torch

from flyai_amd import kvlayout, ops
from oracle import shared as oracle_shared
from oracle import verify as oracle

from shared_batches import DEV, Batch, check

pytestmark = pytest.mark.gpu

HKV, HQ, D, V, OWN = 2, 16, 64, 1008, 192


class Model:
    """One attention layer between an embedding and a head: qkv is a token's row of a table."""

    def __init__(self, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.table = torch.randn(V, (HQ + 2 * HKV) * D, generator=g).to(torch.bfloat16).to(DEV)
        self.head = (torch.randn(V, HQ * D, generator=g) * 0.5).to(torch.bfloat16).to(DEV)
        self.sinks = torch.randn(HQ, generator=g).to(DEV)
        angle = torch.arange(4096)[:, None] * (1e-4 ** (torch.arange(D // 2) / (D // 2)))
        self.cos, self.sin = (f(angle).to(torch.bfloat16).to(DEV) for f in (torch.cos, torch.sin))


class Streams:
    """Streams behind prefixes (-1: behind none) whose caches hold prompts of random keys; K drafts a step."""

    def __init__(self, model, prefixes, of, prompts, K, temps, seed=0):
        self.m, self.K, self.S = model, K, len(of)
        b = Batch(prefixes, [(0, n, p) for n, p in zip(prompts, of)], Hkv=HKV, seed=seed)
        # the prompts' slabs again with room behind them
        n = len(prefixes)
        self.bases = b.bases[:n] + [b.bases[n] + i * HKV * OWN * D for i in range(self.S)]
        self.elems = b.bases[n] + self.S * HKV * OWN * D
        k, v = (torch.full((self.elems,), float("nan"), dtype=torch.bfloat16) for _ in "kv")
        k[:b.bases[n]], v[:b.bases[n]] = b.k[:b.bases[n]].cpu(), b.v[:b.bases[n]].cpu()
        for i, m in enumerate(prompts):
            at = slice(self.bases[n + i], self.bases[n + i] + HKV * OWN * D)
            kvlayout.scatter(k[at], HKV, OWN, "k", b.keys[n + i], torch.arange(m))
            kvlayout.scatter(v[at], HKV, OWN, "v", b.values[n + i], torch.arange(m))
        self.k, self.v, self.batch = k.to(DEV), v.to(DEV), b
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
        i64 = lambda a: torch.tensor(a, dtype=torch.int64, device=DEV)  # noqa: E731
        self.starts, self.last = i32(b.starts), i32([7 * i for i in range(self.S)])
        self.q_lens = i32([K + 1] * self.S)
        self.slabs = dict(kv_base=i64(self.bases[n:]), kv_cap=i32([OWN] * self.S), prefix_of=i32(of), prefix_len=i32(prefixes))
        self.more = dict(prefix_base=i64(self.bases[:n]), prefix_cap=i32(b.caps[:n]))
        self.temp = torch.tensor(temps, dtype=torch.float32, device=DEV)
        self.drafts = torch.zeros(self.S, K, dtype=torch.int32, device=DEV)
        T = self.T = 32  # more rows than tokens, the same for every K: the products of a row do not change
        self.u = torch.zeros(T, dtype=torch.float64, device=DEV)
        self.u_draw = torch.zeros(self.S, dtype=torch.float64, device=DEV)

    def step(self, window):
        """One step, nothing read back: moves last and starts on."""
        m, T = self.m, self.T
        pk = ops.pack_shared(self.q_lens, self.starts, **self.slabs, head_dim=D, max_tokens=T)
        cu, seq = pk["cu_seqlens"].long(), pk["seq_id"].long()
        own = (torch.arange(T, device=DEV) < cu[-1])
        seq = torch.where(own, seq, 0)
        j = torch.where(own, torch.arange(T, device=DEV) - cu[seq], 0)
        chunk = torch.cat((self.last[:, None], self.drafts, torch.full_like(self.last[:, None], -1)), 1)
        tok = chunk[seq, j]
        q = ops.rope_kv_append(m.table[tok.long()], pk["positions"], pk["seq_id"], m.cos, m.sin, HQ, HKV, D, self.slabs["kv_base"],
                               self.slabs["kv_cap"], self.k, self.v, kv_pos=pk["kv_pos"])
        plan = ops.attn_shared_plan(self.q_lens, self.starts, **self.slabs, **self.more, n_kv_heads=HKV, window=window, n_tokens=T,
                                    pool_elems=self.elems)
        out = ops.attn_shared(q, self.k, self.v, m.sinks, plan, out=torch.zeros_like(q))
        logits = ops.linear(out.view(T, HQ * D), m.head)
        draft = torch.where(j + 1 < self.q_lens[seq], chunk[seq, j + 1], -1)
        tokens, counts, p = ops.spec_verify(logits, pk["cu_seqlens"], draft, self.u, self.u_draw, self.temp, 0, 0.9)
        self.last.copy_(tokens[(cu[:-1] + counts - 1).clamp(min=0)])
        self.starts += counts
        return dict(q=q, out=out, logits=logits, draft=draft, tokens=tokens, counts=counts, p=p, status=pk["status"] | plan.status)


PREFIXES, OF, PROMPTS = [700, 130], [0, 1, 0, -1, 0, 1], [0, 5, 63, 64, 1, 20]


@pytest.mark.parametrize("window", [0, 128])
def test_drafted_tokens_are_those_of_single_steps(window):
    """Greedy: whatever is drafted, the tokens are those that one-token steps give, bit for bit the same logits behind them."""
    m, n = Model(), 30
    one = Streams(m, PREFIXES, OF, PROMPTS, 0, [0.0] * len(OF))
    truth = []
    for _ in range(n + 8):
        r = one.step(window)
        assert int(r["status"]) == 0 and bool((r["counts"] == 1).all())
        truth.append(r["tokens"][:one.S].tolist())
    truth = np.array(truth).T  # [S, n + 8]
    K = 3
    many = Streams(m, PREFIXES, OF, PROMPTS, K, [0.0] * len(OF))
    have = [[] for _ in OF]
    sizes = set()
    while min(map(len, have)) < n:
        q = [0 if len(h) >= n else 1 + (len(h) + s) % (K + 1) for s, h in enumerate(have)]  # some streams have fewer drafts, or are done
        drafts = [[int(truth[s, len(h) + i]) if (3 * len(h) + i + s) % 5 else 999 for i in range(K)] for s, h in enumerate(have)]
        many.q_lens.copy_(torch.tensor(q))
        many.drafts.copy_(torch.tensor(drafts))
        before = many.last.clone()
        r = many.step(window)
        assert int(r["status"]) == 0
        counts, tokens, at = r["counts"].tolist(), r["tokens"].tolist(), 0
        for s, h in enumerate(have):
            assert (counts[s] == 0) == (q[s] == 0)
            h += tokens[at:at + counts[s]]
            at += q[s]
            if q[s] == 0:
                many.last[s] = before[s]
            sizes.add(counts[s])
    for s, h in enumerate(have):
        assert h == truth[s, :len(h)].tolist(), s
    assert sizes == {0, 1, 2, 3, 4}


def test_a_step_against_the_formulas():
    """Attention of the appended keys, and the tokens of its logits, in 64 bits."""
    s = Streams(Model(1), PREFIXES, OF, PROMPTS, 2, [0.0, 0.8, 1.0, 1.2, 0.0, 0.5], seed=3)
    rng = np.random.default_rng(5)
    for _ in range(3):
        before = s.starts.tolist()
        s.u.copy_(torch.tensor(rng.random(s.T)))
        s.u_draw.copy_(torch.tensor(rng.random(s.S)))
        s.drafts.copy_(torch.tensor(rng.integers(0, V, (s.S, s.K))))
        r = s.step(0)
        tokens, counts, p = (r[k].cpu().numpy() for k in ("tokens", "counts", "p"))
        draft, logits = r["draft"].cpu().numpy(), r["logits"].cpu()
        k, v, n = s.k.cpu(), s.v.cpu(), len(PREFIXES)
        for b, (of, start) in enumerate(zip(OF, before)):
            P, rows = (PREFIXES[of] if of >= 0 else 0), slice(3 * b, 3 * b + 3)
            at = slice(s.bases[n + b], s.bases[n + b] + HKV * OWN * D)
            held = torch.arange(start + 3 - P)
            keys, values = (kvlayout.gather(x[at], HKV, OWN, w, held) for x, w in ((k, "k"), (v, "v")))
            if of >= 0:
                keys, values = torch.cat((s.batch.keys[of], keys), 1), torch.cat((s.batch.values[of], values), 1)
            want, mag = oracle_shared.attention(r["q"][rows].cpu(), keys, values, start, s.m.sinks.cpu(), 0)
            check(r["out"][rows], want, mag)
            t, pr = oracle.stream(logits[rows].float().numpy(), draft[rows], [None] * 3, float(s.temp[b]), 0, np.float32(0.9),
                                     s.u[rows].cpu().numpy(), float(s.u_draw[b]))
            assert counts[b] == len(t) and tokens[rows].tolist() == list(t) + [-1] * (3 - len(t)), b
            assert np.all(np.abs(p[rows][:len(t)] - np.array(pr)) <= np.array(pr) * 2.0 ** -23)


def test_keys_land_where_kv_pos_says():
    """rope_kv_append with kv_pos: the bits that the same positions have in a slab that starts at position 0."""
    m, T = Model(2), 9
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(T, (HQ + 2 * HKV) * D, generator=g).to(torch.bfloat16).to(DEV)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    pos, seq, kv_pos = i32([130, 131, 132, 133, 900, 901, 64, 65, 66]), i32([0] * 4 + [1] * 2 + [2] * 3), i32([0, 1, 2, 3, 63, 64, 127, 128, -1])
    cap = 1024
    base = torch.arange(3, dtype=torch.int64, device=DEV) * HKV * cap * D
    full = [torch.zeros(3 * HKV * cap * D, dtype=torch.bfloat16, device=DEV) for _ in "kv"]
    q0 = ops.rope_kv_append(qkv, pos, seq, m.cos, m.sin, HQ, HKV, D, base, i32([cap] * 3), *full)
    moved = [torch.zeros(3 * HKV * 128 * D, dtype=torch.bfloat16, device=DEV) for _ in "kv"]
    base2 = torch.arange(3, dtype=torch.int64, device=DEV) * HKV * 128 * D
    q1 = ops.rope_kv_append(qkv, pos, seq, m.cos, m.sin, HQ, HKV, D, base2, i32([128] * 3), *moved, kv_pos=kv_pos)
    assert q0.equal(q1)
    for a, b, which in zip(full, moved, "kv"):
        for s in range(3):
            want = kvlayout.gather(a.cpu()[s * HKV * cap * D:(s + 1) * HKV * cap * D], HKV, cap, which, torch.arange(cap))
            got = kvlayout.gather(b.cpu()[s * HKV * 128 * D:(s + 1) * HKV * 128 * D], HKV, 128, which, torch.arange(128))
            there = torch.zeros(128, dtype=torch.bool)
            for t in range(T):
                if int(seq[t]) == s and 0 <= int(kv_pos[t]) < 128:  # outside the slab: nothing is written
                    assert got[:, int(kv_pos[t])].equal(want[:, int(pos[t])])
                    there[int(kv_pos[t])] = True
            assert not bool(got[:, ~there].any())


def test_rows_of_no_sequence():
    """A batch of fewer tokens than rows: -1 behind the last, and nothing is appended for them."""
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    for q_lens in ([2, 0, 1], [0, 0, 0]):
        T, n = 2100, sum(q_lens)
        pk = ops.pack_shared(i32(q_lens), i32([5, 0, 64]), torch.arange(3, dtype=torch.int64, device=DEV) * HKV * 128 * D, i32([128] * 3),
                             i32([-1, -1, 0]), i32([64]), D, T)
        assert all(bool((pk[k][n:] == -1).all()) and bool((pk[k][:n] >= 0).all()) for k in ("positions", "seq_id", "kv_pos", "kv_slot"))
        m = Model(3)
        pools = [torch.zeros(3 * HKV * 128 * D, dtype=torch.bfloat16, device=DEV) for _ in "kv"]
        ops.rope_kv_append(m.table[torch.arange(T, device=DEV) % V], pk["positions"], pk["seq_id"], m.cos, m.sin, HQ, HKV, D,
                           torch.arange(3, dtype=torch.int64, device=DEV) * HKV * 128 * D, i32([128] * 3), *pools, kv_pos=pk["kv_pos"])
        assert all(int((x != 0).sum()) <= n * HKV * D for x in pools) and (n == 0 or bool(pools[0].any()))


def test_steps_in_a_graph():
    """The loop captured once and replayed: the same tokens, lengths and caches as eager steps, which run between the replays."""
    mk = lambda: Streams(Model(4), PREFIXES, OF, PROMPTS, 2, [0.0, 0.8, 1.0, 1.2, 0.0, 0.5], seed=3)  # noqa: E731
    a, b = mk(), mk()
    for s in (a, b):  # warm, then from the start again
        keep = s.starts.clone(), s.last.clone()
        s.step(0)
        s.starts.copy_(keep[0]), s.last.copy_(keep[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = b.step(0)
    rng = np.random.default_rng(6)
    for i in range(6):
        u, u_draw, drafts = torch.tensor(rng.random(a.T)), torch.tensor(rng.random(a.S)), torch.tensor(rng.integers(0, V, (a.S, a.K)))
        for s in (a, b):
            s.u.copy_(u), s.u_draw.copy_(u_draw), s.drafts.copy_(drafts)
        graph.replay()
        torch.cuda.synchronize()
        want = a.step(0)
        R = a.S * (a.K + 1)
        assert all(got[k][:R].equal(want[k][:R]) for k in want), i
        assert a.starts.equal(b.starts) and a.last.equal(b.last)
        assert a.k.view(torch.int16).equal(b.k.view(torch.int16)) and a.v.view(torch.int16).equal(b.v.view(torch.int16))


def test_two_batches_on_two_streams():
    """Two batches' steps at once, each on a stream of its own: workspaces are the calls' own."""
    mk = lambda i: Streams(Model(5 + i), PREFIXES, OF, PROMPTS, 2, [0.0] * 6, seed=i)  # noqa: E731
    want = [[{k: v.clone() for k, v in s.step(0).items()} for _ in range(4)] for s in (mk(0), mk(1))]
    both = [mk(0), mk(1)]
    lanes = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, lane in enumerate(lanes):
            with torch.cuda.stream(lane):
                got[i].append(both[i].step(0))
    torch.cuda.synchronize()
    R = 18
    for i in range(2):
        for x, y in zip(got[i], want[i]):
            assert all(x[k][:R].equal(y[k][:R]) for k in y)


def test_refused_sequences_are_appended_nowhere():
    """A sequence that starts before its prefix ends, or whose prefix or start is bad, has no slab position at any of its tokens, and the
    keys that lie in its slab stay.  One that runs past its slab, or past the rows, keeps the positions of the tokens that fit."""
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    m, cap, q_lens = Model(6), 64, [3, 4, 2]
    base = torch.arange(3, dtype=torch.int64, device=DEV) * HKV * cap * D
    want = [5, 6, 7, 0, 1, 2, 3, 9, 10]  # of starts (105, 30, 9) behind 100 and 30 positions and none
    for change, bit, lost in (({}, 0, ()), (dict(starts=[98, 30, 9]), ops.BEFORE_PREFIX, (0, 1, 2)), (dict(starts=[105, 29, 9]), ops.BEFORE_PREFIX, (3, 4, 5, 6)),
                              (dict(starts=[105, 30, -1]), ops.BAD_SEQUENCE, (7, 8)), (dict(prefix_of=[0, 2, -1]), ops.BAD_PREFIX, (3, 4, 5, 6)),
                              (dict(prefix_len=[-7, 30]), ops.BAD_PREFIX, (0, 1, 2)), (dict(prefix_len=[107, 30]), ops.BEFORE_PREFIX, (0, 1, 2)),
                              (dict(starts=[162, 30, 9]), ops.PAST_SLAB, ()), (dict(max_tokens=8), ops.PAST_TOKENS, ())):
        args = dict(starts=[105, 30, 9], prefix_of=[0, 1, -1], prefix_len=[100, 30], max_tokens=9)
        args.update(change)
        T = args["max_tokens"]
        pk = ops.pack_shared(i32(q_lens), i32(args["starts"]), base, i32([cap] * 3), i32(args["prefix_of"]), i32(args["prefix_len"]), D, T)
        at = [-1 if t in lost else w for t, w in enumerate(want)][:T]
        if bit == ops.PAST_SLAB:
            at[:3] = [62, 63, 64]
        seq = [0, 0, 0, 1, 1, 1, 1, 2, 2]
        slots = [int(base[seq[t]]) + p * D if 0 <= p < cap else -1 for t, p in enumerate(at)]
        assert int(pk["status"]) == bit and pk["kv_pos"].tolist() == at and pk["kv_slot"].tolist() == slots, change
        pools = [torch.zeros(3 * HKV * cap * D, dtype=torch.bfloat16, device=DEV) for _ in "kv"]
        ops.rope_kv_append(m.table[:T], pk["positions"], pk["seq_id"], m.cos, m.sin, HQ, HKV, D, base, i32([cap] * 3), *pools, kv_pos=pk["kv_pos"])
        for pool, which in zip(pools, "kv"):
            for s in range(3):
                rows = kvlayout.gather(pool.cpu()[s * HKV * cap * D:(s + 1) * HKV * cap * D], HKV, cap, which, torch.arange(cap))
                there = {p for t, p in enumerate(at) if seq[t] == s and 0 <= p < cap}
                assert {int(p) for p in torch.nonzero(rows.abs().sum((0, 2)))[:, 0]} == there, (change, s)


def test_idle_sequences_of_another_time():
    """Sequences without tokens whose prefix, start or slab are no longer any: pack_shared and the plan pass over them alike, and the others' rows
    are those of the batch without them."""
    b = Batch([100, 30], [(2, 5, 0), (0, 3, 0), (3, 0, 1), (0, 4, -1), (0, 9, 1), (1, 7, -1)], Hkv=HKV, seed=8)
    want, _ = b.run(0)
    packed = ops.pack_shared(**b.lengths(), head_dim=D, max_tokens=b.T)
    stale = b.lengths()
    for name, i, v in (("prefix_of", 1, 7), ("starts", 3, 2 ** 31 - 1), ("kv_cap", 3, 0), ("kv_base", 3, -8), ("starts", 4, 3)):
        stale[name][i] = v
    got = ops.pack_shared(**stale, head_dim=D, max_tokens=b.T)
    assert int(got["status"]) == 0
    assert all(got[k].equal(packed[k]) for k in ("cu_seqlens", "positions", "seq_id", "kv_pos", "kv_slot"))
    out, plan = b.run(0, **stale)
    assert int(plan.status) == 0 and out.equal(want)
    stale["starts"][1] = -1  # a start that is none is reported, with tokens or without
    assert int(ops.pack_shared(**stale, head_dim=D, max_tokens=b.T)["status"]) == int(b.plan(0, **stale).status) == ops.BAD_SEQUENCE
