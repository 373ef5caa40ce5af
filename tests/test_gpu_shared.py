"""ops.pack_shared and ops.attn_shared against the oracle: sequences behind shared prefixes."""
import pytest
import torch

from flyai_amd import kvlayout, ops
from oracle import shared as oracle
from shared_batches import DEV, Batch, check

pytestmark = pytest.mark.gpu


def packed(b, max_tokens=None):
    return ops.pack_shared(**b.lengths(), head_dim=64, max_tokens=b.T if max_tokens is None else max_tokens)


@pytest.mark.parametrize("S,q", [(1, 1), (3, 5), (64, 1), (65, 9), (1025, 3), (8192, 2), (3, 3000)])
def test_pack_shared(S, q):
    prefixes = [0, 1, 700, 64]
    b = Batch.__new__(Batch)
    b.prefixes, b.Hkv = prefixes, 2
    b.q_lens = [(i * 7 + q) % (q + 1) for i in range(S)]
    b.prefix_of = [i % 5 - 1 for i in range(S)]
    b.starts = [(prefixes[p] if p >= 0 else 0) + 13 * i % 50 for i, p in enumerate(b.prefix_of)]
    b.caps = [0] * 4 + [64 * (1 + (50 + n) // 64) for n in b.q_lens]
    b.bases = [0] * 4 + [2 ** 33 + 4096 * i for i in range(S + 1)]
    b.T = sum(b.q_lens)
    got = packed(b, b.T + 5)
    n = len(prefixes)
    want = oracle.pack(b.q_lens, b.starts, b.bases[n:-1], b.caps[n:], b.prefix_of, prefixes, 64)
    for name, w in zip(("cu_seqlens", "positions", "seq_id", "kv_pos", "kv_slot", "kv_len"), want):
        t = got[name] if name in ("cu_seqlens", "kv_len") else got[name][:b.T]
        assert t.tolist() == w, name
    assert got["status"].item() == 0


def test_pack_shared_refusals():
    """Each bad sequence sets its bit and gets no slot; the others are packed as they would be alone."""
    b = Batch([100, 30], [(2, 5, 0), (3, 0, 1), (1, 4, -1), (2, 9, 0)])
    base = packed(b)
    n = len(b.prefixes)

    def with_(**change):
        args = b.lengths()
        for name, (i, v) in change.items():
            args[name][i] = v
        return ops.pack_shared(**args, head_dim=64, max_tokens=b.T)

    rows = {0: slice(0, 2), 1: slice(2, 5), 2: slice(5, 6), 3: slice(6, 8)}
    for change, bit, seq in ((dict(starts=(0, 99)), ops.BEFORE_PREFIX, 0), (dict(starts=(1, 30 + b.caps[n + 1] - 2)), ops.PAST_SLAB, 1),
                             (dict(prefix_of=(3, 2)), ops.BAD_PREFIX, 3), (dict(starts=(2, -5)), ops.BAD_SEQUENCE, 2),
                             (dict(starts=(2, 2 ** 31 - 1)), ops.PAST_SLAB, 2), (dict(prefix_len=(1, -4)), ops.BAD_PREFIX, 1)):
        got = with_(**change)
        assert got["status"].item() == bit, change
        assert -1 in got["kv_slot"][rows[seq]].tolist()
        for other, r in rows.items():
            if other != seq:
                assert got["kv_slot"][r].equal(base["kv_slot"][r])
    got = ops.pack_shared(**b.lengths(), head_dim=64, max_tokens=b.T - 1)
    assert got["status"].item() == ops.PAST_TOKENS and got["positions"].equal(base["positions"][:-1])
    args = b.lengths()
    args["q_lens"][1] = -7
    got = ops.pack_shared(**args, head_dim=64, max_tokens=b.T)
    assert got["status"].item() == ops.BAD_SEQUENCE and got["cu_seqlens"].tolist() == [0, 2, 2, 3, 5]


PREFIXES = [1, 63, 64, 65, 130, 513, 1999]


@pytest.mark.parametrize("window", [0, 1, 64, 128, 700])
@pytest.mark.parametrize("P", PREFIXES)
def test_one_prefix(P, window):
    """Rows of one to forty tokens behind one prefix, own keys from none to several chunks."""
    seqs = [(1, 0, 0), (1, 37, 0), (4, 60, 0), (5, 3, 0), (2, 129, 0), (17, 0, 0), (40, 100, 0), (3, 1200, 0)]
    b = Batch([P], seqs, seed=P + window)
    got, plan = b.run(window)
    assert plan.status.item() == 0
    check(got, *b.expected(window))


@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 16, 17, 33])
def test_few_tokens(n, window):
    """One token each: a wave's item, one tile, and past it."""
    b = Batch([333], [(1, i % 5, 0) for i in range(n)], Hkv=1, seed=n)
    got, _ = b.run(window)
    check(got, *b.expected(window))


@pytest.mark.parametrize("window", [0, 128])
def test_many_prefixes(window):
    """Prefixes with many, few and no sequences, of length zero, and sequences without one."""
    prefixes = [300, 0, 77, 1030, 5, 64]
    seqs = [(1, 10, 0)] * 20 + [(2, 0, 1), (1, 64, 2), (3, 500, 2), (4, 8, 3), (6, 0, 3), (1, 0, 4), (1, 700, -1), (9, 0, -1), (0, 4, 0), (2, 63, -1)]
    b = Batch(prefixes, seqs, Hkv=3, seed=5)
    got, plan = b.run(window)
    assert plan.status.item() == 0
    check(got, *b.expected(window))


@pytest.mark.parametrize("spread", [0.01, 3.0])
def test_spreads(spread):
    """Near-equal scores, and scores of a hundred that a few keys win."""
    b = Batch([1500], [(3, 20, 0), (1, 0, 0), (2, 300, 0)], seed=9, spread=spread)
    got, _ = b.run(0)
    check(got, *b.expected(0))


def test_rows_do_not_depend_on_the_batch():
    """The same sequences alone, with others of their prefix, and in a batch large enough that an item takes all the chunks of a range."""
    for window in (0, 128, 900):
        seqs = [(2, 600, 0), (5, 3, 0), (1, 0, 1), (3, 1100, -1)]
        small = Batch([2000, 700], seqs, Hkv=8, seed=3)
        got, _ = small.run(window)
        t = 0
        for b, s in enumerate(seqs):  # alone
            one, _ = small.run(window, q_lens=torch.tensor([s[0] if i == b else 0 for i in range(len(seqs))], dtype=torch.int32, device=DEV))
            # (its rows come first then: the same queries have to be there)
            alone = Batch.__new__(Batch)
            alone.__dict__.update(small.__dict__)
            alone.q = small.q.roll(-t, 0)
            one, _ = alone.run(window, q_lens=torch.tensor([s[0] if i == b else 0 for i in range(len(seqs))], dtype=torch.int32, device=DEV))
            assert one[:s[0]].equal(got[t:t + s[0]]), (window, b)
            t += s[0]
        crowd = Batch([2000, 700], seqs + [(4, 50, i % 2) for i in range(300)], Hkv=8, seed=3)
        n = len(small.prefixes) + len(seqs)
        for i in range(n):  # the same keys
            crowd.keys[i], crowd.values[i] = small.keys[i], small.values[i]
        k, v = crowd.k.cpu(), crowd.v.cpu()
        k[:small.elems], v[:small.elems] = small.k.cpu(), small.v.cpu()
        crowd.k, crowd.v = k.to(DEV), v.to(DEV)
        crowd.q[:small.T], crowd.sinks = small.q, small.sinks
        many, plan = crowd.run(window)
        assert plan.status.item() == 0
        assert many[:small.T].equal(got), window
        want = crowd.expected(window)
        check(many, *want)


def test_masked_values_of_any_kind():
    """Infinities and NaN in keys and values that some rows see and others do not reach only the rows that see them."""
    for window in (0, 70):
        b = Batch([200], [(6, 30, 0), (3, 0, 0), (1, 64, 0)], seed=1)
        own = b.values[1]  # the first sequence's own slab: its fourth new token
        own[0, 33, 5], own[0, 33, 6], own[1, 34, 7] = float("inf"), float("-inf"), float("nan")
        b.keys[1][1, 35, 9] = float("nan")
        b.values[0][0, 160, 11] = float("inf")  # seen through the window by some
        b.rewrite(0)
        b.rewrite(1)
        got, _ = b.run(window)
        want, mag = b.expected(window)
        got = got.double().cpu()
        assert got.isnan().equal(want.isnan()) and got.isinf().equal(want.isinf()), window
        inf = want.isinf()
        assert got[inf].equal(want[inf])
        ok = want.isfinite()
        assert bool(ok.any(0).any()) and not bool(ok.all())
        check(torch.where(ok, got, 0.0), torch.where(ok, want, 0.0), torch.where(ok & mag.isfinite(), mag, 0.0))


def test_refused_sequences_are_zeros():
    b = Batch([100, 30], [(2, 5, 0), (3, 0, 1), (1, 4, -1), (2, 9, 0)])
    base, _ = b.run(0)
    rows = {0: slice(0, 2), 1: slice(2, 5), 2: slice(5, 6), 3: slice(6, 8)}
    n = len(b.prefixes)

    def changed(name, i, v):
        t = b.lengths()[name] if name in b.lengths() else torch.tensor(b.bases[:n], dtype=torch.int64, device=DEV)
        t[i] = v
        return {name: t}

    for change, bit, seqs in ((changed("starts", 0, 99), ops.BEFORE_PREFIX, (0,)), (changed("starts", 1, 30 + b.caps[n + 1] - 2), ops.PAST_SLAB, (1,)),
                              (changed("prefix_of", 3, 2), ops.BAD_PREFIX, (3,)), (changed("starts", 2, -5), ops.BAD_SEQUENCE, (2,)),
                              (changed("starts", 2, 2 ** 31 - 1), ops.PAST_SLAB, (2,)), (changed("prefix_len", 1, 65), ops.BAD_PREFIX, (1,)),
                              (changed("prefix_len", 0, -1), ops.BAD_PREFIX, (0, 3)), (changed("prefix_base", 0, b.elems - 64), ops.BAD_PREFIX, (0, 3)),
                              (changed("prefix_base", 0, 2 ** 62), ops.BAD_PREFIX, (0, 3)), (changed("kv_base", 2, b.elems), ops.BAD_SEQUENCE, (2,)),
                              (changed("kv_base", 2, -8), ops.BAD_SEQUENCE, (2,)), (changed("kv_base", 2, 2 ** 63 - 8), ops.BAD_SEQUENCE, (2,)),
                              (changed("kv_base", 2, 4), ops.BAD_SEQUENCE, (2,)), (changed("kv_cap", 2, 2 ** 31 - 64), ops.BAD_SEQUENCE, (2,)),
                              (changed("kv_cap", 2, 100), ops.BAD_SEQUENCE, (2,))):
        got, plan = b.run(0, **change)
        assert plan.status.item() == bit, change
        for s, r in rows.items():
            assert got[r].equal(torch.zeros_like(got[r]) if s in seqs else base[r]), (change, s)


def test_more_tokens_than_rows():
    """The sequence that does not fit is refused whole; rows behind the last sequence stay as they were."""
    b = Batch([100], [(2, 5, 0), (3, 0, 0), (4, 7, 0)], extra_rows=3)
    full, plan = b.run(0)
    assert plan.status.item() == 0
    out = torch.full((b.T, 16, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    got, _ = b.run(0, out=out)
    assert got[:9].equal(full[:9]) and bool((got[9:] == 7).all())
    plan = b.plan(0, n_tokens=8)
    got = ops.attn_shared(b.q[:8].to(DEV).contiguous(), b.k, b.v, b.sinks.to(DEV), plan)
    assert plan.status.item() == ops.PAST_TOKENS
    assert got[:5].equal(full[:5]) and not bool(got[5:].any())


def test_no_tokens():
    b = Batch([100], [(0, 5, 0), (0, 0, -1)], extra_rows=2)
    out = torch.full((2, 16, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    got, plan = b.run(0, out=out)
    assert plan.status.item() == 0 and bool((got == 7).all())


def test_captured_and_replayed_with_other_lengths():
    """Plan and attention in a graph: the lengths, on the GPU, change between replays; eager calls run between them."""
    b = Batch([700], [(2, 400, 0), (1, 300, 0), (3, 500, -1)], Hkv=8, seed=2)
    lengths = b.lengths()
    q, sinks = b.q.to(DEV), b.sinks.to(DEV)
    n = len(b.prefixes)
    more = dict(prefix_base=torch.tensor(b.bases[:n], dtype=torch.int64, device=DEV), prefix_cap=torch.tensor(b.caps[:n], dtype=torch.int32, device=DEV),
                n_kv_heads=8, window=0, n_tokens=b.T, pool_elems=b.elems)

    def step():
        pk = ops.pack_shared(**lengths, head_dim=64, max_tokens=b.T)
        return pk["kv_slot"], ops.attn_shared(q, b.k, b.v, sinks, ops.attn_shared_plan(**lengths, **more))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        slots, out = step()
    starts = lengths["starts"].clone()
    for back in (0, 100, 3, 290):
        lengths["starts"].copy_(starts - back)
        graph.replay()
        torch.cuda.synchronize()
        want_slots, want = step()
        assert slots.equal(want_slots) and out.equal(want), back


def test_other_stream():
    b = Batch([900], [(2, 100, 0), (1, 30, 0)], Hkv=8, seed=2)
    want, _ = b.run(128)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got, _ = b.run(128)
    s.synchronize()
    assert got.equal(want)


def test_positions_past_32_bits_of_elements():
    """A slab at an element offset past 2^31."""
    b = Batch([130], [(2, 70, 0), (1, 3, 0)], Hkv=2, seed=4)
    want, _ = b.run(0)
    far = 2 ** 31 + 4096
    k = torch.empty(far + b.elems, dtype=torch.bfloat16, device=DEV)
    v = torch.empty_like(k)
    k[far:], v[far:] = b.k, b.v
    n = len(b.prefixes)
    plan = b.plan(0, kv_base=b.lengths()["kv_base"] + far, prefix_base=torch.tensor(b.bases[:n], dtype=torch.int64, device=DEV) + far,
                  pool_elems=k.numel())
    got = ops.attn_shared(b.q.to(DEV), k, v, b.sinks.to(DEV), plan)
    assert got.equal(want)


def test_a_plan_of_another_shape():
    """Nothing is done with it."""
    b = Batch([130], [(2, 70, 0), (1, 3, 0), (9, 100, 0)], Hkv=2, seed=4)
    plan = b.plan(0)
    q, sinks = b.q.to(DEV), b.sinks.to(DEV)
    for change in (dict(n_tokens=b.T - 1), dict(n_seqs=2), dict(n_prefixes=0), dict(n_kv_heads=1)):
        other = ops.AttnSharedPlan(**{**{n: getattr(plan, n) for n in plan.__slots__}, **change})
        T, Hkv = other.n_tokens, other.n_kv_heads
        out = torch.full((T, 8 * Hkv, 64), 7.0, dtype=torch.bfloat16, device=DEV)
        ops.attn_shared(q[:T, :8 * Hkv].contiguous(), b.k, b.v, sinks[:8 * Hkv].contiguous(), other, out=out)
        assert bool((out == 7).all()), change


@pytest.mark.parametrize("window", [0, 5000])
@pytest.mark.parametrize("P", [6145, 18433, 18432, 27700, 33000])
def test_long_prefixes(P, window):
    """Chunks of other lengths, and own keys of several chunks."""
    b = Batch([P], [(1, 900, 0), (3, 0, 0), (9, 385, 0)], Hkv=1, seed=P)
    got, plan = b.run(window)
    assert int(plan.status) == 0
    check(got, *b.expected(window))


@pytest.mark.parametrize("n,Hkv,P", [(1, 8, 1600), (40, 8, 1600), (65, 8, 1600), (90, 8, 1600), (60, 1, 30000), (200, 1, 2000), (20, 16, 9000)])
def test_tiles_and_rounds(n, Hkv, P):
    """Tiles that fill no round of the workgroups, more than one, and whole or split rests: every row's bits are those that its sequence
    has in a batch of its own."""
    b = Batch([P], [(16, 3 * i % 70, 0) for i in range(n)], Hkv=Hkv, seed=n)
    got, _ = b.run(0)
    alone = Batch.__new__(Batch)
    alone.__dict__.update(b.__dict__)
    for i in {0, n // 2, n - 1}:
        alone.seqs, alone.q_lens, alone.starts, alone.prefix_of = ([x[i]] for x in (b.seqs, b.q_lens, b.starts, b.prefix_of))
        alone.q, alone.T = b.q[16 * i:16 * i + 16], 16
        alone.bases, alone.caps = [*b.bases[:1], b.bases[1 + i], None], [b.caps[0], b.caps[1 + i]]
        assert alone.run(0)[0].equal(got[16 * i:16 * i + 16]), i


@pytest.mark.parametrize("window", [0, 90])
@pytest.mark.parametrize("S,n", [(1025, 65), (2500, 300), (4096, 1024)])
def test_thousands_of_sequences(S, n, window):
    """Several sequences a thread of the plan, more prefixes than a wave has lanes, of 0 to 5 tokens, behind a prefix or none."""
    prefixes = [(37 * i) % 150 for i in range(n)]
    b = Batch(prefixes, [((i * 5 + i // 7) % 6, i * 11 % 60, (i * 7) % (n + 1) - 1) for i in range(S)], Hkv=1, seed=S)
    got, plan = b.run(window)
    assert plan.status.item() == 0
    check(got, *b.expected(window))


def test_the_most_rows():
    """65,536 of them."""
    b = Batch([500], [(256, 0, 0 if i % 8 else -1) for i in range(256)], Hkv=1, seed=12)
    assert b.T == 65536
    got, plan = b.run(0)
    assert plan.status.item() == 0
    check(got, *b.expected(0))


class Counted(Batch):
    """All keys zero, so that every key that a row sees has the weight 1, and the sinks too; value (kv head, dim) of position p is 1 where
    (p + shift) % period is 64 * head + dim and 0 else.  A row's result is the number of such positions that it sees over all that it sees and
    one: with up to 120 of them, a key that is lost or taken twice changes it by more than 2^-7 of itself, two half steps of bf16."""

    def __init__(self, prefixes, seqs, Hkv=8, period=512, shift=0):
        one = Batch([1] * len(prefixes), [(s[0], 0, -1) for s in seqs], Hkv=Hkv, seed=1)  # (for the queries)
        self.__dict__.update(one.__dict__)
        self.prefixes, self.seqs, self.period, self.shift = prefixes, seqs, period, shift
        self.prefix_of = [s[2] for s in seqs]
        self.behind = [prefixes[p] if p >= 0 else 0 for p in self.prefix_of]
        self.starts = [b + s[1] for b, s in zip(self.behind, seqs)]
        lens = [*prefixes, *(s[0] + s[1] for s in seqs)]
        self.caps = [max(64, (n + 63) // 64 * 64) for n in lens]
        self.bases = [0]
        for c in self.caps:
            self.bases.append(self.bases[-1] + Hkv * c * 64)
        self.elems = self.bases[-1]
        self.k = torch.full((self.elems,), float("nan"), dtype=torch.bfloat16, device=DEV)
        self.v = self.k.clone()
        for base, cap, n, first in zip(self.bases, self.caps, lens, [0] * len(prefixes) + self.behind):
            if n:
                c = (first + torch.arange(n, device=DEV) + shift) % period
                rows = (c[:, None] == torch.arange(64 * Hkv, device=DEV)).reshape(n, Hkv, 64).transpose(0, 1)
                slab = slice(base, base + Hkv * cap * 64)
                kvlayout.scatter(self.k[slab], Hkv, cap, "k", torch.zeros_like(rows), torch.arange(n))
                kvlayout.scatter(self.v[slab], Hkv, cap, "v", rows, torch.arange(n))
        self.sinks.zero_()

    def counts(self, window):
        """(numbers [T, 64 Hkv], all that a row sees [T])."""
        at = torch.tensor([a + i for a, s in zip(self.starts, self.seqs) for i in range(s[0])])
        lo = (at - window + 1).clamp_min(0) if window else torch.zeros_like(at)
        first = (torch.arange(64 * self.Hkv) - self.shift) % self.period
        below = lambda n: (n[:, None] - first + self.period - 1) // self.period  # noqa: E731
        return below(at + 1) - below(lo), at + 1 - lo

    def check(self, window, **change):
        """P, sums and folds are whole numbers below 2^24, exact; the reciprocal and its product round by 2^-24 each, the result by half a
        step, 2^-8."""
        got, plan = self.run(window, **change)
        assert plan.status.item() == 0
        n, seen = self.counts(window)
        assert int(n.max()) <= 120
        want = (n.double() / (seen + 1).double()[:, None]).reshape(-1, self.Hkv, 1, 64)
        bad = (got.double().cpu().reshape(-1, self.Hkv, 8, 64) - want).abs() > want * (2.0 ** -8 + 2.0 ** -22)
        assert not bool(bad.any()), (int(bad.sum()), torch.nonzero(bad)[:4].tolist())


# one tile less and one more than a head's 64 workgroups, and rests that are split and whole; the sequence of a wave, of a tile and of several
COUNTED = {"few": [(1, 900, 0), (3, 0, 0), (9, 385, 0)], "one": [(1, 0, 0)], "long": [(40, 770, 0), (300, 100, 0)],
           "20": [(16, 3 * i % 70, 0) for i in range(20)], "63": [(16, 3 * i % 70, 0) for i in range(63)], "70": [(16, 5, 0)] * 70,
           "130": [(16, 5, 0)] * 130, "crowd": [(1 + i % 5, 7 * i % 500, i % 2) for i in range(200)]}


@pytest.mark.parametrize("window", [0, 1, 5000])
@pytest.mark.parametrize("P", [1, 1537, 6145, 18433, 33000])
@pytest.mark.parametrize("name", COUNTED)
def test_every_key_counts_once(name, P, window):
    Counted([P, max(P - 700, 0)], COUNTED[name]).check(window)


@pytest.mark.parametrize("window", [0, 5000])
@pytest.mark.parametrize("P", [6145, 18432, 18433, 27700, 33000])
def test_border_keys_decide(P, window):
    """64 positions of each kv head have a key along an axis of its own that outweighs all others for the rows along it: first and last
    positions of blocks and of chunks, the prefix's last, the own slab's first, and both sides of the window's edge."""
    seqs = [(1, 900, 0), (3, 0, 0), (9, 385, 0), (4, 5, 0)]
    b = Batch([P], seqs, Hkv=2, seed=P)
    c = 12.0  # scores 18: e^18 to the 34,000 others' some 1
    rng = torch.Generator().manual_seed(P)
    borders = [torch.arange(step, P, step) for step in (192, 64)]  # chunks are multiples of 192 positions, blocks 64
    for h in range(2):
        edge = [P - 1, 0, P - 2, 63, 64] + [P - 5000 + i for i in (-1, 0, 1, 2, 3) if P > 5001]
        near = [int(s) - i % 2 for steps in borders for i, s in enumerate(steps[torch.randperm(len(steps), generator=rng)])]
        at = list(dict.fromkeys(edge + near))[:64]
        k = b.keys[0][h].float() * 0.05
        k[at] = torch.eye(64) * c
        b.keys[0][h] = k.to(torch.bfloat16)
    for i in range(len(seqs)):
        b.keys[1 + i] *= 0.05
    b.k, b.v = b.k.cpu(), b.v.cpu()
    for i, k in enumerate(b.keys):
        b._write(b.bases[i], b.caps[i], k.shape[1], k, b.values[i])
    b.k, b.v = b.k.to(DEV), b.v.to(DEV)
    axis = torch.arange(b.T * 16).reshape(b.T, 2, 8) % 8 + 8 * (torch.arange(b.T)[:, None, None] % 8)  # a row's, of each kv head
    b.q = (torch.eye(64)[axis.reshape(-1)] * c).reshape(b.T, 16, 64).to(torch.bfloat16)
    got, plan = b.run(window)
    assert plan.status.item() == 0
    want, mag = b.expected(window)
    assert float((want.abs().amax(2) > 0.5).float().mean()) > (0.95 if window == 0 else 0.1)  # the planted values come through
    check(got, want, mag)


def _behind_one_slab(b, n):
    """The batch's prefix under n names."""
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    return dict(prefix_len=i32(b.prefixes * n), prefix_cap=i32(b.caps[:1] * n), prefix_base=torch.tensor(b.bases[:1] * n, dtype=torch.int64, device=DEV))


@pytest.mark.parametrize("n,each,P", [(1024, 1, 6145), (1024, 2, 6145), (300, 3, 27700), (300, 5, 27700)])
def test_chunks_that_the_lists_do_not_hold(n, each, P):
    """Prefixes of few rows (waves) and of more (tiles) with more chunks in all than there are entries stay whole: every key counts once, and
    the rows' bits are those behind the one prefix that all the names mean."""
    of = torch.arange(n * each, dtype=torch.int32, device=DEV) % n
    for shift in (0, 200):
        b = Counted([P], [(1, i % 40, 0) for i in range(n * each)], Hkv=1, shift=shift)
        b.check(0, prefix_of=of, **_behind_one_slab(b, n))
    for t in (b.k, b.v):
        t.copy_(torch.randn(t.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(n)))
    want, _ = b.run(0)
    got, _ = b.run(0, prefix_of=of, **_behind_one_slab(b, n))
    assert got.equal(want) and bool(want.isfinite().all())


def test_chunks_that_the_records_do_not_hold():
    """400 tiles behind 200,000 positions, in 24 chunks each if there were room."""
    b = Counted([200_000], [(16, 3 * i % 70, 0) for i in range(400)], Hkv=1, period=2048, shift=77)
    b.check(0)


def test_an_own_slab_of_more_chunks_than_are_split():
    """A sequence alone of 1.6 million positions of its own: one wave takes them all.  Weights 1, and a value 1 in one of 64 positions of each dim."""
    L, cap = 1_600_001, 1_600_064
    k = torch.zeros(cap * 64, dtype=torch.bfloat16, device=DEV)
    block = torch.empty(64 * 64, dtype=torch.bfloat16)
    kvlayout.scatter(block, 1, 64, "v", torch.eye(64, dtype=torch.bfloat16)[None], torch.arange(64))
    v = block.to(DEV).repeat(cap // 64)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    base = torch.zeros(1, dtype=torch.int64, device=DEV)
    plan = ops.attn_shared_plan(i32(1), i32(L - 1), base, i32(cap), i32(-1), i32(), base[:0], i32(), 1, 0, 1, k.numel())
    q = torch.randn(1, 8, 64, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(DEV)
    got = ops.attn_shared(q, k, v, torch.zeros(8, device=DEV), plan)
    assert plan.status.item() == 0
    n = torch.full((64,), L // 64, dtype=torch.float64)
    n[:L % 64] += 1
    want = n / (L + 1)
    assert bool(((got[0].double().cpu() - want).abs() <= want * 2.0 ** -8).all())
