"""ops.pack_shared and ops.attn_shared against the oracle: sequences behind shared prefixes."""
import pytest
import torch

from flyai_amd import ops
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
