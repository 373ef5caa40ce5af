"""ops.spec_verify against the oracle: tokens and counts equal, probabilities one fp32 rounding off at most."""
import numpy as np
import pytest
import torch

from flyai_amd import ops
from flyai_amd.sampling import Sampler
from oracle import verify as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
V_GPTOSS = 201088


class Case:
    """Streams of rows; logits with heavy ties, a few likely tokens; drafts near the target."""

    def __init__(self, V, rows, params, seed=0, probs="some", bonus=True):
        rng = np.random.default_rng(seed)
        self.V, self.rows, self.params = V, rows, params
        R = sum(rows)
        x = rng.normal(0, 2, (R, V)).astype(np.float32)
        like = rng.integers(0, V, (R, min(V, 24)))
        np.put_along_axis(x, like, rng.normal(8, 2, like.shape).astype(np.float32), 1)
        self.logits = torch.from_numpy(x).to(torch.bfloat16)
        x = self.logits.float().numpy() + rng.normal(0, 0.5, (R, V))
        p = np.exp(x - x.max(1, keepdims=True))
        self.probs = (p / p.sum(1, keepdims=True)).astype(np.float32)
        self.draft = np.array([rng.choice(V, p=q / q.sum()) for q in self.probs.astype(np.float64)], dtype=np.int32)
        self.cu = np.concatenate(([0], np.cumsum(rows))).astype(np.int32)
        if bonus:
            self.draft[[e - 1 for e, n in zip(self.cu[1:], rows) if n]] = -1
        self.probs_row = np.where(rng.random(R) < {"some": 0.5, "all": 1.0, "none": 0.0}[probs], np.arange(R), -1).astype(np.int32)
        if probs == "none":
            self.probs_row[:] = -1
        self.u, self.u_draw = rng.random(R), rng.random(len(rows))

    def run(self, probs=True, **change):
        t = lambda a, d: torch.tensor(np.asarray(a), dtype=d, device=DEV)  # noqa: E731
        args = dict(logits=self.logits.to(DEV), cu_rows=t(self.cu, torch.int32), draft=t(self.draft, torch.int32), u=t(self.u, torch.float64),
                    u_draw=t(self.u_draw, torch.float64), temp=t([p[0] for p in self.params], torch.float32),
                    top_k=t([p[1] for p in self.params], torch.int32), top_p=t([p[2] for p in self.params], torch.float32))
        if probs and (self.probs_row >= 0).any():
            args.update(draft_probs=torch.from_numpy(self.probs).to(DEV), probs_row=t(self.probs_row, torch.int32))
        args.update(change)
        return ops.spec_verify(**args)

    def expected(self):
        x = self.logits.float().numpy()
        tokens, p, counts = np.full(len(x), -1), np.zeros(len(x)), []
        for s, (k0, k1) in enumerate(zip(self.cu[:-1], self.cu[1:])):
            q = [self.probs[self.probs_row[r]] if self.probs_row[r] >= 0 else None for r in range(k0, k1)]
            t, ps = oracle.stream(x[k0:k1], self.draft[k0:k1], q, *self.params[s], self.u[k0:k1], self.u_draw[s])
            tokens[k0:k0 + len(t)], p[k0:k0 + len(t)] = t, ps
            counts.append(len(t))
        return tokens, np.array(counts), p

    def check(self, **change):
        tokens, counts, p = self.run(**change)
        want, n, wp = self.expected()
        assert counts.tolist() == n.tolist()
        assert tokens.tolist() == want.tolist()
        assert np.all(np.abs(p.cpu().numpy().astype(np.float64) - wp) <= wp * 2.0 ** -23)


PARAMS = [(0.0, 0, 1.0), (1.0, 0, 1.0), (0.7, 0, 0.95), (0.9, 40, 1.0), (1.3, 200, 0.9), (2.0, 0, 0.5), (0.3, 1, 1.0), (1.0, 0, 1e-6)]


@pytest.mark.parametrize("probs", ["none", "some", "all"])
@pytest.mark.parametrize("V", [1, 2, 7, 64, 1000, 4096, 4099, 8200, 12345, 32768])
def test_streams(V, probs):
    rows = [5, 1, 0, 3, 9, 2, 4, 1, 6, 5]
    Case(V, rows, [PARAMS[(i + V) % len(PARAMS)] for i in range(len(rows))], seed=V, probs=probs).check()


@pytest.mark.parametrize("params", PARAMS)
def test_full_vocabulary(params):
    Case(V_GPTOSS, [4, 5, 3], [params] * 3, seed=3).check()


def test_many_streams():
    """More streams than a workgroup has threads, most of one or two rows."""
    rows = [i % 3 for i in range(2500)]
    Case(50, rows, [PARAMS[i % len(PARAMS)] for i in range(2500)], seed=1).check()


def test_long_streams():
    """More rows in a stream than a workgroup has threads, every draft accepted up to the last rows."""
    c = Case(16, [1500, 3], [(1.0, 0, 1.0)] * 2, seed=1, probs="none")
    c.u[:1497] = 0.0
    c.check()


def test_no_bonus_row_and_drafts_that_are_none():
    """A stream that ends with an accepted draft draws nothing; a row without a draft ends its stream wherever it is."""
    c = Case(300, [3, 4, 4, 2], [(1.0, 0, 1.0), (0.8, 0, 0.9), (0.0, 0, 1.0), (1.0, 5, 1.0)], seed=5, probs="some", bonus=False)
    c.u[:3] = 0.0
    c.draft[4], c.draft[12] = -1, 300
    c.draft[7:11] = torch.argmax(c.logits[7:11].float(), 1).numpy()
    c.check()


def test_numbers_for_all_streams():
    c = Case(5000, [3, 4], [(0.8, 50, 0.9)] * 2, seed=2)
    c.check()
    c.check(temp=0.8, top_k=50, top_p=0.9)
    c.check(top_k=50)
    g = Case(5000, [3, 4], [(0.0, 0, 1.0)] * 2, seed=2)
    g.check(temp=0, top_k=0, top_p=1.0)


def test_probs_of_every_row():
    c = Case(3000, [4, 3], [(1.0, 0, 1.0)] * 2, seed=8, probs="all")
    c.check(probs_row=None)


@pytest.mark.parametrize("V", [700, 9001])
def test_special_logits(V):
    """Masked tokens (-inf, the type's lowest value), rows that are masked or equal all over, infinities, NaN, tiny and huge values,
    zeros of both signs."""
    rows = [2] * 14
    for params in ((1.0, 0, 1.0), (0.7, 30, 0.9), (0.0, 0, 1.0)):
        c = Case(V, rows, [params] * 14, seed=V)
        x = c.logits
        low = torch.finfo(torch.bfloat16).min
        x[0, 1:], x[1, ::2] = float("-inf"), float("-inf")
        x[2, 5:], x[3, ::3] = low, low
        x[4], x[5] = float("-inf"), low
        x[6], x[7] = 0.0, 3.0
        x[8, 17], x[9, 3] = float("inf"), -float("inf")
        x[10, 5], x[11, 6] = float("nan"), float("nan")
        x[12] *= 2.0 ** -60
        x[13] *= 2.0 ** 40
        x[14] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0)
        x[15] *= 2.0 ** -130
        x[16, 9], x[17, 9] = 1e38, 70000.0
        x[18] = -x[18].abs() - 2.0 ** 30
        x[19, :600] = 2.0 ** -50
        with np.errstate(invalid="ignore", over="ignore"):
            c.check()


@pytest.mark.parametrize("temp", [1e-9, 1e-6, 1e-3, 30.0, 1e6, 1e20, 1e38])
def test_temperatures(temp):
    with np.errstate(invalid="ignore", over="ignore"):
        Case(3001, [3, 3, 2], [(temp, 0, 1.0), (temp, 9, 1.0), (temp, 0, 0.7)], seed=4).check()


def test_equal_logits_over_the_whole_vocabulary():
    """More equal values than 16 bits count: a draw anywhere, top-k keeps all of them, top-p a part."""
    c = Case(V_GPTOSS, [1, 1, 1, 2], [(1.0, 0, 1.0), (1.0, 5, 1.0), (1.0, 0, 0.37), (1.0, 0, 0.5)], seed=6, probs="none")
    c.logits[:] = 1.5
    c.draft[3] = V_GPTOSS // 2 + 7  # behind the last tie that is kept
    c.check()
    c.draft[3] = 5
    c.check()


def test_uniforms_at_their_ends():
    for u in (0.0, 1 - 2.0 ** -53, 1.0, 2.0, -1.0, float("nan")):
        c = Case(999, [2, 2, 3], [(1.0, 0, 1.0), (0.7, 0, 0.8), (1.0, 3, 1.0)], seed=7)
        c.u[:], c.u_draw[:] = u, u
        c.check()


def test_distributions_of_any_kind():
    """q equal to p, larger than one, zero, negative, infinite and NaN entries, all the mass on one token."""
    c = Case(64, [2] * 8, [(1.0, 0, 1.0)] * 8, seed=11, probs="all")
    x = c.logits.float().numpy().astype(np.float64)
    p = np.exp(x - x.max(1, keepdims=True))
    c.probs[:] = p / p.sum(1, keepdims=True)
    c.u[:] = 1 - 2.0 ** -53
    c.probs[2] = 3.0
    c.probs[4] = 0.0
    c.probs[6, ::2] = -1.0
    c.probs[8] = np.inf
    c.probs[10, :60] = np.nan
    c.draft[10] = 62
    c.probs[12], c.probs[12, c.draft[12]] = 0.0, 1.0
    c.probs_row[14] = 16  # outside the rows of q: none
    with np.errstate(invalid="ignore"):
        tokens, counts, pr = c.run()
        c.probs_row[14] = -1
        want, n, wp = c.expected()
    assert tokens.tolist() == want.tolist() and counts.tolist() == n.tolist()


def test_the_samplers_draws():
    """Without distributions the accepted prefix and the draw are those of sample_rows."""
    c = Case(20000, [4, 4, 4], [(0.8, 100, 0.95)] * 3, seed=13, probs="none")
    tokens, counts, p = c.run()
    R = len(c.draft)
    seq = np.repeat(np.arange(3), 4)
    t = lambda a, d: torch.tensor(a, dtype=d, device=DEV)  # noqa: E731
    got = ops.sample_rows(c.logits.to(DEV), 0.8, 100, 0.95, draft=t(c.draft, torch.int32), u=t(c.u_draw[seq], torch.float64),
                          want_p_draft=True, want_draw=True)
    for s in range(3):
        for i in range(counts[s]):
            r = 4 * s + i
            last = i == counts[s] - 1
            if last:
                assert tokens[r] == got["draw"][r]
            else:
                assert tokens[r] == c.draft[r] and p[r] == got["p_draft"][r]
    assert R == 12


def test_rows_behind_the_last_stream():
    c = Case(500, [2, 3], [(1.0, 0, 1.0)] * 2, seed=3, probs="none")
    whole = c.run()
    cu = torch.tensor([0, 2], dtype=torch.int32, device=DEV)
    one = ops.spec_verify(c.logits.to(DEV), cu, torch.tensor(c.draft, device=DEV), torch.tensor(c.u, device=DEV),
                          torch.tensor(c.u_draw[:1], device=DEV), 1.0)
    assert one[1].tolist() == whole[1][:1].tolist() and one[0][:2].equal(whole[0][:2])


def test_malformed_rows_stay_in_bounds():
    """cu_rows past the rows, descending or negative: no row outside the batch is touched, and the call ends."""
    c = Case(500, [2, 3], [(1.0, 0, 1.0)] * 2, seed=3, probs="none")
    for cu in ([0, 2, 99], [3, 1, 5], [-7, 2, 5], [5, 5, 5], [2 ** 31 - 1, -2 ** 31, 4]):
        tokens, counts, p = c.run(cu_rows=torch.tensor(cu, dtype=torch.int32, device=DEV))
        assert int(counts.min()) >= 0 and int(counts.max()) <= 5


def test_lossless():
    """The first token of 200,000 streams is distributed as the target, whatever the drafter: each frequency within five deviations."""
    V, n = 20, 200000
    rng = np.random.default_rng(0)
    x = torch.tensor(rng.normal(0, 1.5, V), dtype=torch.bfloat16)
    p = torch.softmax(x.double(), 0).numpy()
    q = rng.dirichlet(np.ones(V)).astype(np.float32)
    for lookup in (False, True):
        draft = np.full(n, 7) if lookup else rng.choice(V, n, p=q / q.sum(dtype=np.float64))
        total = np.zeros(V)
        for part in np.array_split(draft, 4):
            m = len(part)
            t = lambda a, d: torch.tensor(a, dtype=d, device=DEV)  # noqa: E731
            kw = {} if lookup else dict(draft_probs=t(q[None], torch.float32), probs_row=torch.zeros(m, dtype=torch.int32, device=DEV))
            tokens, counts, _ = ops.spec_verify(x.to(DEV).expand(m, V).contiguous(), torch.arange(m + 1, dtype=torch.int32, device=DEV),
                                                t(part, torch.int32), t(rng.random(m), torch.float64), t(rng.random(m), torch.float64), 1.0, **kw)
            assert bool((counts == 1).all())
            total += np.bincount(tokens.cpu().numpy(), minlength=V)
        assert np.all(np.abs(total - n * p) <= 5 * np.sqrt(n * p * (1 - p))), (total / n - p)


def test_captured_and_replayed():
    c = Case(30000, [5, 3, 4], [(1.0, 0, 1.0), (0.7, 0, 0.9), (0.0, 0, 1.0)], seed=9)
    args = dict(logits=c.logits.to(DEV), u=torch.tensor(c.u, device=DEV))
    c.run(**args)
    torch.cuda.synchronize()
    t = lambda a, d: torch.tensor(np.asarray(a), dtype=d, device=DEV)  # noqa: E731
    kw = dict(cu_rows=t(c.cu, torch.int32), draft=t(c.draft, torch.int32), u_draw=t(c.u_draw, torch.float64),
              temp=t([p[0] for p in c.params], torch.float32), top_k=t([p[1] for p in c.params], torch.int32),
              top_p=t([p[2] for p in c.params], torch.float32), draft_probs=torch.from_numpy(c.probs).to(DEV), probs_row=t(c.probs_row, torch.int32))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.spec_verify(**args, **kw)
    for i in range(4):
        args["u"].copy_(torch.rand(len(c.u), dtype=torch.float64))
        args["logits"].copy_(args["logits"].roll(i, 1))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, ops.spec_verify(**args, **kw)):
            assert got.equal(want)


def test_refusals():
    c = Case(100, [2, 2], [(1.0, 0, 1.0)] * 2, seed=1)
    n = len(c.draft)
    for change, error in ((dict(top_k=-1), ops._lib.FlyaiError), (dict(draft=torch.zeros(n + 1, dtype=torch.int32, device=DEV)), ValueError),
                          (dict(logits=c.logits.float().to(DEV)), TypeError), (dict(u=torch.rand(n, device=DEV)), TypeError),
                          (dict(temp=torch.ones(3, device=DEV)), ValueError), (dict(logits=c.logits), ValueError),
                          (dict(draft_probs=torch.zeros(3, 100, device=DEV), probs_row=None), ValueError),
                          (dict(draft_probs=None), ValueError),
                          (dict(draft_probs=torch.zeros(n, 99, device=DEV)), ValueError)):
        with pytest.raises(error):
            c.run(**change)


@pytest.mark.parametrize("temp,top_k,top_p", [(0.0, 0, 1.0), (0.8, 0, 0.9), (1.0, 50, 1.0)])
@pytest.mark.parametrize("probs", ["none", "all"])
def test_sampler_accept_batch(temp, top_k, top_p, probs):
    """Sampler.accept_batch: the oracle's tokens for the uniforms that the sampler's generator gives; greedy, accept's."""
    drafts = [3, 0, 5, 1]
    c = Case(1000, [n + 1 for n in drafts], [(temp, top_k, np.float32(top_p))] * 4, seed=11, probs=probs)
    rows = [r for r in range(len(c.draft)) if c.draft[r] >= 0]
    lists = [[int(c.draft[r]) for r in range(a, e - 1)] for a, e in zip(c.cu[:-1], c.cu[1:])]
    c.probs_row[[e - 1 for e in c.cu[1:]]] = -1
    gen = np.random.Generator(np.random.PCG64(5))
    c.u, c.u_draw = gen.random(len(c.u)), gen.random(4)
    sm = Sampler(temp=temp, top_p=top_p, top_k=top_k, seed=5, device=DEV)
    got = sm.accept_batch(c.logits.to(DEV), lists, probs=torch.from_numpy(c.probs[rows]).to(DEV) if probs == "all" else None)
    want, counts, _ = c.expected()
    assert got == [want[a:a + n].tolist() for a, n in zip(c.cu, counts)]
    if temp == 0:
        assert got == [sm.accept(c.logits[a:e].to(DEV), d)[:len(g)] for a, e, d, g in zip(c.cu[:-1], c.cu[1:], lists, got)]
    assert sm.accept_batch(c.logits[:0].to(DEV), []) == []
    with pytest.raises(ValueError):
        sm.accept_batch(c.logits.to(DEV), lists[:-1])
    with pytest.raises(ValueError):
        sm.accept_batch(c.logits.to(DEV), [[1000, 0, 0], *lists[1:]])


@pytest.mark.parametrize("value", [0.0, 1.5])
@pytest.mark.parametrize("V", [5000, 20003])
def test_drafts_that_are_ties_at_the_border(V, value):
    """Half of the ids share the border's value (as +0 and -0 too): a draft among them is kept by its rank in id order."""
    c = Case(V, [2] * 12, [(1.0, 0, np.float32(0.5))] * 12, seed=3, probs="none")
    rng = np.random.default_rng(V)
    x = np.full(c.logits.shape, -1.0, dtype=np.float32)
    ties = np.sort(rng.permutation(V)[:V // 2])
    x[:, ties] = np.where(rng.random(len(ties)) < 0.5, value, -value if value == 0 else value)
    c.logits = torch.from_numpy(x).to(torch.bfloat16)
    w = np.float64(V // 2) + (V - V // 2) * np.exp(-1.0 - value)
    keep = int(0.5 * w)  # about: the ids around the last that is kept
    c.draft[::2] = ties[[0, 1, 7, keep // 2, *range(keep - 4, keep + 4)]]
    c.u[:] = 0.0
    c.check()
    assert 0 < len(set(c.expected()[1].tolist())) <= 2


@pytest.mark.parametrize("streams", [6, 90])
@pytest.mark.parametrize("value", [-float("inf"), float(torch.finfo(torch.bfloat16).min), -100.0, 0.0, -1e-30])
@pytest.mark.parametrize("share", [0.7, 0.9995])
def test_masked_ids(value, share, streams):
    """Most ids masked, by several values: batches of fewer rows than CUs and of more."""
    params = [(1.0, 0, 1.0), (0.7, 0, np.float32(0.95)), (1.0, 30, 1.0)] * (streams // 3)
    c = Case(5003, [3] * streams, params, seed=streams)
    m = torch.rand(c.logits.shape, generator=torch.Generator().manual_seed(1)) < share
    m[:, 7] = False
    c.logits[m] = value
    c.check()


def test_a_table_without_rows():
    """draft_probs of no rows, and probs_row that names none: drafts without a distribution."""
    c = Case(3000, [4, 2], [(0.8, 0, np.float32(0.9))] * 2, seed=8, probs="none")
    c.check(draft_probs=torch.empty(0, 3000, device=DEV), probs_row=torch.full((6,), -1, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("V", [1, 3, 65, 513, 5003])
def test_nothing_is_left(V):
    """A distribution that leaves no weight, for more streams than CUs: every stream draws the first id of maximal weight, with the
    maximum alone and shared, with filters and without."""
    S = 600
    c = Case(V, [2] * S, [PARAMS[1 + i % (len(PARAMS) - 1)] for i in range(S)], seed=V, probs="none")
    c.logits[::4] = torch.where(torch.arange(V) % 5 == 2, 9.0, c.logits[::4].float()).to(torch.bfloat16)
    c.probs = np.full((1, V), 3.0, dtype=np.float32)
    c.probs_row[:] = 0
    c.u[:] = 0.9
    tokens, counts, _ = c.expected()
    assert counts.tolist() == [1] * S and (V < 4 or len(set(tokens[::2].tolist())) > 2)
    c.check()


@pytest.mark.parametrize("probs", ["none", "some"])
@pytest.mark.parametrize("V,streams", [(16400, 300), (40003, 260), (V_GPTOSS, 24)])
def test_weights_by_table(V, streams, probs):
    """Streams without a filter that have enough ids a workgroup for a table of the common values' weights (on any number of CUs up to
    256 here), and rows longer than their first loads: masked ids of several values, values below and above the table's, zeros of both signs,
    the rejected draft among them, ties of the maximum; greedy and filtered streams between them."""
    params = [(1.0, 0, 1.0), (30.0, 0, 1.0), (0.7, 0, 1.0), (1.0, 0, 1.0), (0.0, 0, 1.0), (0.8, 40, np.float32(0.95))]
    c = Case(V, [1 + i % 2 for i in range(streams)], [params[i % len(params)] for i in range(streams)], seed=V, probs=probs)
    R, g = len(c.draft), torch.Generator().manual_seed(V)
    x = c.logits.float()
    low = float(torch.finfo(torch.bfloat16).min)
    some = lambda share: torch.rand(V, generator=g) < share  # noqa: E731
    for r in range(R):
        x[r, some(0.5)] = (float("-inf"), low, -100.0, -300.0, 0.0, 1.0)[r % 6]
        for value in (2.0 ** -30, -2.0 ** -30, 0.0, -0.0, 2.0 ** -24, -2.0 ** -25, -255.0, -256.0, -float("inf")):
            x[r, some(0.002)] = value
        if r % 3 == 0:  # a maximum above the table, more than once
            x[r, some(3.0 / V)] = 300.0
        x[r, 7 + r % 3] = 290.0 if r % 5 == 0 else 12.0
    c.logits = x.to(torch.bfloat16)
    top = torch.argmax(c.logits.float(), 1).numpy()
    c.draft = np.where((c.draft >= 0) & (np.arange(R) % 4 == 1), top, c.draft).astype(np.int32)  # a draft that has most of the weight
    c.u[1::2] = 1 - 2.0 ** -53
    with np.errstate(invalid="ignore", over="ignore"):
        tokens, counts, _ = c.expected()
        assert {1, 2} == set(counts.tolist()) and len(set(tokens.tolist())) > streams // 2
        c.check()
