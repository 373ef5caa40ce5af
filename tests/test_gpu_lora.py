"""ops.linear_lora on the GPU against the same sums in 64 bits, row by row.

Tolerance of a row's feature: every fp32 sum is off by at most (its terms) * 2^-24 of the sum of the terms' sizes (bf16
products are exact in fp32), over K terms of the projection, K of h and the rank's of d; h is kept in two bf16 terms, off by
2^-17 of itself; and y is rounded once to bf16 (half a step, 2^-8), a second time with a residual."""
import pytest
import torch

from flyai_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def _inputs(M, K, segments, n, R, seed, ranks=None):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    N, S = sum(segments), len(segments)
    t = lambda shape, s: (torch.randn(shape, device=DEV, generator=g) * s).to(BF16)
    ranks = [max(1, R - 7 * i) if i % 3 else R for i in range(n)] if ranks is None else ranks
    return {"x": t((M, K), 1.0), "w": t((N, K), 0.02), "b": t((N,), 0.05), "lora_a": t((n, S * R, K), 0.02),
            "lora_b": t((n, N, R), 0.05), "scale": torch.rand(n, device=DEV, generator=g) * 2 - 0.5,
            "ranks": torch.tensor(ranks, dtype=torch.int32, device=DEV), "segments": segments}


def _adapters(M, n, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-1, n, (M,), generator=g, dtype=torch.int32).to(DEV)


def _exact(c, adapter, residual=None):
    """(y, tolerance) in 64 bits."""
    x, w = c["x"].double(), c["w"].double()
    n, N, R = c["lora_b"].shape
    K, S = x.shape[1], len(c["segments"])
    y = x @ w.t()
    size = x.abs() @ w.abs().t()
    if c["b"] is not None:
        y, size = y + c["b"].double(), size + c["b"].double().abs()
    tol = size * (K + 16) * 2.0 ** -24
    for t, a in enumerate(adapter.tolist()):
        if not 0 <= a < n:
            continue
        r = min(max(int(c["ranks"][a]), 0), R)
        col = 0
        for s, width in enumerate(c["segments"]):
            A = c["lora_a"][a, s * R:s * R + r].double()
            B = c["lora_b"][a, col:col + width, :r].double()
            sc = c["scale"][a].double()
            h, hs = sc * (A @ x[t]), sc.abs() * (A.abs() @ x[t].abs())
            d, ds = B @ h, B.abs() @ hs
            y[t, col:col + width] += d
            tol[t, col:col + width] += ds * (K + R + 16) * 2.0 ** -24 + (B.abs() @ h.abs()) * 2.0 ** -17
            col += width
    tol = tol + 2.0 ** -8 * (y.abs() + tol)
    if residual is not None:
        y = y + residual.double()
        tol = tol + 2.0 ** -8 * (y.abs() + tol)
    return y, tol


def _check(got, c, adapter, residual=None):
    want, tol = _exact(c, adapter, residual)
    assert got.dtype == BF16 and got.shape == want.shape
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), (float((err - tol).max()), float(err.max()))


def _run(c, adapter, **kw):
    return ops.linear_lora(c["x"], c["w"], c["b"], c["lora_a"], c["lora_b"], c["scale"], c["ranks"], adapter,
                           segments=c["segments"], **kw)


SHAPES = [  # M, K, segments, adapters, R
    (1, 32, (16,), 1, 16),
    (1, 2880, (4096, 512, 512), 3, 16),
    (2, 64, (16, 16, 16, 16), 2, 48),
    (5, 160, (112,), 4, 128),
    (15, 2880, (512,), 1, 32),
    (16, 96, (64, 32), 16, 16),
    (17, 4096, (2880,), 5, 64),
    (48, 2880, (1024, 128, 128), 12, 64),
    (63, 8192, (48,), 3, 32),
    (64, 448, (320,), 2, 80),
    (65, 2880, (512, 64, 64), 7, 32),
    (155, 4096, (2880,), 7, 32),
    (255, 512, (256, 80), 9, 16),
    (256, 512, (256, 80), 9, 16),
    (257, 96, (144, 16), 3, 32),
    (300, 2880, (512, 64, 64), 40, 64),
    (700, 1056, (272,), 2, 112),
    (40, 64, (32,), 70, 16),        # more adapters than a wave's lanes
    (290, 96, (48,), 300, 16),      # more than a workgroup's threads
    (700, 64, (64,), 600, 16),
    (4500, 64, (32, 32), 5, 32),    # more rows than a workgroup lists at once
]


@pytest.mark.parametrize("M,K,segments,n,R", SHAPES)
def test_matches_64_bits(M, K, segments, n, R):
    c = _inputs(M, K, segments, n, R, M + K)
    adapter = _adapters(M, n, M)
    _check(_run(c, adapter), c, adapter)


@pytest.mark.parametrize("M,K,segments,n,R", [
    (1000, 512, (4096, 512, 512), 9, 48),
    (769, 192, (4096, 1008), 40, 128),     # rows and features that end inside a tile
    (960, 64, (5120,), 3, 16),
    (1000, 128, (4096, 960), 2, 64),
    (803, 1088, (5072,), 300, 32),         # an adapter or two a row
    (33000, 64, (16,), 3, 16),             # few features
])
@pytest.mark.parametrize("residual", [False, True])
def test_large_batches(M, K, segments, n, R, residual):
    """Batches of several rounds of tiles, and their rows' bits in a small one."""
    c = _inputs(M, K, segments, n, R, M + n)
    adapter = _adapters(M, n, M)
    res = torch.randn(M, sum(segments), device=DEV).to(BF16) if residual else None
    got = _run(c, adapter, **({"residual": res.clone()} if residual else {}))
    _check(got, c, adapter, res)
    some = torch.arange(3, M, M // 20, device=DEV)
    few = _run(dict(c, x=c["x"][some]), adapter[some], **({"residual": res[some]} if residual else {}))
    assert torch.equal(few, got[some])
    if not residual:
        none = adapter < 0
        assert torch.equal(got[none], ops.linear(c["x"], c["w"], c["b"])[none])


@pytest.mark.parametrize("M", [1, 31, 130, 400])
def test_residual_and_no_bias(M):
    c = _inputs(M, 512, (256, 64), 3, 32, 3)
    c["b"] = None
    adapter = _adapters(M, 3, 4)
    res = torch.randn(M, 320, device=DEV).to(BF16)
    old = res.clone()
    assert _run(c, adapter, residual=res) is res
    _check(res, c, adapter, old)


@pytest.mark.parametrize("M", [7, 100, 333])
def test_rows_by_sequence(M):
    """Adapters of sequences through row_seq: the bits of adapters of rows; a sequence out of range has none."""
    c = _inputs(M, 2880, (512, 64, 64), 4, 32, 5)
    of_seq = torch.tensor([2, -1, 0, 3, 9, 1], dtype=torch.int32, device=DEV)
    seq = torch.arange(M, device=DEV, dtype=torch.int32) * 8 // M - 1          # -1 .. 6
    rows = torch.where((seq >= 0) & (seq < 6), of_seq[seq.clamp(0, 5).long()], -1).to(torch.int32)
    assert torch.equal(_run(c, of_seq, row_seq=seq), _run(c, rows))


@pytest.mark.parametrize("M,n_seqs", [(50, 65), (200, 300), (900, 700)])
def test_many_sequences(M, n_seqs):
    """More sequences than a wave's lanes, a workgroup's threads, and the tiled kernel's: the bits of adapters of rows."""
    c = _inputs(M, 128, (64, 16), 7, 16, 14)
    of_seq = _adapters(n_seqs, 7, 15)
    g = torch.Generator().manual_seed(16)
    seq = torch.randint(0, n_seqs, (M,), generator=g, dtype=torch.int32).to(DEV)
    rows = of_seq[seq.long()].contiguous()
    got = _run(c, of_seq, row_seq=seq)
    assert torch.equal(got, _run(c, rows))
    _check(got, c, rows)


@pytest.mark.parametrize("M", [1, 40, 90, 137, 255, 256, 600])
def test_rows_without_adapter_are_linear(M):
    c = _inputs(M, 2880, (512, 64, 64), 3, 32, 6)
    plain = ops.linear(c["x"], c["w"], c["b"])
    none = torch.full((M,), -1, dtype=torch.int32, device=DEV)
    assert torch.equal(_run(c, none), plain)
    some = none.clone()
    some[::3] = torch.tensor(1, dtype=torch.int32)
    got = _run(c, some)
    keep = some < 0
    assert torch.equal(got[keep], plain[keep])
    zero = dict(c, ranks=torch.zeros_like(c["ranks"]))
    assert torch.equal(_run(zero, some).float(), plain.float())


def test_a_row_depends_on_itself_alone():
    """The same row in batches of every kind of kernel, beside other adapters: the same bits."""
    c = _inputs(600, 2880, (512, 64, 64), 6, 32, 7)
    adapter = _adapters(600, 6, 7)
    adapter[0], adapter[1] = 2, -1
    whole = _run(c, adapter)
    for M in (1, 2, 16, 17, 64, 65, 200, 256, 511):
        part = _run(dict(c, x=c["x"][:M].contiguous()), adapter[:M].contiguous())
        assert torch.equal(part, whole[:M]), M
    perm = torch.randperm(600, device=DEV)
    assert torch.equal(_run(dict(c, x=c["x"][perm].contiguous()), adapter[perm].contiguous()), whole[perm])


@pytest.mark.parametrize("M", [12, 100, 300])
def test_broken_adapters_and_rows_stay_apart(M):
    """NaN and infinities in one adapter, in one row, past a rank and in an adapter that nobody uses reach nobody else."""
    c = _inputs(M, 512, (128, 32), 4, 32, 8, ranks=[32, 9, 16, 32])
    adapter = torch.arange(M, device=DEV, dtype=torch.int32) % 3 - 1   # -1, 0, 1
    want = _run(c, adapter)
    bad = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    bad["lora_a"][0, 3], bad["lora_b"][0, 5] = float("nan"), float("inf")
    bad["lora_a"][2:], bad["lora_b"][2:], bad["scale"][2:] = float("nan"), float("nan"), float("nan")
    bad["lora_a"].view(4, 2, 32, 512)[1, :, 9:] = float("nan")
    bad["lora_b"][1, :, 9:] = float("inf")
    bad["x"][4] = float("nan")
    got = _run(bad, adapter)
    fine = adapter != 0
    fine[4] = False
    assert torch.equal(got[fine], want[fine]) and bool(torch.isfinite(got[fine].float()).all())
    assert bool(got[4].isnan().all()) and bool(got[1, :128].float().isnan().any())


@pytest.mark.parametrize("M,segments", [(300, (64, 64)), (1000, (4096, 1024))])
@pytest.mark.parametrize("one", [False, True])
def test_columns_past_a_rank_reach_nobody(M, segments, one):
    """NaN and infinities past every rank, in tiles of one adapter and of several; then one adapter broken, others whole."""
    c = _inputs(M, 192, segments, 5, 64, 20, ranks=[64, 41, 16, 33, 32])
    adapter = torch.full((M,), 1, dtype=torch.int32, device=DEV) if one else torch.arange(M, device=DEV, dtype=torch.int32) % 6 - 1
    want = _run(c, adapter)
    _check(want, c, adapter)
    for a, r in enumerate(c["ranks"].tolist()):
        c["lora_b"][a, :, r:] = float("nan") if a % 2 else float("inf")
        c["lora_a"].view(5, 2, 64, 192)[a, :, r:] = float("nan")
    assert torch.equal(_run(c, adapter), want)
    c["lora_b"][3], c["lora_a"][3] = float("nan"), float("inf")
    fine = adapter != 3
    assert torch.equal(_run(c, adapter)[fine], want[fine])


def test_large_h_keeps_its_infinity():
    c = _inputs(3, 64, (32,), 1, 16, 9)
    c["scale"][:] = 3e38
    c["x"][:] = 100.0
    c["lora_a"][:] = 1.0
    c["lora_b"][:] = 1.0
    got = _run(c, torch.zeros(3, dtype=torch.int32, device=DEV))
    assert bool((got.float() == float("inf")).all())


@pytest.mark.parametrize("M", [3, 300])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_h_between_the_largest_bf16_and_fp32(M, sign):
    """h of 3.4e38 rounds to an infinite bf16; with B = 1/2 the result is finite."""
    c = _inputs(M, 64, (64,), 1, 16, 19, ranks=[1])
    c["x"][:] = 0
    c["x"][:, 0] = 1
    c["lora_a"][:] = sign
    c["scale"][:] = 3.4e38
    c["lora_b"][:] = 0.5
    adapter = torch.zeros(M, dtype=torch.int32, device=DEV)
    _check(_run(c, adapter), c, adapter)


def test_ranks_out_of_range_are_clamped():
    c = _inputs(20, 160, (64,), 2, 32, 10, ranks=[32, 0])
    adapter = _adapters(20, 2, 10)
    want = _run(c, adapter)
    c["ranks"] = torch.tensor([999, -5], dtype=torch.int32, device=DEV)
    assert torch.equal(_run(c, adapter), want)


def test_empty_batch_other_stream_and_two_at_once():
    c = _inputs(33, 512, (128, 32), 3, 32, 11)
    adapter = _adapters(33, 3, 11)
    empty = _run(dict(c, x=c["x"][:0]), adapter[:0])
    assert empty.shape == (0, 160)
    want = _run(c, adapter)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append([_run(c, adapter) for _ in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for gs in got for g in gs)


@pytest.mark.parametrize("M,segments", [(50, (1024, 64)), (500, (1024, 64)), (1000, (4096, 1024))])
def test_calls_repeat_their_bits(M, segments):
    c = _inputs(M, 2880, segments, 7, 32, 21)
    adapter = _adapters(M, 7, 21)
    want = _run(c, adapter)
    for _ in range(30):
        assert torch.equal(_run(c, adapter), want)


@pytest.mark.parametrize("M", [6, 300])
def test_captured(M):
    """A captured call replays on what its inputs, the adapter of each row among them, hold then."""
    c = _inputs(M, 512, (128, 32), 3, 32, 12)
    adapter = _adapters(M, 3, 12)
    _run(c, adapter)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = _run(c, adapter)
    for i in range(3):
        c["x"].copy_(torch.randn(M, 512, device=DEV).to(BF16))
        adapter.copy_(_adapters(M, 3, 20 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, _run(c, adapter))


def test_unaligned_bias_and_views():
    """A bias that starts anywhere; matrices and rows must start at 16 bytes."""
    c = _inputs(70, 64, (32,), 2, 16, 17)
    adapter = _adapters(70, 2, 17)
    want = _run(c, adapter)
    c["b"] = torch.cat([c["b"][:1], c["b"]])[1:]
    assert c["b"].data_ptr() % 16 and torch.equal(_run(c, adapter), want)
    c["x"] = torch.cat([c["x"].view(-1)[:1], c["x"].view(-1)])[1:].view(70, 64)
    with pytest.raises(RuntimeError, match="aligned"):
        _run(c, adapter)


def test_residual_over_x_is_refused():
    c = _inputs(300, 64, (64,), 2, 16, 18)
    before = c["x"].clone()
    with pytest.raises(RuntimeError, match="overlaps"):
        _run(c, _adapters(300, 2, 18), residual=c["x"])
    torch.cuda.synchronize()
    assert torch.equal(c["x"], before)


def test_refusals():
    c = _inputs(4, 64, (32, 16), 2, 16, 13)
    ad = torch.zeros(4, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        _run(c, ad[:3])
    with pytest.raises(TypeError):
        _run(c, ad.long())
    with pytest.raises(ValueError):
        _run(dict(c, segments=(48,)), ad)                 # lora_a has two segments' rows
    with pytest.raises(RuntimeError, match="segment"):
        _run(dict(c, segments=(40, 8)), ad)
    with pytest.raises(RuntimeError, match="features"):
        _run(dict(c, segments=(16, 16)), ad)
    with pytest.raises(RuntimeError, match="segment"):
        _run(dict(c, segments=(2 ** 32 + 32, 16)), ad)    # not 32
    with pytest.raises(TypeError):
        _run(dict(c, scale=c["scale"].double()), ad)
    with pytest.raises(ValueError):
        _run(dict(c, ranks=c["ranks"].cpu()), ad)
    with pytest.raises(ValueError):
        _run(dict(c, lora_a=c["lora_a"].transpose(1, 2)), ad)
