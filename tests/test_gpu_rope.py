"""ops.rope on the GPU against the rotation in 64 bits.

Tolerance: the reduced angle is rounded by at most 2^-25, sin and cos are evaluated within 2^-23 and their Taylor rest is
2e-9, together under 2^-22; the scaling, two products and the sum add 4 roundings of 2^-24; the output is rounded once
more by half a step of its type."""
import pytest
import torch

from flyai_amd import ops
from flyai_amd.rope import YarnRotary, rope_frequencies

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _turn(x, positions, inv_freq, layout, scaling=1.0, inverse=False):
    """(result, the pair's magnitude at every element) in 64 bits."""
    rot = 2 * inv_freq.numel()
    x = x.double()
    ang = positions.double()[:, None, None] * inv_freq
    c, s = ang.cos() * scaling, ang.sin() * scaling * (-1 if inverse else 1)
    i = torch.arange(rot // 2, device=x.device)
    first, second = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
    out, mag = x.clone(), torch.zeros_like(x)
    u, v = x[..., first], x[..., second]
    out[..., first], out[..., second] = u * c - v * s, v * c + u * s
    mag[..., first] = mag[..., second] = (u.abs() + v.abs()) * abs(scaling)
    return out, mag


def _check(got, x, positions, inv_freq, layout, **kw):
    want, mag = _turn(x, positions, inv_freq, layout, **kw)
    tol = mag * (2.0 ** -22 + 4 * 2.0 ** -24)
    tol = tol + torch.finfo(x.dtype).eps / 2 * (want.abs() + tol)
    tol = tol + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps  # denormal outputs: half of the smallest step
    rot = 2 * inv_freq.numel()
    tol[..., rot:] = 0
    assert got.dtype == x.dtype and got.shape == x.shape
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


def _x(shape, dtype, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.randn(shape, device=DEV, generator=g).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,H,D,rot", [(1, 1, 2, 2), (1, 72, 64, 64), (3, 5, 80, 32), (7, 3, 192, 64), (5, 2, 66, 50),
                                       (33, 1, 64, 24), (2, 3, 256, 130), (130, 9, 128, 128), (3, 1, 2048, 2048),
                                       (1500, 4, 64, 64), (2049, 71, 64, 40)])
def test_rope_matches_64_bits(dtype, layout, T, H, D, rot):
    inv, _ = rope_frequencies(rot, 150000.0)
    pos = torch.randint(-5, 200000, (T,), dtype=torch.int32, device=DEV)
    pos[0] = 0
    x = _x((T, H, D), dtype, T + D)
    for inverse in (False, True):
        _check(ops.rope(x, pos, inv, layout=layout, scaling=1.25, inverse=inverse), x, pos, inv, layout, scaling=1.25,
               inverse=inverse)


def test_rope_far_positions():
    """Every int32 position, the largest ones included."""
    inv, _ = rope_frequencies(64, 10000.0)
    far = [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 2, 10 ** 9 + 7, 2 ** 24 + 1, -10 ** 6, 0, 1]
    pos = torch.tensor(far, dtype=torch.int32, device=DEV)
    x = _x((len(far), 3, 64), torch.float32, 5)
    _check(ops.rope(x, pos, inv), x, pos, inv, "half")


@pytest.mark.parametrize("scaling", [None, "linear", "ntk", "yarn"])
def test_rope_scaled_frequencies(scaling):
    inv, att = rope_frequencies(64, 150000.0, scaling, factor=32.0)
    pos = torch.arange(100000, 100050, dtype=torch.int32, device=DEV)
    x = _x((50, 4, 64), torch.bfloat16, 6)
    _check(ops.rope(x, pos, inv, scaling=att), x, pos, inv, "half", scaling=att)


def test_yarn_frequencies_are_the_stage_tables():
    """The stage's fp32 yarn frequencies are rope_frequencies' within fp32 rounding (a few steps)."""
    inv, att = rope_frequencies(64, 150000.0, "yarn", factor=32.0, device="cpu")
    rot = YarnRotary(16, device="cpu")
    assert torch.allclose(inv, rot.inv_freq.double(), rtol=1e-6, atol=0)
    assert abs(att - rot.attention_scaling) < 1e-12


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_views_in_place_and_inverse(layout):
    """q and k heads inside fused rows: read through strides, written in place, the v heads untouched; then turned back."""
    inv, _ = rope_frequencies(64, 10000.0)
    rows = _x((37, 10, 64), torch.float32, 7)
    before = rows.clone()
    pos = torch.arange(4000, 4037, dtype=torch.int32, device=DEV)
    qk = rows[:, :8]
    assert ops.rope(qk, pos, inv, layout=layout, out=qk) is qk
    _check(qk, before[:, :8], pos, inv, layout)
    assert torch.equal(rows[:, 8:], before[:, 8:])
    back = ops.rope(qk, pos, inv, layout=layout, inverse=True)
    assert float((back - before[:, :8]).abs().max()) < 1e-5
    # heads outermost, and an output that is a view too
    x = _x((4, 21, 64), torch.float32, 8).transpose(0, 1)
    buf = torch.zeros(21, 5, 64, device=DEV)
    ops.rope(x, pos[:21], inv, layout=layout, out=buf[:, 1:])
    _check(buf[:, 1:], x, pos[:21], inv, layout)
    assert not buf[:, 0].any()
    # a start that only the element's own size divides
    odd = _x((21 * 66 + 1,), torch.float32, 9)[1:].view(21, 1, 66)
    _check(ops.rope(odd, pos[:21], inv, layout=layout), odd, pos[:21], inv, layout)


def test_rope_gradient_is_the_inverse():
    """The inverse against differences: sum(g * rope(x)) has the gradient rope(g, inverse)."""
    inv, att = rope_frequencies(32, 10000.0, "yarn", factor=4.0)
    pos = torch.tensor([0, 9, 5000], dtype=torch.int32, device=DEV)
    x, g = _x((3, 2, 48), torch.float32, 10), _x((3, 2, 48), torch.float32, 11)
    grad = ops.rope(g, pos, inv, scaling=att, inverse=True)
    want, mag = _turn(g, pos, inv, "half", scaling=att, inverse=True)
    assert float((grad.double() - want).abs().max()) <= float(mag.max()) * 2.0 ** -21
    d, eps = _x((3, 2, 48), torch.float32, 12), 0.5
    f = lambda t: (g.double() * ops.rope(t, pos, inv, scaling=att).double()).sum()
    diff = (f(x + eps * d) - f(x - eps * d)) / (2 * eps)  # linear in x: the step's size does not matter
    assert abs(float(diff - (grad.double() * d.double()).sum())) < 1e-3


def test_rope_non_finite_values_stay_in_their_pair():
    inv, _ = rope_frequencies(64, 10000.0)
    pos = torch.arange(3, dtype=torch.int32, device=DEV)
    x = _x((3, 2, 80), torch.bfloat16, 13)
    y = ops.rope(x, pos, inv)
    x2 = x.clone()
    x2[1, 0, 5], x2[2, 1, 79] = float("nan"), float("inf")
    y2 = ops.rope(x2, pos, inv)
    hit = torch.zeros_like(y, dtype=torch.bool)
    hit[1, 0, 5] = hit[1, 0, 37] = hit[2, 1, 79] = True
    assert torch.equal(y[~hit], y2[~hit]) and bool(y2[1, 0, [5, 37]].isnan().all()) and bool(y2[2, 1, 79].isinf())


def test_rope_empty_and_other_stream():
    inv, _ = rope_frequencies(64, 10000.0)
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    assert ops.rope(torch.empty(0, 4, 64, device=DEV), none, inv).shape == (0, 4, 64)
    x, pos = _x((64, 8, 64), torch.bfloat16, 14), torch.arange(64, dtype=torch.int32, device=DEV)
    want = ops.rope(x, pos, inv)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.rope(x, pos, inv)
    s.synchronize()
    assert torch.equal(got, want)


def test_rope_captured():
    inv, _ = rope_frequencies(64, 10000.0)
    x, pos = _x((5, 8, 64), torch.bfloat16, 15), torch.arange(5, dtype=torch.int32, device=DEV)
    out = torch.empty_like(x)
    ops.rope(x, pos, inv, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rope(x, pos, inv, out=out)
    for i in range(3):
        x.copy_(_x(x.shape, torch.bfloat16, 20 + i))
        pos.add_(1000)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.rope(x, pos, inv))
