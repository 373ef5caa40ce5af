"""Edges of the operators that serve many requests, on the GPU."""
import math
from fractions import Fraction

import pytest
import torch

from flyai_amd import ops
from flyai_amd.lora import AdapterBank
from flyai_amd.rope import YarnRotary
from flyai_amd.runtime import KVWorkspace, RaggedStage
from flyai_amd.serving import GptOssModel
from flyai_amd.weights import GptOssShape, synthetic_layer

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def _two_pi(bits):
    """2 pi as a Fraction, good to 2^-bits: pi = 16 atan(1/5) - 4 atan(1/239) in integers."""
    one = 1 << (bits + 16)

    def atan_inverse(n):
        total, term, k = 0, one // n, 1
        while term:
            total += term // k if k % 4 == 1 else -(term // k)
            term //= n * n
            k += 2
        return total

    return 2 * Fraction(16 * atan_inverse(5) - 4 * atan_inverse(239), one)


def _exact_cos_sin(position, frequency, two_pi):
    """cos and sin of position * frequency, the product and its remainder by 2 pi exact: off by the 2^-51 or so of a double's
    remainder and its cos and sin."""
    angle = Fraction(position) * Fraction(frequency)
    rest = float(angle - round(angle / two_pi) * two_pi)
    return math.cos(rest), math.sin(rest)


def test_rope_angles_are_exact_at_far_positions():
    """cos and sin of the exact angle, read off the pair (1, 0), at frequencies and positions where the product's own rounding to 64
    bits is up to 2^-23.

    Tolerance, in units of u = 2^-25 (half an fp32 step in [0.5, 1)): the reduced angle's rounding u, times at most 0.88 in sin and
    0.71 in cos; the last fma's rounding u; in cos the rounding of z = r^2 under 0.62, u / 2 of the result, and its polynomial's,
    u / 2 times 0.62; in sin that of r^3's polynomial, u / 4 times 0.49 and what r z < 0.49 loses, u / 2 / 6.  The Taylor rest
    is 2e-9 = 0.07 u.  Below 2.6 u; 3 u is asked for."""
    g = torch.Generator().manual_seed(3)
    freq = torch.rand(64, generator=g, dtype=torch.float64) * 0.5 + 0.5
    pos = torch.randint(2 ** 31 - 10 ** 6, 2 ** 31, (24,), generator=g, dtype=torch.int64)
    pos[:4] = torch.tensor([2 ** 31 - 1, -2 ** 31, 2 ** 30 + 1, 10 ** 9 + 7])
    two_pi = _two_pi(160)
    want = torch.tensor([[_exact_cos_sin(int(p), float(f), two_pi) for f in freq] for p in pos], dtype=torch.float64)
    x = torch.zeros(len(pos), 1, 128, device=DEV)
    x[..., 0::2] = 1.0
    y = ops.rope(x, pos.to(torch.int32).to(DEV), freq.to(DEV), layout="interleaved").double().cpu()
    err = (y.view(len(pos), 64, 2) - want).abs()
    assert float(err.max()) <= 3 * 2.0 ** -25, float(err.max()) * 2 ** 25


@pytest.mark.parametrize("M,K,segments", [(1, 64, (32,)), (70, 64, (32,)), (300, 128, (192, 64)), (300, 96, (48, 16)),
                                          (1000, 128, (4096, 960))])   # the last: tiles of 192 rows
@pytest.mark.parametrize("residual", [False, True])
def test_a_bias_that_starts_anywhere(M, K, segments, residual):
    """Every kernel that adds the bias reads it at any 2-byte start: the bits of an aligned one."""
    g = torch.Generator(device=DEV)
    g.manual_seed(M + K)
    t = lambda *shape: torch.randn(shape, device=DEV, generator=g).to(BF16)
    N, S, n, R = sum(segments), len(segments), 2, 16
    x, w, b, la, lb, old = t(M, K), t(N, K), t(N), t(n, S * R, K), t(n, N, R), t(M, N)
    scale, ranks = torch.ones(n, device=DEV), torch.tensor([16, 9], dtype=torch.int32, device=DEV)
    adapter = (torch.arange(M, device=DEV) % 3 - 1).to(torch.int32)
    run = lambda bias: ops.linear_lora(x, w, bias, la, lb, scale, ranks, adapter, segments=segments,
                                       residual=old.clone() if residual else None)
    want = run(b)
    for off in (1, 2, 3):
        odd = torch.cat([b[:off], b])[off:]
        assert odd.data_ptr() % 16 == 2 * off and torch.equal(run(odd), want), off


def _adapter(shape, n_layers, r, seed, size):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    t = lambda *s: (torch.randn(*s, device=DEV, generator=g) * size).to(BF16)
    H, nq, nkv = shape.hidden, shape.n_q_heads * shape.head_dim, shape.n_kv_heads * shape.head_dim
    return [{"q": (t(r, H), t(nq, r)), "k": (t(r, H), t(nkv, r)), "v": (t(r, H), t(nkv, r)), "o": (t(r, nq), t(H, r))}
            for _ in range(n_layers)]


def _served(with_bank):
    shape = GptOssShape(n_experts=8)
    layers = [synthetic_layer(shape, 70 + i, DEV, sliding=(i == 0)) for i in range(2)]
    g = torch.Generator(device=DEV)
    g.manual_seed(7)
    t = lambda *s: torch.randn(*s, device=DEV, generator=g)
    embed, norm_w, lm = t(1024, shape.hidden).to(BF16), 1.0 + 0.1 * t(shape.hidden), (0.02 * t(1024, shape.hidden)).to(BF16)
    bank = None
    if with_bank:
        bank = AdapterBank(shape, 2, 3, 16, DEV)
        bank.load(0, _adapter(shape, 2, 16, 1, 0.1), 2.0)
        bank.load(2, _adapter(shape, 2, 5, 2, 0.1), 1.0)
    return GptOssModel(shape, layers, embed, norm_w, lm, YarnRotary(256, device=DEV), 4, 256, 64, DEV, lora=bank)


def test_a_served_model_takes_adapters_by_request():
    """GptOssModel.step(adapters=): four requests greedily continued in one batch commit what each commits alone with its own
    adapter; None and -1 are a model without a bank."""
    model, plain = _served(True), _served(False)
    prompts = [[3, 1, 4, 1, 5], [9, 2, 6], [5, 3, 5, 8, 9, 7, 9], [9, 2, 6]]

    def serve(m, which, ads, steps=6):
        chunks, starts, out = [prompts[i] for i in which], [0] * len(which), [[] for _ in which]
        for _ in range(steps):
            toks = m.step(chunks, starts, which, [True] * len(which), ads)
            starts = [s + len(c) for s, c in zip(starts, chunks)]
            chunks = [[t] for t in toks]
            for o, t in zip(out, toks):
                o.append(t)
        return out

    ads = [0, None, 2, 0]
    together = serve(model, [0, 1, 2, 3], ads)
    for i in range(4):
        assert serve(model, [i], [ads[i]]) == [together[i]], i
    without = serve(plain, [0, 1, 2, 3], None)
    assert serve(model, [0, 1, 2, 3], [None, -1, -1, None]) == serve(model, [0, 1, 2, 3], None) == without
    assert together[1] == without[1] and together[0] != without[0] and together[1] != together[3]
    with pytest.raises(RuntimeError, match="outside"):
        model.step([[1]], [0], [0], [True], [3])
    with pytest.raises(RuntimeError, match="has none"):
        plain.step([[1]], [0], [0], [True], [0])


def test_a_bank_bound_anew_between_steps_on_a_side_stream():
    """Steps on a stream of their own, the bank replaced between them from the default stream: each step has its own bank's
    result."""
    shape = GptOssShape(n_experts=8)
    layers = [synthetic_layer(shape, 80, DEV, sliding=False)]
    kv = KVWorkspace(1, 1, 256, shape.n_kv_heads, shape.head_dim, DEV)
    st = RaggedStage(shape, layers, YarnRotary(256, device=DEV), kv, max_tokens=64, max_seqs=1)
    banks = []
    for i in range(2):
        banks.append(AdapterBank(shape, 1, 1, 16, DEV))
        banks[-1].load(0, _adapter(shape, 1, 16, 3 + i, 0.05), 1.0)
    rows = torch.randn(40, shape.hidden, device=DEV).to(BF16)
    want = []
    for b in banks:
        st.set_lora(b)
        want.append(st.forward(rows.clone(), [40], [0], [0], [0]))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for i in (0, 1, 0, 1):
        st.set_lora(banks[i])
        h = rows.clone()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            st.forward(h, [40], [0], [0], [0])
        h.record_stream(side)
        side_result = h
        st.set_lora(banks[1 - i])                                    # drops the workspace of the step just queued
        torch.empty(1 << 20, dtype=torch.uint8, device=DEV).fill_(255)
        side.synchronize()
        assert torch.equal(side_result, want[i]), i
