"""Refusals of the adapters', rotary and slab operators through the C ABI: every one comes back as an error code before
anything is launched, so they run without a GPU (the pointers are never read)."""
import ctypes as C

import numpy as np
import pytest
import torch

from flyai_amd import _lib
from flyai_amd.rope import rope_frequencies

PTR = C.c_void_p(0x100000)
ODD = C.c_void_p(0x100002)


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


def _lora(lib, M=4, N=48, K=64, n=2, R=16, segments=(32, 16), x=PTR, a=PTR, adapter=PTR, row_seq=None, n_seqs=0, y=PTR, ws=PTR):
    return lib.flyai_linear_lora_bf16(x, PTR, None, M, N, K, a, PTR, PTR, PTR, n, R, (C.c_int32 * len(segments))(*segments),
                                      len(segments), adapter, row_seq, n_seqs, y, None, ws, None)


@pytest.mark.parametrize("change", [
    {"M": -1}, {"M": (1 << 19) + 1}, {"N": 40}, {"K": 48}, {"K": 8224}, {"n": 0}, {"R": 8}, {"R": 24}, {"R": 144},
    {"segments": (48, 8)}, {"segments": (24, 24)}, {"segments": (32,)}, {"segments": (16, 16, 16, 16)}, {"segments": (64, -16)},
    {"segments": (2 ** 31 - 16, 2 ** 31 - 16)}, {"segments": (16,) * 5}, {"x": None}, {"x": ODD}, {"a": ODD}, {"a": None}, {"adapter": None},
    {"row_seq": PTR, "n_seqs": 0}, {"y": None}, {"ws": None}, {"ws": ODD}])
def test_lora_refusals(lib, change):
    assert _lora(lib, **change) == _lib.FLYAI_EINVAL
    assert lib.flyai_last_error()


def test_lora_result_over_x(lib):
    """x is read while the result is written: as residual it would be read half updated."""
    for at in (0x100000, 0x100000 + 4 * 64 * 2 - 16, 0x100000 - 4 * 48 * 2 + 16):
        assert _lora(lib, y=C.c_void_p(at)) == _lib.FLYAI_EINVAL
        assert b"overlaps" in lib.flyai_last_error()


def test_lora_of_no_rows(lib):
    assert _lora(lib, M=0) == 0
    assert lib.flyai_linear_lora_workspace_bytes(0, 48, 64, 16, 2) == 0
    small, large = (int(lib.flyai_linear_lora_workspace_bytes(m, 5120, 2880, 64, 3)) for m in (255, 256))
    # below 256 rows the projection leaves one plane of partial sums per 512 of K, from 256 rows one
    assert small >= 255 * (6 * 5120 * 4 + 3 * 64 * 4) and large >= 256 * (5120 * 4 + 3 * 64 * 4)


def _rope(lib, x=PTR, xt=256, xh=64, pos=PTR, T=2, H=4, D=64, rot=64, dtype=0, out=C.c_void_p(0x200000), ot=256, oh=64):
    return lib.flyai_rope(x, xt, xh, pos, PTR, 1.0, T, H, D, rot, dtype, 0, 0, out, ot, oh, None)


@pytest.mark.parametrize("change", [
    {"T": -1}, {"H": 0}, {"rot": 0}, {"rot": 33}, {"rot": 66}, {"dtype": 3}, {"dtype": -1}, {"xt": -256}, {"x": None}, {"pos": None},
    {"out": None}, {"ot": 128}, {"oh": 32}, {"oh": 0}, {"ot": 0}, {"out": C.c_void_p(0x100080)}, {"out": PTR, "ot": 512},
    {"T": (1 << 22) + 1}, {"H": 1 << 17}, {"D": 4096, "rot": 2050, "xh": 4096, "oh": 4096, "xt": 1 << 20, "ot": 1 << 20}])
def test_rope_refusals(lib, change):
    assert _rope(lib, **change) == _lib.FLYAI_EINVAL
    assert lib.flyai_last_error()


def test_rope_of_no_tokens(lib):
    assert _rope(lib, T=0) == 0


def _slab(base, cap):
    return _lib.KvSlab(base, cap, 0)


def _fork(lib, src=(0, 128), dsts=((2 * 128 * 64, 128),), lo=0, hi=10, layer=8 * 128 * 64, elems=8 * 128 * 64, L=2, heads=2, D=64,
          k=PTR, dk=PTR):
    many = (_lib.KvSlab * max(1, len(dsts)))(*[_slab(*d) for d in dsts])
    one = _slab(*src)
    return lib.flyai_kv_fork(k, PTR, layer, elems, dk, PTR, layer, elems, L, heads, D, C.byref(one), many, len(dsts), lo, hi, None)


@pytest.mark.parametrize("change,code", [
    ({"hi": 129}, _lib.FLYAI_ERANGE), ({"dsts": ((2 * 128 * 64, 64),), "hi": 65}, _lib.FLYAI_ERANGE),
    ({"dsts": ((7 * 128 * 64, 128),)}, _lib.FLYAI_ERANGE), ({"src": (7 * 128 * 64, 128)}, _lib.FLYAI_ERANGE),
    ({"dsts": ((64, 128),)}, _lib.FLYAI_EINVAL), ({"dsts": ((4 * 128 * 64, 128), (5 * 128 * 64, 128))}, _lib.FLYAI_EINVAL),
    ({"lo": 11}, _lib.FLYAI_EINVAL), ({"lo": -1}, _lib.FLYAI_EINVAL), ({"src": (0, 100)}, _lib.FLYAI_EINVAL),
    ({"src": (-8, 128)}, _lib.FLYAI_EINVAL), ({"src": (4, 128)}, _lib.FLYAI_EINVAL), ({"D": 128}, _lib.FLYAI_EINVAL),
    ({"L": 0}, _lib.FLYAI_EINVAL), ({"heads": 0}, _lib.FLYAI_EINVAL), ({"k": None}, _lib.FLYAI_EINVAL),
    ({"dk": C.c_void_p(0x100008)}, _lib.FLYAI_EINVAL), ({"layer": 4 * 128 * 64}, _lib.FLYAI_EINVAL)])
def test_fork_refusals(lib, change, code):
    assert _fork(lib, **change) == code
    assert lib.flyai_last_error()


@pytest.mark.parametrize("base", [2 ** 63 - 8, 2 ** 63 - 128 * 128, 2 ** 62])
def test_slabs_at_the_end_of_64_bits(lib, base):
    """A base whose slab would end past 2^63 is past the pool, not before it."""
    assert _fork(lib, src=(base, 128)) == _lib.FLYAI_ERANGE
    assert _fork(lib, dsts=((base, 128),)) == _lib.FLYAI_ERANGE
    assert _compact(lib, [(base, 128, 0, 1)], [1]) == _lib.FLYAI_ERANGE
    assert _compact(lib, [(base, 128, 0, 1)], [0]) == _lib.FLYAI_ERANGE


def test_overlapping_pools(lib):
    """K and V in one place, or a source that lies across the destination's layers: two workgroups would race."""
    slab, L = 2 * 128 * 64, 2
    elems = 8 * 128 * 64

    def fork(src_k, src_v, k, v, src_layer=elems):
        src, dst = _slab(0, 128), _slab(slab, 128)
        return lib.flyai_kv_fork(src_k, src_v, src_layer, elems, k, v, elems, elems, L, 2, 64, C.byref(src), C.byref(dst), 1, 0, 10, None)

    at = lambda layers: 0x100000 + layers * elems * 2                # whole pools of one layer behind each other
    for case in [(at(0), at(2), at(0), at(0)), (at(0), at(2), at(0), at(1)), (at(4), at(6), at(0), at(1)),   # K across V
                 (at(1), at(4), at(0), at(4)), (at(0), at(3), at(0), at(4)), (at(6), at(8), at(0) + 16, at(8)),  # the source across
                 (at(4), at(0), at(0), at(4)), (at(8), at(9), at(0), at(8)), (at(0), at(4), at(0), at(4), 2 * elems)]:
        assert fork(*case) == _lib.FLYAI_EINVAL, case
        assert b"overlap" in lib.flyai_last_error()
    assert _compact(lib, [(0, 128, 0, 1)], [1]) == _lib.FLYAI_EINVAL
    assert b"overlap" in lib.flyai_last_error()


def test_fork_of_nothing(lib):
    assert _fork(lib, lo=10) == 0
    assert _fork(lib, dsts=()) == 0


def _compact(lib, moves, keep, elems=8 * 128 * 64, v=PTR):
    rows = (_lib.KvMove * max(1, len(moves)))(*[_lib.KvMove(b, c, s, n, 0) for b, c, s, n in moves])
    flat = np.asarray(keep, dtype=np.int32)
    return lib.flyai_kv_compact(PTR, v, elems, elems, 2, 2, 64, rows, len(moves), flat.ctypes.data_as(C.c_void_p), None)


@pytest.mark.parametrize("moves,keep,code", [
    ([(0, 128, 100, 2)], [0, 28], _lib.FLYAI_ERANGE), ([(0, 128, 127, 2)], [0, 0], _lib.FLYAI_ERANGE),
    ([(7 * 128 * 64, 128, 0, 1)], [1], _lib.FLYAI_ERANGE), ([(0, 128, 0, 1)], [-1], _lib.FLYAI_EINVAL),
    ([(0, 128, 0, 1)], [2 ** 31 - 1], _lib.FLYAI_ERANGE), ([(0, 128, -1, 1)], [1], _lib.FLYAI_EINVAL),
    ([(0, 128, 0, -1)], [1], _lib.FLYAI_EINVAL), ([(0, 96, 0, 1)], [1], _lib.FLYAI_EINVAL),
    ([(0, 128, 0, 1), (64, 128, 0, 1)], [1, 1], _lib.FLYAI_EINVAL), ([(0, 128, 0, 1), (0, 128, 50, 1)], [1, 1], _lib.FLYAI_EINVAL)])
def test_compact_refusals(lib, moves, keep, code):
    assert _compact(lib, moves, keep) == code
    assert lib.flyai_last_error()


def test_moves_must_ascend(lib):
    for keep in ([1, 0], [4, 4]):
        assert _compact(lib, [(0, 128, 0, 2)], keep) == _lib.FLYAI_EINVAL
        assert b"ascending" in lib.flyai_last_error()


def test_compact_of_nothing(lib):
    assert _compact(lib, [], []) == 0
    assert _compact(lib, [(0, 128, 5, 0)], []) == 0
    assert _compact(lib, [(0, 128, 5, 3)], [0, 1, 2]) == 0           # every row stays
    assert _compact(lib, [], [], v=None) == _lib.FLYAI_EINVAL


def test_adapter_bank_on_the_host():
    """What does not fit changes nothing; parameters under training are read, not tied to the bank."""
    from flyai_amd.lora import AdapterBank
    from flyai_amd.runtime import GptOssShape

    shape = GptOssShape(hidden=64, n_q_heads=8, n_kv_heads=1, head_dim=64)
    bank = AdapterBank(shape, 2, 2, 16, "cpu")
    a, b = torch.nn.Parameter(torch.randn(3, 64)), torch.nn.Parameter(torch.randn(512, 3))
    for _ in range(2):
        bank.load(1, [{"q": (a, b)}, {}], 0.5)
    assert not any(t.requires_grad for t in (bank.qkv_a, bank.qkv_b, bank.scale, bank.ranks))
    assert torch.equal(bank.qkv_a[0, 1, :3], a.detach().bfloat16()) and torch.equal(bank.qkv_b[0, 1, :512, :3], b.detach().bfloat16())
    assert not bool(bank.qkv_a[1].any()) and bank.ranks.tolist() == [0, 3] and bank.scale.tolist() == [0.0, 0.5]
    before = bank.qkv_a.clone()
    for layers, scale in [([{"q": (a.detach().numpy(), b)}, {}], 1.0), ([{"q": (a.detach().long(), b)}, {}], 1.0),
                          ([{"q": (a[0], b)}, {}], 1.0), ([{"q": (a, b)}, {}], "1/16"), ([{"q": (a, b)}], 1.0)]:
        with pytest.raises(ValueError):
            bank.load(1, layers, scale)
        assert torch.equal(bank.qkv_a, before) and bank.ranks.tolist() == [0, 3]


def test_rope_frequencies():
    inv, att = rope_frequencies(64, 10000.0, device="cpu")
    assert att == 1.0 and inv.dtype == torch.float64 and inv.shape == (32,)
    assert inv[0] == 1.0 and abs(float(inv[31]) - 10000.0 ** (-62 / 64)) < 1e-18
    lin, _ = rope_frequencies(64, 10000.0, "linear", factor=8.0, device="cpu")
    assert torch.equal(lin, inv / 8)
    ntk, _ = rope_frequencies(64, 10000.0, "ntk", factor=8.0, device="cpu")
    assert ntk[0] == 1.0 and abs(float(ntk[31] * 8 / inv[31]) - 1) < 1e-12
    yarn, att = rope_frequencies(64, 10000.0, "yarn", factor=8.0, device="cpu")
    assert yarn[0] == inv[0] and abs(float(yarn[31] * 8 / inv[31]) - 1) < 1e-12 and att > 1.2
    for bad in ({"rot_dim": 63}, {"rot_dim": 0}, {"base": 1.0}, {"factor": 0.5}, {"scaling": "other"}, {"original_max": 0},
                {"rot_dim": 2, "scaling": "ntk"}):
        with pytest.raises(ValueError):
            rope_frequencies(**{"rot_dim": 64, "device": "cpu", **bad})
