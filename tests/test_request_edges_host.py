"""Edges of the calls that serve many requests, on the host: what a C argument would take modulo 2^32, and what is refused
before a launch.  The stage is bound to addresses that are never read; a call that passes every check stops at the unset
workspace."""
import ctypes as C
import weakref
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from flyai_amd import _lib, ops
from flyai_amd._lib import ContextOverflow, FlyaiError
from flyai_amd.runtime import KVWorkspace, RaggedStage

FAKE = 0x100000
HIDDEN, CAP = 64, 128


@pytest.fixture
def stage(monkeypatch):
    """A RaggedStage of one layer with a bank of two adapters, and no workspace."""
    lib = _lib.lib()
    cfg = _lib.StageConfig(n_layers=1, hidden=HIDDEN, n_q_heads=8, n_kv_heads=1, head_dim=64, n_experts=4, top_k=2, intermediate=64,
                           window=128, max_tokens=64, max_seqs=4, max_attn_items=64, rope_positions=4096, attn_split_keys=1024,
                           rms_eps=1e-5, attn_prefill_min=32)
    h = C.c_void_p()
    assert lib.flyai_stage_create(C.byref(cfg), C.byref(h)) == 0
    kv = KVWorkspace(1, 2, CAP, 1, 64, "cpu")
    names = ("ln1", "ln2", "wqkv", "bqkv", "wo", "bo", "sinks", "router_w", "router_b", "w13_packed", "b13", "w2_packed", "b2",
             "k_pool", "v_pool")
    d = _lib.LayerDesc(**{f: FAKE for f in names}, sliding=0, pad=0, kv_pool_elems=kv.k[0].numel())
    assert lib.flyai_stage_set_layer(h, 0, C.byref(d)) == 0
    rows = (_lib.LoraLayer * 1)(_lib.LoraLayer(FAKE, FAKE, FAKE, FAKE))
    bank = _lib.StageLora(2, 16, FAKE, FAKE, rows, FAKE, int(lib.flyai_stage_lora_workspace_bytes(h, 16)))
    assert lib.flyai_stage_set_lora(h, C.byref(bank)) == 0
    st = object.__new__(RaggedStage)
    st.__dict__.update(_h=h, _destroy=lib.flyai_stage_destroy, _sync=lambda d: None, device=torch.device("cpu"), kv=kv,
                       shape=SimpleNamespace(hidden=HIDDEN))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: SimpleNamespace(cuda_stream=None))
    return st


def _tree(st, start=3, **kw):
    return st.forward_tree(torch.zeros(2, HIDDEN, dtype=torch.bfloat16), start, [-1, 0], [0, 1], 0, **kw)


def test_adapter_ids_past_32_bits(stage):
    """An id is the bank's or refused: taken modulo 2^32, 2^32 would be adapter 0 and 2^32 - 1 none."""
    for good in (None, -1, 0, 1):
        with pytest.raises(FlyaiError, match="workspace not set"):
            _tree(stage, adapter=good)
    for bad in (2, -2, 2 ** 31, 2 ** 32 - 1, 2 ** 32, 2 ** 32 + 1, -2 ** 32, -2 ** 32 - 1, 2 ** 64):
        with pytest.raises(FlyaiError, match="outside"):
            _tree(stage, adapter=bad)


def test_starts_past_32_bits(stage):
    """A position past the context overflows it: taken modulo 2^32, 2^32 would write K/V over the first positions."""
    with pytest.raises(FlyaiError, match="workspace not set"):
        _tree(stage, CAP - 2)
    rows = torch.zeros(2, HIDDEN, dtype=torch.bfloat16)
    step = lambda starts: stage.forward(rows, [1, 1], starts, [0, 1])
    with pytest.raises(FlyaiError, match="workspace not set"):
        step(np.array([CAP - 1, 0]))
    for far in (CAP, 2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 62):
        with pytest.raises(ContextOverflow):
            _tree(stage, far)
        with pytest.raises(ContextOverflow):
            step(np.array([0, far]))
    for below in (-1, -2 ** 32, -2 ** 32 + 3):
        with pytest.raises(FlyaiError, match="start"):
            _tree(stage, below)
        with pytest.raises(FlyaiError, match="start"):
            step(np.array([0, below]))


def test_rebinding_waits_for_running_steps(stage, monkeypatch):
    """A step on another stream may still use the adapters' workspace, the bank or the stage's workspace when they are bound anew:
    the device is waited for while the old ones are held, and before the next step may use the new one's memory."""
    from flyai_amd import runtime
    from flyai_amd.lora import AdapterBank
    from flyai_amd.weights import GptOssShape

    stage.shape = GptOssShape(hidden=HIDDEN, n_q_heads=8, n_kv_heads=1, head_dim=64)
    stage.layers, stage.workspace, stage.lora, stage._lora_ws = [None], torch.empty(1), None, None
    bank = lambda: AdapterBank(stage.shape, 1, 2, 16, "cpu")
    waits = []
    for new in (bank(), bank(), None):
        old = weakref.ref(stage._lora_ws) if stage._lora_ws is not None else lambda: True
        old_bank = weakref.ref(stage.lora) if stage.lora is not None else lambda: True
        stage._sync = lambda d: waits.append(old() is not None and old_bank() is not None)
        stage.set_lora(new)
        assert waits and all(waits) and (stage._lora_ws is None) == (new is None) and stage.lora is new
        del new
        waits.clear()
    # the stage's own workspace (the C call needs a device: here it only says how large)
    monkeypatch.setattr(runtime, "lib", lambda: SimpleNamespace(flyai_stage_workspace_bytes=lambda h: 512,
                                                                flyai_stage_set_workspace=lambda *a: 0))
    stage.staging, old = torch.empty(8), weakref.ref(stage.workspace)
    stage._sync = lambda d: waits.append(old() is not None)
    stage.set_workspace()
    assert waits and all(waits) and old() is None


@pytest.mark.parametrize("change", [{"hidden": 96}, {"hidden": 32}, {"head_dim": 32}, {"head_dim": 128}])
def test_stages_are_of_whole_tiles(change):
    """What a step with adapters rests on from 256 rows on: K and the q, k and v segments in multiples of 64, one plane of sums."""
    sizes = dict(n_layers=1, hidden=HIDDEN, n_q_heads=8, n_kv_heads=1, head_dim=64, n_experts=4, top_k=2, intermediate=64, window=128,
                 max_tokens=300, max_seqs=4, max_attn_items=64, rope_positions=4096, attn_split_keys=1024, rms_eps=1e-5,
                 attn_prefill_min=32)
    cfg, h = _lib.StageConfig(**{**sizes, **change}), C.c_void_p()
    assert _lib.lib().flyai_stage_create(C.byref(cfg), C.byref(h)) == _lib.FLYAI_EINVAL and not h


def test_lora_workspace_has_no_plane_that_no_kernel_writes():
    """One segment and K % 64 == 0: from 256 rows on the tiled kernel ends the projection, and h is all that is kept."""
    size = lambda *a: int(_lib.lib().flyai_linear_lora_workspace_bytes(*a))
    for M, N, K, R in ((256, 2880, 4096, 64), (2096, 2880, 4096, 16), (1 << 19, 5120, 2880, 128)):
        h = M * ((R + 31) // 32 * 32) * 4 + M * 8                # two bf16 terms a column; adapter and rank
        assert h <= size(M, N, K, R, 1) <= h + 512
        assert size(M, N, K - 32, R, 1) >= h + 4 * M * N         # another kernel's, with a finalize behind it
        assert size(M, N, K, R, 2) >= 2 * h - 8 * M + 4 * M * N  # segments may straddle a wave's features
    assert size(255, 2880, 4096, 64, 1) >= 255 * (8 * 2880 * 4 + 64 * 4 + 8)


def test_segments_are_read_at_every_call():
    """The cached C array is found by the widths themselves: a tensor that holds one may change between calls, and what is no
    integer is refused each time."""
    width = torch.tensor(64)
    assert list(ops._segments((width, 32))[1]) == [64, 32]
    width.fill_(16)
    assert list(ops._segments((width, 32))[1]) == [16, 32]
    for _ in range(2):
        assert list(ops._segments((64, 32))[1]) == [64, 32] and ops._segments(())[0] == 0
        with pytest.raises(TypeError):
            ops._segments((64.0, 32))


def test_a_source_needs_both_pools():
    k = torch.zeros(2, 1024, dtype=torch.bfloat16)
    for pools in ({"src_k": k}, {"src_v": k}):
        with pytest.raises(ValueError, match="both"):
            ops.kv_fork(k, k, 1, (0, 64), [(64 * 64, 64)], 0, 1, **pools)
