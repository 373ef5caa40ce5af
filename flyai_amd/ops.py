"""Torch-tensor wrappers around the C ABI (one call = one HIP launch sequence on the current stream).

PyTorch provides device memory and the stream; every computation happens in libflyai_stage.so.
Each wrapper checks dtype / device / contiguity / shape on the host before the launch."""
import ctypes as C
import functools
import operator
import struct

import numpy as np
import torch

from . import _lib
from ._lib import check, lib


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


def _need(t, dtype, shape=None, name="tensor"):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be on the GPU")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return t


def pack_ragged(q_lens, starts, kv_base, kv_cap, head_dim, max_tokens):
    """Device int32 q_lens/starts/kv_cap [S], int64 kv_base [S] -> dict of packed index tensors."""
    S = q_lens.numel()
    for n, t, dt in (("q_lens", q_lens, torch.int32), ("starts", starts, torch.int32),
                     ("kv_cap", kv_cap, torch.int32), ("kv_base", kv_base, torch.int64)):
        _need(t, dt, (S,), n)
    dev = q_lens.device
    out = dict(cu_seqlens=torch.empty(S + 1, dtype=torch.int32, device=dev),
               positions=torch.empty(max_tokens, dtype=torch.int32, device=dev),
               seq_id=torch.empty(max_tokens, dtype=torch.int32, device=dev),
               kv_len=torch.empty(S, dtype=torch.int32, device=dev),
               kv_slot=torch.empty(max_tokens, dtype=torch.int64, device=dev),
               status=torch.empty(1, dtype=torch.int32, device=dev))
    check(lib().flyai_pack_ragged(_ptr(q_lens), _ptr(starts), _ptr(kv_base), _ptr(kv_cap), S, head_dim,
                                  max_tokens, _ptr(out["cu_seqlens"]), _ptr(out["positions"]),
                                  _ptr(out["seq_id"]), _ptr(out["kv_len"]), _ptr(out["kv_slot"]),
                                  _ptr(out["status"]), _stream()))
    return out


def router_topk_softmax(x, w, b, k, want_logits=False):
    T, H = x.shape
    E = w.shape[0]
    _need(x, torch.bfloat16, (T, H), "x")
    _need(w, torch.bfloat16, (E, H), "router weight")
    _need(b, torch.bfloat16, (E,), "router bias")
    ids = torch.empty(T, k, dtype=torch.int32, device=x.device)
    wts = torch.empty(T, k, dtype=torch.float32, device=x.device)
    logits = torch.empty(T, E, dtype=torch.float32, device=x.device)
    check(lib().flyai_router_topk_softmax(_ptr(x), _ptr(w), _ptr(b), T, H, E, k, _ptr(ids), _ptr(wts),
                                          _ptr(logits), _stream()))
    return (ids, wts, logits) if want_logits else (ids, wts)


def moe_permute(ids, n_experts):
    T, k = ids.shape
    _need(ids, torch.int32, (T, k), "topk_ids")
    dev = ids.device
    hist = torch.empty(n_experts, dtype=torch.int32, device=dev)
    offsets = torch.empty(n_experts + 1, dtype=torch.int32, device=dev)
    perm = torch.empty(T * k, dtype=torch.int32, device=dev)
    inv = torch.empty(T * k, dtype=torch.int32, device=dev)
    check(lib().flyai_moe_permute(_ptr(ids), T, k, n_experts, _ptr(hist), _ptr(offsets), _ptr(perm),
                                  _ptr(inv), _stream()))
    return hist, offsets, perm, inv


def moe_route_permute(x, w, b, k):
    """Router + histogram/permute as the stage runs it -> (ids, weights, hist, offsets, perm, inv)."""
    T, H = x.shape
    E = w.shape[0]
    _need(x, torch.bfloat16, (T, H), "x")
    _need(w, torch.bfloat16, (E, H), "router weight")
    _need(b, torch.bfloat16, (E,), "router bias")
    dev = x.device
    ids = torch.empty(T, k, dtype=torch.int32, device=dev)
    wts = torch.empty(T, k, dtype=torch.float32, device=dev)
    logits = torch.empty(T, E, dtype=torch.float32, device=dev)
    hist = torch.empty(E, dtype=torch.int32, device=dev)
    offsets = torch.empty(E + 1, dtype=torch.int32, device=dev)
    perm = torch.empty(T * k, dtype=torch.int32, device=dev)
    inv = torch.empty(T * k, dtype=torch.int32, device=dev)
    check(lib().flyai_moe_route_permute(_ptr(x), _ptr(w), _ptr(b), T, H, E, k, _ptr(ids), _ptr(wts),
                                        _ptr(logits), _ptr(hist), _ptr(offsets), _ptr(perm), _ptr(inv),
                                        _stream()))
    return ids, wts, hist, offsets, perm, inv


def moe_combine(y_perm, inv, topk_w, residual=None, out=None):
    T, k = topk_w.shape
    H = y_perm.shape[1]
    _need(y_perm, torch.float32, (T * k, H), "y_perm")
    _need(inv, torch.int32, (T * k,), "inv")
    _need(topk_w, torch.float32, (T, k), "topk_w")
    if residual is not None:
        _need(residual, torch.bfloat16, (T, H), "residual")
    if out is None:
        out = torch.empty(T, H, dtype=torch.bfloat16, device=y_perm.device)
    _need(out, torch.bfloat16, (T, H), "out")
    check(lib().flyai_moe_combine(_ptr(y_perm), _ptr(inv), _ptr(topk_w), T, k, H, _ptr(residual),
                                  _ptr(out), _stream()))
    return out


def mxfp4_packed_bytes(E, N, K):
    return int(lib().flyai_mxfp4_packed_bytes(E, N, K))


def mxfp4_repack(blocks, scales):
    """HF layout blocks u8 [E, N, K/32, 16] + scales u8 [E, N, K/32] -> packed u8 buffer."""
    E, N, G, _ = blocks.shape
    _need(blocks, torch.uint8, (E, N, G, 16), "blocks")
    _need(scales, torch.uint8, (E, N, G), "scales")
    packed = torch.empty(mxfp4_packed_bytes(E, N, G * 32), dtype=torch.uint8, device=blocks.device)
    check(lib().flyai_mxfp4_repack(_ptr(blocks), _ptr(scales), E, N, G * 32, _ptr(packed), _stream()))
    return packed


def moe_gate_up(x, perm, offsets, k, w13_packed, b13, n_experts, inter):
    T, H = x.shape
    _need(x, torch.bfloat16, (T, H), "x")
    _need(perm, torch.int32, (T * k,), "perm")
    _need(offsets, torch.int32, (n_experts + 1,), "offsets")
    _need(b13, torch.float32, (n_experts, 2 * inter), "b13")
    _need(w13_packed, torch.uint8, (mxfp4_packed_bytes(n_experts, 2 * inter, H),), "w13_packed")
    h = torch.empty(T * k, inter, dtype=torch.bfloat16, device=x.device)
    check(lib().flyai_moe_gate_up_mxfp4(_ptr(x), _ptr(perm), _ptr(offsets), T, k, _ptr(w13_packed),
                                        _ptr(b13), n_experts, H, inter, _ptr(h), _stream()))
    return h


def moe_down(h, offsets, w2_packed, b2, n_experts, hidden):
    P, inter = h.shape
    _need(h, torch.bfloat16, (P, inter), "h")
    _need(offsets, torch.int32, (n_experts + 1,), "offsets")
    _need(b2, torch.float32, (n_experts, hidden), "b2")
    _need(w2_packed, torch.uint8, (mxfp4_packed_bytes(n_experts, hidden, inter),), "w2_packed")
    y = torch.empty(P, hidden, dtype=torch.float32, device=h.device)
    check(lib().flyai_moe_down_mxfp4(_ptr(h), _ptr(offsets), P, _ptr(w2_packed), _ptr(b2), n_experts,
                                     hidden, inter, _ptr(y), _stream()))
    return y


def mx_act_quant(x):
    """bf16 [M, K] -> the two-term e4m3 form: (bytes u8 [2M, K], E8M0 scale bytes u8 [2M, row bytes] in
    MFMA order); row r holds the high term of x[r], row M + r its low term."""
    M, K = x.shape
    _need(x, torch.bfloat16, (M, K), "x")
    q = torch.empty(2 * M, K, dtype=torch.uint8, device=x.device)
    s = torch.empty(int(lib().flyai_mx_act_scale_bytes(2 * M, K)), dtype=torch.uint8, device=x.device)
    check(lib().flyai_mx_act_quant(_ptr(x), M, K, _ptr(q), _ptr(s), _stream()))
    return q, s.view(2 * M, -1) if M else s.view(0, 0)


def moe_gate_up_fp8act(x, xq, xs, perm, offsets, k, w13_packed, b13, n_experts, inter):
    """gate_up with the dense groups on the scaled MFMA (two-term fp8 activations xq/xs = mx_act_quant(x))."""
    T, H = x.shape
    _need(x, torch.bfloat16, (T, H), "x")
    _need(xq, torch.uint8, (2 * T, H), "xq")
    _need(xs, torch.uint8, (2 * T, int(lib().flyai_mx_act_scale_bytes(1, H))), "xs")
    _need(perm, torch.int32, (T * k,), "perm")
    _need(offsets, torch.int32, (n_experts + 1,), "offsets")
    _need(b13, torch.float32, (n_experts, 2 * inter), "b13")
    _need(w13_packed, torch.uint8, (mxfp4_packed_bytes(n_experts, 2 * inter, H),), "w13_packed")
    h = torch.empty(T * k, inter, dtype=torch.bfloat16, device=x.device)
    check(lib().flyai_moe_gate_up_mxfp4_fp8act(_ptr(x), _ptr(xq), _ptr(xs), _ptr(perm), _ptr(offsets), T, k,
                                               _ptr(w13_packed), _ptr(b13), n_experts, H, inter, _ptr(h),
                                               _stream()))
    return h


def moe_down_fp8act(h, hq, hs, offsets, w2_packed, b2, n_experts, hidden):
    """down with the dense groups on the scaled MFMA (two-term fp8 activations hq/hs = mx_act_quant(h))."""
    P, I = h.shape
    _need(h, torch.bfloat16, (P, I), "h")
    _need(hq, torch.uint8, (2 * P, I), "hq")
    _need(hs, torch.uint8, (2 * P, int(lib().flyai_mx_act_scale_bytes(1, I))), "hs")
    _need(offsets, torch.int32, (n_experts + 1,), "offsets")
    _need(b2, torch.float32, (n_experts, hidden), "b2")
    _need(w2_packed, torch.uint8, (mxfp4_packed_bytes(n_experts, hidden, I),), "w2_packed")
    y = torch.empty(P, hidden, dtype=torch.float32, device=h.device)
    check(lib().flyai_moe_down_mxfp4_fp8act(_ptr(h), _ptr(hq), _ptr(hs), _ptr(offsets), P, _ptr(w2_packed),
                                            _ptr(b2), n_experts, hidden, I, _ptr(y), _stream()))
    return y


def rmsnorm(x, w, eps=1e-5):
    T, H = x.shape
    _need(x, torch.bfloat16, (T, H), "x")
    _need(w, torch.float32, (H,), "weight")
    y = torch.empty_like(x)
    check(lib().flyai_rmsnorm(_ptr(x), _ptr(w), T, H, eps, _ptr(y), _stream()))
    return y


def linear(x, w, b=None, residual=None):
    """y = bf16(x W^T + b); with residual, residual <- bf16(residual + y) (returned)."""
    M, K = x.shape
    N = w.shape[0]
    _need(x, torch.bfloat16, (M, K), "x")
    _need(w, torch.bfloat16, (N, K), "weight")
    if b is not None:
        _need(b, torch.bfloat16, (N,), "bias")
    y = None
    if residual is not None:
        _need(residual, torch.bfloat16, (M, N), "residual")
    else:
        y = torch.empty(M, N, dtype=torch.bfloat16, device=x.device)
    ws = torch.empty(max(1, int(lib().flyai_linear_workspace_bytes(M, N, K)) // 4), dtype=torch.float32,
                     device=x.device)
    check(lib().flyai_linear_bf16(_ptr(x), _ptr(w), _ptr(b), M, N, K, _ptr(y), _ptr(residual), _ptr(ws),
                                  _stream()))
    return residual if residual is not None else y


def rope_kv_append(qkv, positions, seq_id, cos_tab, sin_tab, n_q_heads, n_kv_heads, head_dim,
                   kv_base, kv_cap, k_pool, v_pool, kv_pos=None):
    """kv_pos int32: where a token's K and V go in its slab, when that is not its position (``pack_shared``)."""
    T = qkv.shape[0]
    _need(qkv, torch.bfloat16, (T, (n_q_heads + 2 * n_kv_heads) * head_dim), "qkv")
    _need(positions, torch.int32, None, "positions")
    _need(seq_id, torch.int32, None, "seq_id")
    _need(cos_tab, torch.bfloat16, None, "cos")
    _need(sin_tab, torch.bfloat16, cos_tab.shape, "sin")
    _need(kv_base, torch.int64, None, "kv_base")
    _need(kv_cap, torch.int32, kv_base.shape, "kv_cap")
    _need(k_pool, torch.bfloat16, None, "k_pool")
    _need(v_pool, torch.bfloat16, k_pool.shape, "v_pool")
    if positions.numel() < T or seq_id.numel() < T:
        raise ValueError("positions/seq_id shorter than the token count")
    q = torch.empty(T, n_q_heads, head_dim, dtype=torch.bfloat16, device=qkv.device)
    if kv_pos is not None:
        _need(kv_pos, torch.int32, None, "kv_pos")
        if kv_pos.numel() < T:
            raise ValueError("kv_pos shorter than the token count")
        check(lib().flyai_rope_kv_append_at(_ptr(qkv), _ptr(positions), _ptr(kv_pos), _ptr(seq_id), _ptr(cos_tab), _ptr(sin_tab),
                                            cos_tab.shape[0], T, n_q_heads, n_kv_heads, head_dim, _ptr(kv_base), _ptr(kv_cap),
                                            _ptr(q), _ptr(k_pool), _ptr(v_pool), _stream()))
        return q
    check(lib().flyai_rope_kv_append(_ptr(qkv), _ptr(positions), _ptr(seq_id), _ptr(cos_tab),
                                     _ptr(sin_tab), cos_tab.shape[0], T, n_q_heads, n_kv_heads, head_dim, _ptr(kv_base),
                                     _ptr(kv_cap), _ptr(q), _ptr(k_pool), _ptr(v_pool), _stream()))
    return q


def attn_plan(q_lens, starts, n_kv_heads, window, split_keys, max_items=1 << 20):
    """Host planner -> (items int32 [n, 8], groups int32 [g, 8], n_small) on the CPU."""
    S = len(q_lens)
    ql = (C.c_int32 * S)(*[int(v) for v in q_lens])
    st = (C.c_int32 * S)(*[int(v) for v in starts])
    max_groups = (S + sum((int(v) + 3) // 4 for v in q_lens)) * n_kv_heads
    items = (_lib.AttnItem * max_items)()
    groups = (_lib.AttnGroup * max_groups)()
    ni, ng, ns = C.c_int32(0), C.c_int32(0), C.c_int32(0)
    check(lib().flyai_attn_plan(ql, st, S, n_kv_heads, window, split_keys, items, max_items, groups,
                                max_groups, C.byref(ni), C.byref(ng), C.byref(ns)))
    it = torch.frombuffer(bytearray(items), dtype=torch.int32).view(max_items, 8)[:ni.value].clone()
    gr = torch.frombuffer(bytearray(groups), dtype=torch.int32).view(max_groups, 8)[:ng.value].clone()
    return it, gr, ns.value


def attn_plan_prefill(q_lens, starts, n_kv_heads, window, split_keys, prefill_min, max_items=1 << 20):
    """attn_plan with sequences of q_len >= prefill_min as prefill items -> (items, groups, n_small,
    pitems) on the CPU."""
    S = len(q_lens)
    ql = (C.c_int32 * S)(*[int(v) for v in q_lens])
    st = (C.c_int32 * S)(*[int(v) for v in starts])
    max_groups = (S + sum((int(v) + 3) // 4 for v in q_lens)) * n_kv_heads
    max_pitems = (S + sum((int(v) + 15) // 16 for v in q_lens)) * n_kv_heads
    items = (_lib.AttnItem * max_items)()
    groups = (_lib.AttnGroup * max_groups)()
    pitems = (_lib.AttnItem * max_pitems)()
    ni, ng, ns, npi = C.c_int32(0), C.c_int32(0), C.c_int32(0), C.c_int32(0)
    check(lib().flyai_attn_plan_prefill(ql, st, S, n_kv_heads, window, split_keys, prefill_min, items, max_items,
                                        groups, max_groups, pitems, max_pitems, C.byref(ni), C.byref(ng),
                                        C.byref(ns), C.byref(npi)))
    it = torch.frombuffer(bytearray(items), dtype=torch.int32).view(max_items, 8)[:ni.value].clone()
    gr = torch.frombuffer(bytearray(groups), dtype=torch.int32).view(max_groups, 8)[:ng.value].clone()
    pit = torch.frombuffer(bytearray(pitems), dtype=torch.int32).view(max_pitems, 8)[:npi.value].clone()
    return it, gr, ns.value, pit


def attn_prefill(q, k_pool, v_pool, kv_base, kv_cap, sinks, window, pitems, n_kv_heads, out):
    """Run prefill items (attn_plan_prefill) into the rows of out bf16 [T, Hq, 64]."""
    T, Hq, D = q.shape
    _need(q, torch.bfloat16, (T, Hq, D), "q")
    _need(out, torch.bfloat16, (T, Hq, D), "out")
    pit = pitems.to(q.device).contiguous()
    check(lib().flyai_attn_prefill(_ptr(q), _ptr(k_pool), _ptr(v_pool), _ptr(kv_base), _ptr(kv_cap), _ptr(sinks),
                                   window, Hq, n_kv_heads, D, _ptr(pit), pitems.shape[0], _ptr(out), _stream()))
    return out


def attn_ragged(q, k_pool, v_pool, kv_base, kv_cap, sinks, window, items, groups, n_small, n_kv_heads):
    """q bf16 [T, Hq, 64]; items/groups/n_small from attn_plan (moved to the GPU here)."""
    T, Hq, D = q.shape
    _need(q, torch.bfloat16, (T, Hq, D), "q")
    _need(sinks, torch.float32, (Hq,), "sinks")
    dev = q.device
    items_d = items.to(dev).contiguous()
    groups_d = groups.to(dev).contiguous()
    parts = torch.empty(max(1, int(lib().flyai_attn_partials_bytes(items.shape[0])) // 4),
                        dtype=torch.float32, device=dev)
    out = torch.empty_like(q)
    check(lib().flyai_attn_ragged(_ptr(q), _ptr(k_pool), _ptr(v_pool), _ptr(kv_base), _ptr(kv_cap),
                                  _ptr(sinks), window, Hq, n_kv_heads, D, _ptr(items_d), items.shape[0],
                                  n_small, _ptr(groups_d), groups.shape[0], _ptr(parts), _ptr(out),
                                  _stream()))
    return out


# ---- many requests at once: adapters, rotary positions, the cache's slabs ------------------------

def _need_all(device, *tensors):
    """``_need`` of each (name, tensor, dtype, shape), and all on one device; the checks that pass cost little."""
    for name, t, dtype, shape in tensors:
        try:
            if t.dtype is dtype and t.shape == shape and t.is_contiguous() and t.get_device() == device >= 0:
                continue
        except AttributeError:  # (no tensor)
            pass
        _need(t, dtype, shape, name)
        raise ValueError(f"{name} is on {t.device}, the first tensor on another device")


def _on(device, fn, *args):
    """fn(*args, the current stream of the device) with the device current: a launch goes to the current device."""
    if device == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    if rc:
        check(rc)


def _address(t):
    return t.data_ptr() if t is not None else None


def _segments(widths):
    """(how many, their int32 array), the array made once for the same widths."""
    return _segment_array(tuple([operator.index(w) for w in widths]))


@functools.lru_cache(maxsize=64)
def _segment_array(widths):
    return len(widths), (C.c_int32 * len(widths))(*map(_position, widths))


@functools.lru_cache(maxsize=256)
def _lora_workspace_bytes(M, N, K, R, S):
    return max(16, int(lib().flyai_linear_lora_workspace_bytes(M, N, K, R, S)))


def linear_lora(x, w, b, lora_a, lora_b, scale, ranks, adapter, segments=None, row_seq=None, residual=None):
    """``linear`` with a low-rank adapter of its own for each row: y = bf16(x W^T + b + s_a (x A_a^T) B_a^T), with residual
    residual <- bf16(residual + y) (returned; it must not overlap x).  lora_a bf16 [n, S * R, K], lora_b bf16 [n, N, R], scale fp32 [n], ranks
    int32 [n] (adapter a uses the first ranks[a] of R rows of each segment's A and columns of B; nothing past them is
    used); R a multiple of 16 up to 128.  segments: the S (at most 4) widths of the output's runs that have an A of
    their own (None: one of N).  adapter int32: of each row [M], or with row_seq int32 [M] of each sequence; ids outside
    [0, n) mean no adapter, and such a row has ``linear``'s bits.  A row's result depends on that row alone.  h = s_a x A_a^T is
    kept to 16 significant bits, in two terms: where B is infinite the result may be NaN in place of an infinity."""
    M, K = x.shape
    N = w.shape[0]
    S, widths = _segments((N,) if segments is None else segments)
    if lora_b.dim() != 3:
        raise ValueError("lora_b must be [adapters, N, R]")
    n, _, R = lora_b.shape
    dev, bf16, i32 = x.get_device(), torch.bfloat16, torch.int32
    n_ids = adapter.numel()
    _need_all(dev, ("x", x, bf16, (M, K)), ("weight", w, bf16, (N, K)), ("lora_b", lora_b, bf16, (n, N, R)),
              ("lora_a", lora_a, bf16, (n, S * R, K)), ("scale", scale, torch.float32, (n,)), ("ranks", ranks, i32, (n,)),
              ("adapter", adapter, i32, (M,) if row_seq is None else (n_ids,)))
    if b is not None:
        _need_all(dev, ("bias", b, bf16, (N,)))
    if row_seq is not None:
        _need_all(dev, ("row_seq", row_seq, i32, (M,)))
    y = None
    if residual is not None:
        _need_all(dev, ("residual", residual, bf16, (M, N)))
    else:
        y = torch.empty(M, N, dtype=bf16, device=x.device)
    ws = torch.empty(_lora_workspace_bytes(M, N, K, R, S), dtype=torch.uint8, device=x.device)
    _on(dev, lib().flyai_linear_lora_bf16, x.data_ptr(), w.data_ptr(), _address(b), M, N, K, lora_a.data_ptr(),
        lora_b.data_ptr(), scale.data_ptr(), ranks.data_ptr(), n, R, widths, S, adapter.data_ptr(),
        _address(row_seq), n_ids, _address(y), _address(residual), ws.data_ptr())
    return residual if residual is not None else y


_ROPE_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_ROPE_LAYOUTS = {"half": 0, "interleaved": 1}


def rope(x, positions, inv_freq, layout="half", scaling=1.0, inverse=False, out=None):
    """Rotary positions on x [T, H, D] (bf16, fp16 or fp32; a view whose last dim is contiguous, such as the q and k heads
    of fused projection rows): dims [0, 2 * len(inv_freq)) of each head are turned by positions[t] * inv_freq[i] (int32 [T],
    fp64; ``rope.rope_frequencies`` gives scaled ones) and multiplied by scaling, the others copied.  Pairs are (i, i +
    rot/2) ("half") or (2i, 2i + 1) ("interleaved").  inverse turns back: the gradient of the rotation.  out: a tensor
    of x's shape and type (x itself: in place; otherwise wholly before or behind x in memory), None: a new contiguous one."""
    if not isinstance(x, torch.Tensor) or x.dim() != 3:
        raise ValueError("x must be a [T, H, D] tensor")
    dev = x.get_device()
    if dev < 0:
        raise ValueError("x must be on the GPU")
    dtype = _ROPE_TYPES.get(x.dtype)
    if dtype is None:
        raise TypeError(f"x must be bf16, fp16 or fp32, got {x.dtype}")
    if layout not in _ROPE_LAYOUTS:
        raise ValueError(f"layout must be one of {sorted(_ROPE_LAYOUTS)}, got {layout!r}")
    T, H, D = x.shape
    pairs = inv_freq.numel()
    _need_all(dev, ("positions", positions, torch.int32, (T,)), ("inv_freq", inv_freq, torch.float64, (pairs,)))
    if out is None:
        out = torch.empty(T, H, D, dtype=x.dtype, device=x.device)
        ot, oh, od = H * D, D, 1
    else:
        if out.dtype != x.dtype or out.shape != x.shape or out.get_device() != dev:
            raise ValueError(f"out must be {x.dtype} of shape {tuple(x.shape)} on {x.device}")
        ot, oh, od = out.stride()
    xt, xh, xd = x.stride()
    if D > 1 and (xd != 1 or od != 1):
        raise ValueError("the last dim of x and out must be contiguous")
    if T == 0 or H == 0:
        return out
    _on(dev, lib().flyai_rope, x.data_ptr(), xt, xh, positions.data_ptr(), inv_freq.data_ptr(), float(scaling), T, H, D, 2 * pairs,
        dtype, _ROPE_LAYOUTS[layout], 1 if inverse else 0, out.data_ptr(), ot, oh)
    return out


def _kv_pools(k, v):
    """(layers, elements a layer, device) of K and V pools [L, n] (or one layer's [n])."""
    if not isinstance(k, torch.Tensor) or k.dim() not in (1, 2):
        raise ValueError("k and v must be pools of one shape, [layers, elements] or [elements]")
    shape, dev, bf16 = k.shape, k.get_device(), torch.bfloat16
    if not (isinstance(v, torch.Tensor) and k.dtype is bf16 and v.dtype is bf16 and v.shape == shape and v.get_device() == dev >= 0
            and k.is_contiguous() and v.is_contiguous()):
        _need_all(dev, ("k", k, bf16, shape), ("v", v, bf16, shape))
    return (shape[0] if len(shape) == 2 else 1), shape[-1], dev


_KV_SLAB, _KV_MOVE = struct.Struct("qii"), struct.Struct("qiiii")  # flyai_kv_slab, flyai_kv_move


def kv_fork(k, v, n_kv_heads, src, dsts, lo, hi, src_k=None, src_v=None):
    """Copy positions [lo, hi) of slab src to the same positions of the slabs dsts, every layer, in one launch for every 64 of
    them.  k, v: pools bf16 [L, elements] in the tiled slab layout; a slab is (base, cap).  src_k, src_v: the pools that hold src, when
    they are others.  Nothing outside [lo, hi) changes.  Positions past a slab raise ContextOverflow."""
    if (src_k is None) != (src_v is None):
        raise ValueError("a source in other pools needs both src_k and src_v")
    L, n, dev = _kv_pools(k, v)
    sn = n
    if src_k is None:
        src_k, src_v = k, v
    else:
        sL, sn, sdev = _kv_pools(src_k, src_v)
        if sL != L or sdev != dev:
            raise ValueError(f"the source's pools have {sL} layers on device {sdev}, the others {L} on {dev}")
    slabs = _packed(_KV_SLAB, [(b, c, 0) for b, c in (src, *dsts)])
    lo, hi = (_position(p) for p in (lo, hi))
    _on(dev, lib().flyai_kv_fork, src_k.data_ptr(), src_v.data_ptr(), sn, sn, k.data_ptr(), v.data_ptr(), n, n, L, _position(n_kv_heads),
        64, slabs[:_KV_SLAB.size], slabs[_KV_SLAB.size:], len(dsts), lo, hi)


def _position(p):
    """An int32 that is out of range where p is: what a C int would make of a larger one may be a position."""
    if type(p) is int and -1 <= p <= 0x7fffffff:  # (most of them: a third of the time)
        return p
    return min(max(operator.index(p), -1), 0x7fffffff)


def _host_positions(keep):
    """The int32s of a list, an array or a CPU tensor of positions, as bytes."""
    try:
        if isinstance(keep, (list, tuple, range)):
            if not keep or keep[0] >= 0:  # ascending from there: the C call checks
                return struct.pack(f"{len(keep)}i", *keep)
        else:
            a = np.asarray(keep).reshape(-1)
            if a.size == 0 or (a.dtype.kind in "iu" and a.min() >= 0 and a.max() <= 0x7fffffff):
                return a.astype(np.int32).tobytes()
    except (TypeError, struct.error):
        pass
    raise ValueError("keep must hold positions (non-negative integers)")


def _packed(layout, rows):
    try:
        return b"".join([layout.pack(*r) for r in rows])
    except struct.error:
        raise ValueError("slabs and starts must be integers in range") from None


def kv_compact(k, v, n_kv_heads, moves):
    """For each move (base, cap, start, keep): position start + i of the slab takes what position start + keep[i] held
    before the call, every layer.  keep: host integers (list, numpy or CPU tensor), strictly ascending.  The moves' slabs
    must not overlap.  A launch takes up to 16 slabs and 336 of their 64-position blocks, a slab's counted from its first
    position that moves to its last that stays; more take more launches."""
    L, n, dev = _kv_pools(k, v)
    keeps = [_host_positions(m[3]) for m in moves]
    rows = _packed(_KV_MOVE, [(base, cap, start, len(a) // 4, 0) for (base, cap, start, _), a in zip(moves, keeps)])
    _on(dev, lib().flyai_kv_compact, k.data_ptr(), v.data_ptr(), n, n, L, _position(n_kv_heads), 64, rows, len(moves), b"".join(keeps))


# ---- batches that share prompts -----------------------------------------------------------------

# The status word of pack_shared and of a plan
PAST_SLAB, PAST_TOKENS, BEFORE_PREFIX, BAD_PREFIX, BAD_SEQUENCE = 1, 2, 4, 8, 16


def pack_shared(q_lens, starts, kv_base, kv_cap, prefix_of, prefix_len, head_dim, max_tokens):
    """``pack_ragged`` for sequences behind shared prefixes: sequence b's first prefix_len[prefix_of[b]] positions lie in a slab
    that it shares (prefix_of negative: none), its own slab (kv_base, kv_cap) holds what follows.  Device int32 q_lens,
    starts (the first new token's position), kv_cap, prefix_of [S], prefix_len [n], int64 kv_base [S] -> dict of cu_seqlens,
    positions, seq_id, kv_len as in ``pack_ragged``, kv_pos int32 (a token's slab position), kv_slot int64 (its element, -1 past
    the slab) and status (PAST_SLAB, ... bits; 0: all is well).  A sequence of BEFORE_PREFIX, BAD_PREFIX or BAD_SEQUENCE gets no kv_pos and
    kv_slot (-1); of one past its slab or max_tokens the tokens that fit keep theirs.  That slabs lie in the pools is not checked here, but by
    ``attn_shared_plan``.  max_tokens may be more than the batch has: positions, seq_id, kv_pos
    and kv_slot are -1 behind its last token, and ``rope_kv_append`` skips such rows.  Lengths may come from the GPU: nothing is read
    back."""
    S, n = q_lens.numel(), prefix_len.numel()
    i32 = torch.int32
    dev = q_lens.get_device()
    _need_all(dev, ("q_lens", q_lens, i32, (S,)), ("starts", starts, i32, (S,)), ("kv_base", kv_base, torch.int64, (S,)),
              ("kv_cap", kv_cap, i32, (S,)), ("prefix_of", prefix_of, i32, (S,)), ("prefix_len", prefix_len, i32, (n,)))
    max_tokens = _position(max_tokens)
    m = max(max_tokens, 0)
    # (one allocation for the int32s: six would cost more than the kernel)
    ints, kv_slot = q_lens.new_empty(2 * S + 2 + 3 * m), kv_base.new_empty(m)
    p = ints.data_ptr()
    cu, pos, seq, kv_pos, kv_len = p, p + 4 * (S + 1), p + 4 * (S + 1 + m), p + 4 * (S + 1 + 2 * m), p + 4 * (S + 1 + 3 * m)
    _on(dev, lib().flyai_pack_shared, q_lens.data_ptr(), starts.data_ptr(), kv_base.data_ptr(), kv_cap.data_ptr(), prefix_of.data_ptr(),
        prefix_len.data_ptr(), S, n, _position(head_dim), max_tokens, cu, pos, seq, kv_pos, kv_slot.data_ptr(), kv_len, kv_len + 4 * S)
    cu, pos, seq, kv_pos, kv_len, status = ints.split_with_sizes((S + 1, m, m, m, S, 1))
    return dict(cu_seqlens=cu, positions=pos, seq_id=seq, kv_pos=kv_pos, kv_len=kv_len, kv_slot=kv_slot, status=status)


class AttnSharedPlan:
    """The work lists of a batch and a window (``attn_shared_plan``), on the GPU.  status int32 [1]: PAST_SLAB, ... bits."""

    __slots__ = ("buffer", "n_tokens", "n_seqs", "n_prefixes", "n_kv_heads", "window", "pool_elems")

    def __init__(self, buffer, n_tokens, n_seqs, n_prefixes, n_kv_heads, window, pool_elems):
        self.buffer, self.n_tokens, self.n_seqs, self.n_prefixes = buffer, n_tokens, n_seqs, n_prefixes
        self.n_kv_heads, self.window, self.pool_elems = n_kv_heads, window, pool_elems

    @property
    def status(self):
        return self.buffer[3:4]


@functools.lru_cache(maxsize=256)
def _attn_shared_sizes(T, S, n, Hkv):
    """int32s of a plan, fp32s of a workspace."""
    return max(4, int(lib().flyai_attn_shared_plan_bytes(T, S, n)) // 4), max(4, int(lib().flyai_attn_shared_workspace_bytes(T, Hkv)) // 4)


def attn_shared_plan(q_lens, starts, kv_base, kv_cap, prefix_of, prefix_len, prefix_base, prefix_cap, n_kv_heads, window, n_tokens,
                     pool_elems):
    """The work lists of ``attn_shared`` for a batch as in ``pack_shared`` and a window (0: full attention): made on the GPU, once for
    all layers of a step.  prefix_len, prefix_cap int32 [n], prefix_base int64 [n]: the prefixes' lengths and slabs, in the same pools
    as the sequences' (pool_elems elements each).  n_tokens: rows of q (the batch's tokens, or more)."""
    S, n = q_lens.numel(), prefix_len.numel()
    i32, i64 = torch.int32, torch.int64
    dev = q_lens.get_device()
    _need_all(dev, ("q_lens", q_lens, i32, (S,)), ("starts", starts, i32, (S,)), ("kv_base", kv_base, i64, (S,)),
              ("kv_cap", kv_cap, i32, (S,)), ("prefix_of", prefix_of, i32, (S,)), ("prefix_len", prefix_len, i32, (n,)),
              ("prefix_base", prefix_base, i64, (n,)), ("prefix_cap", prefix_cap, i32, (n,)))
    T, Hkv, window = _position(n_tokens), _position(n_kv_heads), _position(window)
    size, _ = _attn_shared_sizes(T, S, n, Hkv)
    plan = AttnSharedPlan(q_lens.new_empty(size), T, S, n, Hkv, window, operator.index(pool_elems))
    _on(dev, lib().flyai_attn_shared_plan, q_lens.data_ptr(), starts.data_ptr(), kv_base.data_ptr(), kv_cap.data_ptr(),
        prefix_of.data_ptr(), prefix_len.data_ptr(), prefix_base.data_ptr(), prefix_cap.data_ptr(), S, n, Hkv, window, T,
        plan.pool_elems, plan.buffer.data_ptr())
    return plan


def attn_shared(q, k_pool, v_pool, sinks, plan, out=None):
    """Attention of a batch that shares prefixes (``attn_ragged`` with each prefix's keys read once for all the rows behind it): q bf16
    [T, Hq, 64] rotated, k_pool and v_pool bf16 (the slabs that the plan names), sinks fp32 [Hq], Hq = 8 kv heads.  Returns
    out bf16 [T, Hq, 64] (None: a new one); rows behind the last sequence are left as they were, those of a sequence that the plan
    refused (plan.status) are zeros.  A row's bits depend on its own sequence, its prefix and the window, not on the batch.
    K and V outside the positions that a row sees may hold anything; an infinity in V that it sees with a weight below fp32's range counts for
    nothing or as NaN, which may differ between batches.  Each call allocates its workspace: 63 MB for 64 tokens of 8 kv heads, 361 for
    1,478, 2.5 GB for 65,536 (room for what may be split)."""
    T, Hkv = plan.n_tokens, plan.n_kv_heads
    dev, bf16 = q.get_device(), torch.bfloat16
    _need_all(dev, ("q", q, bf16, (T, 8 * Hkv, 64)), ("k_pool", k_pool, bf16, k_pool.shape), ("v_pool", v_pool, bf16, k_pool.shape),
              ("sinks", sinks, torch.float32, (8 * Hkv,)), ("plan", plan.buffer, torch.int32, plan.buffer.shape))
    if k_pool.numel() < plan.pool_elems:
        raise ValueError(f"the pools have {k_pool.numel()} elements, the plan was made for {plan.pool_elems}")
    if out is None:
        out = q.new_empty(q.shape)
    else:
        _need_all(dev, ("out", out, bf16, q.shape))
    _, size = _attn_shared_sizes(T, plan.n_seqs, plan.n_prefixes, Hkv)
    ws = sinks.new_empty(size)
    _on(dev, lib().flyai_attn_shared, q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), sinks.data_ptr(), 8 * Hkv, Hkv, 64, T,
        plan.n_seqs, plan.n_prefixes, plan.buffer.data_ptr(), ws.data_ptr(), out.data_ptr())
    return out


# ---- DeepSeek-V3-shaped FP8 MoE ------------------------------------------------------------------

def router_grouped_sigmoid(x, w, e_bias, n_group, topk_group, k, route_scale):
    """Grouped sigmoid routing on fp32 logits -> (ids int32 [T,k] ascending, weights fp32 [T,k],
    logits fp32 [T,E])."""
    T, H = x.shape
    E = w.shape[0]
    _need(x, torch.bfloat16, (T, H), "x")
    _need(w, torch.bfloat16, (E, H), "router weight")
    if e_bias is not None:
        _need(e_bias, torch.float32, (E,), "e_bias")
    dev = x.device
    logits = torch.empty(T, E, dtype=torch.float32, device=dev)
    ids = torch.empty(T, k, dtype=torch.int32, device=dev)
    wts = torch.empty(T, k, dtype=torch.float32, device=dev)
    check(lib().flyai_router_grouped_sigmoid(_ptr(x), _ptr(w), _ptr(e_bias), T, H, E, n_group, topk_group,
                                             k, float(route_scale), _ptr(logits), _ptr(ids), _ptr(wts),
                                             _stream()))
    return ids, wts, logits


def fp8_act_quant(x):
    """bf16 [M, K] -> (e4m3 bytes u8 [M, K], E8M0 scale bytes u8 [M, K/128])."""
    M, K = x.shape
    _need(x, torch.bfloat16, (M, K), "x")
    q = torch.empty(M, K, dtype=torch.uint8, device=x.device)
    s = torch.empty(M, K // 128, dtype=torch.uint8, device=x.device)
    check(lib().flyai_fp8_act_quant(_ptr(x), M, K, _ptr(q), _ptr(s), _stream()))
    return q, s


def fp8_packed_bytes(E, N, K):
    return int(lib().flyai_fp8_packed_bytes(E, N, K))


def fp8_repack(w1, s1, w3=None, s3=None):
    """e4m3 bytes w [E, N, K] + E8M0 block scales [E, ceil(N/128), K/128] -> packed u8 buffer.
    With w3/s3 (gate_up), rows of w1 and w3 are interleaved and the packed N is 2N."""
    E, N, K = w1.shape
    sb = (E, (N + 127) // 128, K // 128)
    _need(w1, torch.uint8, (E, N, K), "w1")
    _need(s1, torch.uint8, sb, "s1")
    if w3 is not None:
        _need(w3, torch.uint8, (E, N, K), "w3")
        _need(s3, torch.uint8, sb, "s3")
    Np = 2 * N if w3 is not None else N
    packed = torch.empty(fp8_packed_bytes(E, Np, K), dtype=torch.uint8, device=w1.device)
    check(lib().flyai_fp8_repack(_ptr(w1), _ptr(s1), _ptr(w3), _ptr(s3), E, N, K, _ptr(packed), _stream()))
    return packed


def moe_gate_up_fp8(xq, xs, perm, offsets, k, topk_w, w13_packed, n_experts, inter, n_shared=0):
    """Rows of expert e: token perm[p] // k (perm None: token p); h = bf16(silu(bf16 gate) * bf16 up
    * topk_w[perm[p]]) (topk_w None: 1) -> h bf16 [P + n_shared, inter], P = routed rows.  With
    n_shared > 0 the packed buffer holds the shared expert as expert n_experts; its rows P.. take
    tokens 0 .. n_shared-1 with weight 1."""
    T, H = xq.shape
    _need(xq, torch.uint8, (T, H), "xq")
    _need(xs, torch.uint8, (T, H // 128), "xs")
    _need(offsets, torch.int32, (n_experts + 1,), "offsets")
    if not 0 <= n_shared <= T:
        raise ValueError("n_shared must be in [0, T]")
    P = T * k if perm is not None else T
    if perm is not None:
        _need(perm, torch.int32, (P,), "perm")
    if topk_w is not None:
        _need(topk_w, torch.float32, None, "topk_w")
        if topk_w.numel() != P:
            raise ValueError("topk_w must hold one weight per routed row")
    groups = n_experts + (n_shared > 0)
    _need(w13_packed, torch.uint8, (fp8_packed_bytes(groups, 2 * inter, H),), "w13_packed")
    h = torch.empty(P + n_shared, inter, dtype=torch.bfloat16, device=xq.device)
    check(lib().flyai_moe_gate_up_fp8(_ptr(xq), _ptr(xs), _ptr(perm), _ptr(offsets), k, _ptr(topk_w),
                                      _ptr(w13_packed), n_experts, H, inter, n_shared, _ptr(h), _stream()))
    return h


def moe_down_fp8(hq, hs, offsets, w2_packed, n_experts, hidden, n_shared=0):
    """y[p] = bf16(hq[p] . W2[e]) for routed rows and, with n_shared > 0, the shared expert's rows
    (the last n_shared rows of hq) -> y bf16 [rows, hidden]."""
    R, inter = hq.shape
    _need(hq, torch.uint8, (R, inter), "hq")
    _need(hs, torch.uint8, (R, inter // 128), "hs")
    _need(offsets, torch.int32, (n_experts + 1,), "offsets")
    groups = n_experts + (n_shared > 0)
    _need(w2_packed, torch.uint8, (fp8_packed_bytes(groups, hidden, inter),), "w2_packed")
    y = torch.empty(R, hidden, dtype=torch.bfloat16, device=hq.device)
    check(lib().flyai_moe_down_fp8(_ptr(hq), _ptr(hs), _ptr(offsets), _ptr(w2_packed), n_experts, hidden,
                                   inter, n_shared, _ptr(y), _stream()))
    return y


def moe_combine_sum(y_perm, inv, k, shared=None, residual=None, out=None):
    """out[t] = bf16(sum_s y_perm[inv[t*k+s]] + shared[t]) (fp32), then bf16(residual + out)."""
    P, H = y_perm.shape
    T = P // k
    _need(y_perm, torch.bfloat16, (P, H), "y_perm")
    _need(inv, torch.int32, (P,), "inv")
    for n, t in (("shared", shared), ("residual", residual)):
        if t is not None:
            _need(t, torch.bfloat16, (T, H), n)
    if out is None:
        out = torch.empty(T, H, dtype=torch.bfloat16, device=y_perm.device)
    _need(out, torch.bfloat16, (T, H), "out")
    check(lib().flyai_moe_combine_sum(_ptr(y_perm), _ptr(inv), T, k, H, _ptr(shared), _ptr(residual),
                                      _ptr(out), _stream()))
    return out


def bf16_tile_repack(w):
    """nn.Linear weight bf16 [N, K] -> MFMA-fragment tiles (u8 buffer) for lm_head_argmax."""
    N, K = w.shape
    _need(w, torch.bfloat16, (N, K), "w")
    n = int(lib().flyai_bf16_tile_packed_bytes(N, K))
    if n == 0:
        raise ValueError("bf16_tile_repack needs N % 16 == 0 and K % 32 == 0")
    packed = torch.empty(n, dtype=torch.uint8, device=w.device)
    check(lib().flyai_bf16_tile_repack(_ptr(w), N, K, _ptr(packed), _stream()))
    return packed


def embed_gather(table, ids):
    """table bf16 [V, H], ids int32 [T] (device) -> bf16 [T, H]."""
    V, H = table.shape
    _need(table, torch.bfloat16, (V, H), "table")
    _need(ids, torch.int32, None, "ids")
    out = torch.empty(ids.numel(), H, dtype=torch.bfloat16, device=table.device)
    check(lib().flyai_embed_gather(_ptr(table), _ptr(ids), ids.numel(), H, V, _ptr(out), _stream()))
    return out


def lm_head_argmax(x, w_packed, vocab, rows=None, want_logits=False, workspace=None):
    """Greedy token of each selected row: x bf16 [R, H] final-normed hidden rows; rows int32 [n]
    (device; None: all R rows); returns ids int32 [n] (and bf16 logits [n, vocab])."""
    R, H = x.shape
    _need(x, torch.bfloat16, (R, H), "x")
    n = R if rows is None else rows.numel()
    if rows is not None:
        _need(rows, torch.int32, (n,), "rows")
    _need(w_packed, torch.uint8, (int(lib().flyai_bf16_tile_packed_bytes(vocab, H)),), "w_packed")
    ids = torch.empty(n, dtype=torch.int32, device=x.device)
    logits = torch.empty(n, vocab, dtype=torch.bfloat16, device=x.device) if want_logits else None
    need = int(lib().flyai_lm_head_workspace_bytes(n, vocab))
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=x.device)
    check(lib().flyai_lm_head_argmax(_ptr(x), _ptr(rows), n, H, _ptr(w_packed), vocab, _ptr(ids),
                                     _ptr(logits), _ptr(workspace), _stream()))
    return (ids, logits) if want_logits else ids


def sample_rows(logits, temp, top_k=0, top_p=1.0, draft=None, u=None, want_p_draft=False, want_draw=False,
                want_probs=False):
    """Temperature / top-k / top-p over bf16 logits rows [R, V].  draft int32 [R]
    (device, -1 = none) and u float64 [R] (device uniforms in [0, 1)) are optional; returns a dict with
    the requested outputs: p_draft fp32 [R], draw int32 [R] (needs u unless temp <= 0), probs fp32 [R, V]."""
    R, V = logits.shape
    _need(logits, torch.bfloat16, (R, V), "logits")
    if draft is not None:
        _need(draft, torch.int32, (R,), "draft")
    if u is not None:
        _need(u, torch.float64, (R,), "u")
    if want_draw and u is None and temp > 0:
        raise ValueError("a sampled draw needs uniforms u")
    dev = logits.device
    out = {}
    if want_p_draft:
        out["p_draft"] = torch.empty(R, dtype=torch.float32, device=dev)
    if want_draw:
        out["draw"] = torch.empty(R, dtype=torch.int32, device=dev)
    if want_probs:
        out["probs"] = torch.empty(R, V, dtype=torch.float32, device=dev)
    ws = torch.empty(int(lib().flyai_sample_workspace_bytes(R, V)), dtype=torch.uint8, device=dev)
    check(lib().flyai_sample_rows_ws(_ptr(logits), R, V, float(temp), int(top_k), float(top_p), _ptr(draft), _ptr(u),
                                     _ptr(out.get("p_draft")), _ptr(out.get("draw")), _ptr(out.get("probs")),
                                     _ptr(ws), _stream()))
    return out


@functools.lru_cache(maxsize=256)
def _spec_verify_bytes(R, V, S):
    return int(lib().flyai_spec_verify_workspace_bytes(R, V, S)) + 15


def spec_verify(logits, cu_rows, draft, u, u_draw, temp, top_k=0, top_p=1.0, draft_probs=None, probs_row=None):
    """Drafted tokens of many streams verified at once (``Sampler.accept``'s rule).  Stream s has the rows cu_rows[s] ..
    cu_rows[s + 1] - 1 of logits bf16 [R, V] (cu_rows int32 [S + 1], ascending); row r judges the token draft[r] (int32 [R]; -1: none, as in the
    last row of a stream, whose token is a bonus).  temp, top_k, top_p: numbers, or fp32, int32, fp32 [S] for each stream (temp <= 0:
    greedy).  draft_probs fp32 [n, V]: the distributions that the drafts were drawn from, row probs_row[r] (int32 [R]; -1: none;
    None: row r) for row r; a draft without one was not drawn.  u fp64 [R] and u_draw fp64 [S]: uniforms in [0, 1) for the
    acceptances and for each stream's draw.

    Returns (tokens int32 [R], counts int32 [S], p fp32 [R]), all on the GPU: in a stream's rows its accepted drafts, then the drawn
    token, then -1; how many tokens it got; and each token's probability under the filtered target (0 behind the end).  Rows of no stream
    are not written."""
    R, V = logits.shape
    S = cu_rows.numel() - 1
    if S < 0:
        raise ValueError("cu_rows needs at least one entry")
    dev = logits.get_device()
    f32, i32, f64 = torch.float32, torch.int32, torch.float64
    _need_all(dev, ("logits", logits, torch.bfloat16, (R, V)), ("cu_rows", cu_rows, i32, (S + 1,)), ("draft", draft, i32, (R,)),
              ("u", u, f64, (R,)), ("u_draw", u_draw, f64, (S,)))
    params = [None, None, None]
    for i, (name, v, dtype) in enumerate((("temp", temp, f32), ("top_k", top_k, i32), ("top_p", top_p, f32))):
        if isinstance(v, torch.Tensor):
            _need_all(dev, (name, v, dtype, (S,)))
            params[i] = v
    temp, top_k, top_p = (d if p is not None else v for p, v, d in zip(params, (temp, top_k, top_p), (0.0, 0, 1.0)))
    n = 0
    if draft_probs is not None:
        n = draft_probs.shape[0]
        _need_all(dev, ("draft_probs", draft_probs, f32, (n, V)))
        if probs_row is None and n != R:
            raise ValueError(f"draft_probs has {n} rows for {R} rows of logits: probs_row has to say whose they are")
    elif probs_row is not None:
        raise ValueError("probs_row without draft_probs")
    if probs_row is not None:
        _need_all(dev, ("probs_row", probs_row, i32, (R,)))
    tokens, counts, p = draft.new_empty(R), draft.new_empty(S), draft.new_empty(R, dtype=f32)
    ws = u.new_empty(_spec_verify_bytes(R, V, S) // 8)
    _on(dev, lib().flyai_spec_verify, logits.data_ptr(), R, V, cu_rows.data_ptr(), S, draft.data_ptr(), u.data_ptr(), u_draw.data_ptr(),
        _address(params[0]), _address(params[1]), _address(params[2]), float(temp), _position(top_k), float(top_p), _address(draft_probs), n,
        _address(probs_row), tokens.data_ptr(), counts.data_ptr(), p.data_ptr(), ws.data_ptr())
    return tokens, counts, p


def sample_probs(probs, u):
    """One draw from a fp32 probability vector [V] (device) at uniform u in [0, 1): int32 [1] on device."""
    V = probs.numel()
    _need(probs, torch.float32, (V,), "probs")
    out = torch.empty(1, dtype=torch.int32, device=probs.device)
    check(lib().flyai_sample_probs(_ptr(probs), V, float(u), _ptr(out), _stream()))
    return out
