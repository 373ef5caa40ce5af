"""Batches whose sequences share prefixes: packing, and attention over a prefix and a sequence's own keys, in 64 bits.

No counterpart in the reference, where a prompt's K/V is copied to every stream (``BatchedFastVerify.load_prefix``,
``phase0/batchverify.py:125-130``); the attention is ``oracle/attention.py``'s over the two runs of keys behind one another."""
import torch


def pack(q_lens, starts, kv_base, kv_cap, prefix_of, prefix_len, head_dim):
    """(cu_seqlens, positions, seq_id, kv_pos, kv_slot, kv_len) of well-formed sequences, as lists."""
    cu, pos, sid, kpos, slot = [0], [], [], [], []
    for b, n in enumerate(q_lens):
        behind = prefix_len[prefix_of[b]] if prefix_of[b] >= 0 else 0
        for i in range(n):
            p = starts[b] + i
            pos.append(p)
            sid.append(b)
            kpos.append(p - behind)
            slot.append(kv_base[b] + (p - behind) * head_dim if 0 <= p - behind < kv_cap[b] else -1)
        cu.append(cu[-1] + n)
    return cu, pos, sid, kpos, slot, [a + n for a, n in zip(starts, q_lens)]


def attention(q, keys, values, start, sinks, window):
    """q [n, Hq, D] at positions start .. start + n - 1; keys, values [Hkv, start + n, D] (the prefix's, then the sequence's own) ->
    (out, sum of p |v|), each fp64 [n, Hq, D].  Keys and values that a row does not see may hold anything."""
    n, Hq, D = q.shape
    Hkv, L, _ = keys.shape
    at, j = torch.arange(start, start + n)[:, None], torch.arange(L)
    seen = (j <= at) & ((j > at - window) if window else True)                  # [n, L]
    q = q.double().permute(1, 0, 2).reshape(Hkv, Hq // Hkv, n, D)
    score = torch.matmul(q, keys.double().transpose(1, 2)[:, None]) * D ** -0.5  # [Hkv, 8, n, L]
    score = torch.where(seen, score, float("-inf"))
    sink = sinks.double().reshape(Hkv, Hq // Hkv, 1, 1).expand(-1, -1, n, 1)
    p = torch.softmax(torch.cat((score, sink), 3), 3)[..., :-1]
    v = values.double()[:, None]
    if bool(torch.isfinite(v).all()):
        out, mag = torch.matmul(p, v), torch.matmul(p, v.abs())
    else:  # 0 x inf where a row does not see the value
        pv = torch.where(seen[..., None], p[..., None] * v[:, :, None], 0.0)
        out, mag = pv.sum(3), pv.abs().sum(3)
    return out.permute(2, 0, 1, 3).reshape(n, Hq, D), mag.permute(2, 0, 1, 3).reshape(n, Hq, D)
