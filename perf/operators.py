"""The operators of a step that serves many requests at once, as they are measured: low-rank adapters beside a shared
projection, rotary positions, and the cache's slabs copied and compacted.

Shapes are the framework's own (GPT-OSS-120B layers: hidden 2880, 64 query and 8 kv heads of 64) or generic.  Slabs hold
K and V in 64-position blocks in the attention kernel's fragment order; ``_slots`` restates where an element lies."""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16
HIDDEN, HQ, HKV, D = 2880, 64, 8, 64
# projection -> (in features, out features by segment): each segment of a fused projection has an A of its own
PROJ = {"qkv": (HIDDEN, (HQ * D, HKV * D, HKV * D)), "o": (HQ * D, (HIDDEN,))}
DTYPES = {"bf16": BF16, "fp16": torch.float16, "fp32": torch.float32}


# ---- the cases ----------------------------------------------------------------------------------------

def listed():
    return [
        # one user with an adapter of its own, one token: latency
        {"name": "lora_1_token", "op": "lora", "proj": "qkv", "rows": 1, "seqs": 1, "adapters": 1, "rank": 16},
        # a decode batch: 48 streams over a dozen adapters of several ranks, some streams with none
        {"name": "lora_48_streams", "op": "lora", "proj": "qkv", "rows": 48, "seqs": 48, "adapters": 12, "rank": 64},
        # ragged verify rows of 32 streams at the output projection
        {"name": "lora_155_rows", "op": "lora", "proj": "o", "rows": 155, "seqs": 32, "adapters": 7, "rank": 32},
        # a step with prompt chunks in it (the benchmark's prefill batch: 2048 + 48 rows)
        {"name": "lora_chunk_2096", "op": "lora", "proj": "qkv", "rows": 2096, "seqs": 49, "adapters": 12, "rank": 64},
        # q and k of a decode step, read in place of the fused projection's rows
        {"name": "rope_24_streams", "op": "rope", "tokens": 24, "heads": 72, "of": 80, "dim": 64, "rot": 64, "dtype": "bf16",
         "layout": "half", "inverse": False, "far": 131072},
        # a prompt whose heads are rotated in part, neighbouring dims paired
        {"name": "rope_part_3001", "op": "rope", "tokens": 3001, "heads": 32, "of": 32, "dim": 192, "rot": 64, "dtype": "fp16",
         "layout": "interleaved", "inverse": False, "far": 1000000},
        # the gradient of a long prompt's queries in 32 bits
        {"name": "rope_grad_8192", "op": "rope", "tokens": 8192, "heads": 64, "of": 64, "dim": 128, "rot": 128, "dtype": "fp32",
         "layout": "half", "inverse": True, "far": 16777216},
        # the accepted path of one stream's drafted tree, moved up behind its committed context
        {"name": "compact_tree", "op": "compact", "layers": 12, "slots": 1, "cap": 2048, "start": 1500, "keep": "tree", "rows": 6},
        # cache eviction: the first four positions and the latest part of a long context stay
        {"name": "compact_evict_4", "op": "compact", "layers": 8, "slots": 4, "cap": 8192, "start": 0, "keep": "ends", "rows": 2045},
        # scattered positions of a context stay, picked by their weight
        {"name": "compact_scattered", "op": "compact", "layers": 12, "slots": 2, "cap": 6000, "start": 0, "keep": "picked", "rows": 1501},
        # one more sample of a short prompt
        {"name": "fork_short", "op": "fork", "layers": 12, "lo": 0, "hi": 77, "cap": 1024, "copies": 1},
        # a prompt shared by four samples
        {"name": "fork_3001_by_4", "op": "fork", "layers": 18, "lo": 0, "hi": 3001, "cap": 3200, "copies": 4},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("lora", "lora", "rope", "rope", "compact", "fork"))
    if op == "lora":
        rows = _log_int(rng, 1, 2000)
        seqs = min(rows, _log_int(rng, 1, 64))
        return {"op": op, "proj": rng.choice(("qkv", "o")), "rows": rows, "seqs": seqs,
                "adapters": min(seqs, _log_int(rng, 1, 24)), "rank": rng.choice((16, 32, 48, 64))}
    if op == "rope":
        dim = rng.choice((64, 80, 96, 128, 192))
        heads = rng.randint(1, 48)
        return {"op": op, "tokens": _log_int(rng, 1, 8000), "heads": heads, "of": heads + rng.choice((0, 0, 8, 16)), "dim": dim,
                "rot": rng.choice((dim, dim, dim // 2, 32)), "dtype": rng.choice(("bf16", "fp16", "fp32")),
                "layout": rng.choice(("half", "interleaved")), "inverse": rng.random() < 0.3, "far": _log_int(rng, 4096, 100000000)}
    if op == "compact":
        cap = _log_int(rng, 256, 8000)
        keep = rng.choice(("tree", "ends", "picked"))
        rows = rng.randint(2, 9) if keep == "tree" else _log_int(rng, 8, cap // 4)
        return {"op": op, "layers": rng.randint(1, 12), "slots": rng.randint(1, 4), "cap": cap,
                "start": rng.randint(0, cap - 100) if keep == "tree" else 0, "keep": keep, "rows": rows}
    hi = _log_int(rng, 1, 4000)
    return {"op": op, "layers": rng.randint(1, 18), "lo": rng.choice((0, 0, rng.randint(0, hi - 1))), "hi": hi,
            "cap": hi + rng.randint(0, 300), "copies": rng.randint(1, 4)}


# ---- what a case's plan is (host values that a program has before the call) ---------------------------

def _lora_plan(case):
    """(q_lens, adapter of each sequence, rank of each adapter): uneven sequences, every adapter in use, ranks R, R/2, R/4."""
    rng = random.Random(case["rows"] * 131 + case["seqs"])
    rows, seqs, n = case["rows"], case["seqs"], case["adapters"]
    if rows >= 4 * seqs:  # one long prompt chunk beside short rows
        q_lens = [1 + (i % 4) for i in range(seqs - 1)]
    else:
        cuts = sorted(rng.sample(range(1, rows), seqs - 1))
        q_lens = [b - a for a, b in zip([0] + cuts, cuts)]
    q_lens.append(rows - sum(q_lens))
    adapter = [i % (n + 1) if i % (n + 1) < n else -1 for i in range(seqs)]
    return q_lens, adapter, [max(1, case["rank"] >> (a % 3)) for a in range(n)]


def _keep(case, slot):
    """The positions (from start) that stay, ascending, first the place each goes to: place i takes position keep[i].
    A position that stays where it is apart, none lies among the places, so that a second pass changes nothing."""
    rng = random.Random(case["cap"] * 17 + case["rows"] * 5 + slot)
    n, length = case["rows"], case["cap"] - case["start"] - 13 * slot
    if case["keep"] == "tree":  # node 0, then one node of each level of a tree eight or more wide
        width = max(8, n)
        return [0] + [1 + (lv - 1) * width + (rng.randrange(width) if lv > 1 else 0) for lv in range(1, n)]
    if case["keep"] == "ends":
        n -= slot
        return list(range(4)) + list(range(length - n + 4, length))
    return list(range(4)) + sorted(rng.sample(range(n, length), n - 4))


def _round64(n):
    return (n + 63) // 64 * 64


def _slots(pos, kind):
    """Element offsets [P, 64] of positions' rows of K or V within a kv head's region."""
    p, d = pos[:, None], torch.arange(D, device=pos.device)[None, :]
    q = p % 64
    block = (p // 64) * 4096
    if kind == "k":
        tile, n = 2 * (q // 32) + (q % 8) // 4, 4 * ((q % 32) // 8) + q % 4
        return block + tile * 1024 + (d // 32) * 512 + (16 * ((d % 32) // 8) + n) * 8 + d % 8
    return block + (q // 32) * 2048 + (d // 16) * 512 + (16 * ((q % 32) // 8) + d % 16) * 8 + q % 8


def _normal(g, shape, scale=1.0, dtype=BF16):
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "lora":
        K, seg = PROJ[case["proj"]]
        N, n, R = sum(seg), case["adapters"], case["rank"]
        q_lens, adapter, ranks = _lora_plan(case)
        s.update(x=_normal(g, (case["rows"], K)), w=_normal(g, (N, K), 0.02), b=_normal(g, (N,), 0.02), segments=seg,
                 lora_a=_normal(g, (n, len(seg) * R, K), 0.02), lora_b=_normal(g, (n, N, R), 0.02),
                 scale=torch.rand(n, device=DEV, generator=g) * 1.5 + 0.5,
                 ranks=torch.tensor(ranks, dtype=torch.int32, device=DEV),
                 adapter=torch.tensor(adapter, dtype=torch.int32, device=DEV),
                 row_seq=torch.tensor(np.repeat(np.arange(len(q_lens)), q_lens), dtype=torch.int32, device=DEV),
                 # the segment of each output feature
                 seg_of=torch.tensor(np.repeat(np.arange(len(seg)), seg), device=DEV))
    elif case["op"] == "rope":
        T, rot = case["tokens"], case["rot"]
        rows = _normal(g, (T, case["of"], case["dim"]), dtype=DTYPES[case["dtype"]])
        start = int(torch.randint(0, case["far"] - T + 1, (1,), device=DEV, generator=g)) if case["far"] > T else 0
        s.update(x=rows[:, :case["heads"]], positions=torch.arange(start, start + T, dtype=torch.int32, device=DEV),
                 inv_freq=150000.0 ** (torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / -rot))
    else:
        n = 1 + case["copies"] if case["op"] == "fork" else case["slots"]
        cap = _round64(case["cap"])
        slab = HKV * cap * D
        s.update(k=_normal(g, (case["layers"], n * slab)), v=_normal(g, (case["layers"], n * slab)),
                 slabs=[(i * slab, cap) for i in range(n)])
        if case["op"] == "compact":
            s["keep"] = [_keep(case, i) for i in range(n)]
    return s


# ---- one pass -----------------------------------------------------------------------------------------

def run(s):
    return {"lora": _lora, "rope": _rope, "compact": _compact, "fork": _fork}[s["case"]["op"]](s)


def _lora(s):
    if own:
        from flyai_amd import ops
        return ops.linear_lora(s["x"], s["w"], s["b"], s["lora_a"], s["lora_b"], s["scale"], s["ranks"], s["adapter"],
                               segments=s["segments"], row_seq=s["row_seq"])
    x, a, b = s["x"].float(), s["lora_a"].float(), s["lora_b"].float()
    n, N, R = b.shape
    S = len(s["segments"])
    ids = torch.arange(n, device=DEV)
    mine = (s["adapter"].long()[s["row_seq"].long()][:, None] == ids) * s["scale"]                 # [M, n]
    live = torch.arange(R, device=DEV) < s["ranks"][:, None]                                       # [n, R]
    h = (x @ a.reshape(n * S * R, -1).t()).reshape(-1, n, S, R) * (mine[:, :, None] * live)[:, :, None]
    there = s["seg_of"] == torch.arange(S, device=DEV)[:, None]                                    # [S, N]
    up = b.transpose(1, 2)[:, None] * there[:, None]                                               # [n, S, R, N]
    y = x @ s["w"].float().t() + h.reshape(-1, n * S * R) @ up.reshape(n * S * R, N) + s["b"].float()
    return y.to(BF16)


def _rope(s):
    c = s["case"]
    if own:
        from flyai_amd import ops
        return ops.rope(s["x"], s["positions"], s["inv_freq"], layout=c["layout"], inverse=c["inverse"])
    x, rot = s["x"].float(), c["rot"]
    angle = s["positions"].double()[:, None] * s["inv_freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    sin = -sin if c["inverse"] else sin
    out = x.clone()
    first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if c["layout"] == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    out[..., first] = x[..., first] * cos - x[..., second] * sin
    out[..., second] = x[..., second] * cos + x[..., first] * sin
    return out.to(s["x"].dtype)


def _elements(slab, positions, kind):
    """Where positions' rows of every kv head of a slab lie in a layer's pool."""
    base, cap = slab
    heads = torch.arange(HKV, device=DEV)[:, None, None] * (cap * D)
    return (base + heads + _slots(positions, kind)).reshape(-1)


def _compact(s):
    c = s["case"]
    if own:
        from flyai_amd import ops
        moves = [(base, cap, c["start"], keep) for (base, cap), keep in zip(s["slabs"], s["keep"])]
        ops.kv_compact(s["k"], s["v"], HKV, moves)
        return s["k"], s["v"]
    keep = [torch.tensor(k, device=DEV) for k in s["keep"]]
    to = [c["start"] + torch.arange(len(k), device=DEV) for k in keep]
    src = {kind: torch.cat([_elements(b, c["start"] + k, kind) for b, k in zip(s["slabs"], keep)]) for kind in "kv"}
    dst = {kind: torch.cat([_elements(b, t, kind) for b, t in zip(s["slabs"], to)]) for kind in "kv"}
    s["k"][:, dst["k"]] = s["k"][:, src["k"]]
    s["v"][:, dst["v"]] = s["v"][:, src["v"]]
    return s["k"], s["v"]


def _fork(s):
    c = s["case"]
    if own:
        from flyai_amd import ops
        ops.kv_fork(s["k"], s["v"], HKV, s["slabs"][0], s["slabs"][1:], c["lo"], c["hi"])
        return s["k"], s["v"]
    pos = torch.arange(c["lo"], c["hi"], device=DEV)
    src = {kind: _elements(s["slabs"][0], pos, kind) for kind in "kv"}
    dst = {kind: torch.stack([_elements(b, pos, kind) for b in s["slabs"][1:]]) for kind in "kv"}
    s["k"][:, dst["k"]] = s["k"][:, src["k"]][:, None]
    s["v"][:, dst["v"]] = s["v"][:, src["v"]][:, None]
    return s["k"], s["v"]


# ---- what a pass cannot do without --------------------------------------------------------------------

def work(case):
    if case["op"] == "lora":
        K, seg = PROJ[case["proj"]]
        M, N, S = case["rows"], sum(seg), len(seg)
        q_lens, adapter, ranks = _lora_plan(case)
        used = sum(ranks[a] for a in set(adapter) if a >= 0)
        row_ranks = sum(q * ranks[a] for q, a in zip(q_lens, adapter) if a >= 0)
        return {"bytes": 2 * (M * K + N * K + N + used * (S * K + N) + M * N),
                "flops": 2 * M * N * K + 2 * row_ranks * (S * K + N)}
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2 * n * case["dim"] * DTYPES[case["dtype"]].itemsize, "flops": 3 * n * case["rot"]}
    row = 2 * case["layers"] * HKV * D * 2  # a position's K and V, every layer and kv head
    if case["op"] == "fork":
        return {"bytes": (1 + case["copies"]) * (case["hi"] - case["lo"]) * row, "flops": 0}
    moved = sum(p != i for slot in range(case["slots"]) for i, p in enumerate(_keep(case, slot)))
    return {"bytes": 2 * moved * row, "flops": 0}


# ---- the definitions, in 64 bits ----------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"lora": _exact_lora, "rope": _exact_rope}.get(case["op"], _exact_cache)(case, s)


def _exact_lora(case, s):
    """Sequence by sequence and segment by segment, over a's own rank alone."""
    q_lens, adapter, ranks = _lora_plan(case)
    R = case["rank"]
    x, w = s["x"].double(), s["w"].double()
    y = torch.nn.functional.linear(x, w) + s["b"].double()
    t = 0
    for q, a in zip(q_lens, adapter):
        col = 0
        for i, width in enumerate(s["segments"] if a >= 0 else ()):
            r = ranks[a]
            down = s["lora_a"][a, i * R:i * R + r].double()
            up = s["lora_b"][a, col:col + width, :r].double()
            y[t:t + q, col:col + width] += s["scale"][a].double() * ((x[t:t + q] @ down.t()) @ up.t())
            col += width
        t += q
    return y


def _exact_rope(case, s):
    """Pairs as complex numbers, turned by e^(i angle)."""
    rot = case["rot"]
    x = s["x"].double()
    part = x[..., :rot].contiguous()
    if case["layout"] == "half":
        part = torch.stack((part[..., :rot // 2], part[..., rot // 2:]), -1).contiguous()
    else:
        part = part.reshape(*part.shape[:-1], rot // 2, 2)
    angle = torch.outer(s["positions"].double(), s["inv_freq"]) * (-1 if case["inverse"] else 1)
    turned = torch.view_as_real(torch.view_as_complex(part) * torch.polar(torch.ones_like(angle), angle)[:, None])
    turned = torch.cat((turned[..., 0], turned[..., 1]), -1) if case["layout"] == "half" else turned.flatten(-2)
    return torch.cat((turned, x[..., rot:]), -1)


def _dense(pool, cap, kind):
    """A copy of a layer's pool as [slab, kv head, position, dim], by the axes of the blocks: of K [tile pair, tile half,
    dim half, dim eighth, row group, row, dim], where a position of the block is (tile pair, row group, tile half, row);
    of V [half, dim sixteenth, key group, dim, key]."""
    if kind == "k":
        b = pool.reshape(-1, HKV, cap // 64, 2, 2, 2, 4, 4, 4, 8)
        return b.permute(0, 1, 2, 3, 7, 4, 8, 5, 6, 9).reshape(-1, HKV, cap, D)
    b = pool.reshape(-1, HKV, cap // 64, 2, 4, 4, 16, 8)
    return b.permute(0, 1, 2, 3, 5, 7, 4, 6).reshape(-1, HKV, cap, D)


def _undense(rows, cap, kind):
    if kind == "k":
        b = rows.reshape(-1, HKV, cap // 64, 2, 4, 2, 4, 2, 4, 8)
        return b.permute(0, 1, 2, 3, 5, 7, 8, 4, 6, 9).reshape(-1)
    b = rows.reshape(-1, HKV, cap // 64, 2, 4, 8, 4, 16)
    return b.permute(0, 1, 2, 3, 6, 4, 7, 5).reshape(-1)


def _exact_cache(case, s):
    cap = s["slabs"][0][1]
    out = []
    for kind in "kv":
        layers = []
        for pool in s[kind]:
            rows = _dense(pool, cap, kind).clone()
            old = rows.clone()
            if case["op"] == "fork":
                rows[1:, :, case["lo"]:case["hi"]] = old[0, :, case["lo"]:case["hi"]]
            else:
                for i, keep in enumerate(s["keep"]):
                    rows[i, :, case["start"]:case["start"] + len(keep)] = old[i][:, [case["start"] + p for p in keep]]
            layers.append(_undense(rows, cap, kind))
        out.append(torch.stack(layers).double())
    return tuple(out)
