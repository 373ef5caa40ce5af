"""The operators of a server whose requests share prompts and draft tokens, as they are measured: a batch packed on the
GPU from its requests' lengths, attention over prefixes that many sequences share, and drafted tokens verified.

Shapes are the framework's own (GPT-OSS-120B: 64 query and 8 kv heads of 64, 201,088 tokens, a window of 128) or generic.
K and V lie in slabs of 64-position blocks in the attention kernel's fragment order; ``_slots`` restates where an element
lies.  A sequence's slab holds what follows its prefix: position p is its slab's position p - (the prefix's length)."""
import math
import random

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16
HQ, HKV, D = 64, 8, 64
VOCAB = 201088
ONE = 2.0 ** 40


# ---- the cases ----------------------------------------------------------------------------------------

def listed():
    return [
        # a decode step's lengths: 24 streams, one token each
        {"name": "pack_24_streams", "op": "pack", "streams": 24, "q": 1, "prefix": 2000, "prefixes": 1, "alone": 0, "own": 300},
        # a deep queue of short drafts over many prompts
        {"name": "pack_4096_streams", "op": "pack", "streams": 4096, "q": 8, "prefix": 9000, "prefixes": 40, "alone": 100, "own": 2000},
        # two samples of one short prompt, one token each: latency
        {"name": "attn_2_streams", "op": "attn", "streams": 2, "q": 1, "prefix": 513, "prefixes": 1, "alone": 0, "own": 40, "window": 0},
        # a decode batch behind one system prompt
        {"name": "attn_48_streams", "op": "attn", "streams": 48, "q": 1, "prefix": 8000, "prefixes": 1, "alone": 0, "own": 300, "window": 0},
        # the same batch's sliding layers: the window reaches back into the prompt for the streams that began lately
        {"name": "attn_window_48", "op": "attn", "streams": 48, "q": 1, "prefix": 1500, "prefixes": 1, "alone": 0, "own": 200, "window": 128},
        # ragged verify rows of three prompts' streams, a few without a prompt among them
        {"name": "attn_drafts_3_prompts", "op": "attn", "streams": 32, "q": 8, "prefix": 16011, "prefixes": 3, "alone": 4, "own": 700, "window": 0},
        # new requests: long questions behind a shared prompt, fed at once
        {"name": "attn_questions", "op": "attn", "streams": 6, "q": 300, "prefix": 4099, "prefixes": 1, "alone": 0, "own": 0, "window": 0},
        # many samples of one long document, three drafted tokens each
        {"name": "attn_256_streams", "op": "attn", "streams": 256, "q": 4, "prefix": 32749, "prefixes": 1, "alone": 0, "own": 500, "window": 0},
        # one stream's four drafted tokens from a lookup (no distribution): latency
        {"name": "verify_1_stream", "op": "verify", "streams": 1, "drafts": 4, "vocab": VOCAB, "probs": "none", "params": "top_p"},
        # a batch whose requests each bring a temperature, top-k and top-p of their own
        {"name": "verify_24_mixed", "op": "verify", "streams": 24, "drafts": 4, "vocab": VOCAB, "probs": "none", "params": "mixed"},
        # ragged drafts of a draft model, its distributions with them
        {"name": "verify_32_ragged", "op": "verify", "streams": 32, "drafts": 7, "vocab": VOCAB, "probs": "some", "params": "mixed"},
        # many streams of eight drafts each, the plain distribution
        {"name": "verify_128_streams", "op": "verify", "streams": 128, "drafts": 8, "vocab": VOCAB, "probs": "all", "params": "plain"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("pack", "attn", "attn", "attn", "verify", "verify", "verify"))
    if op == "verify":
        return {"op": op, "streams": _log_int(rng, 1, 128), "drafts": rng.randint(1, 8),
                "vocab": rng.choice((VOCAB, _log_int(rng, 500, VOCAB))), "probs": rng.choice(("none", "some", "all")),
                "params": rng.choice(("plain", "top_p", "mixed", "mixed"))}
    streams = _log_int(rng, 1, 4096 if op == "pack" else 200)
    case = {"op": op, "streams": streams, "q": rng.choice((1, 1, rng.randint(2, 8))), "prefix": _log_int(rng, 50, 32000),
            "prefixes": rng.randint(1, 40 if op == "pack" else 3), "alone": rng.choice((0, 0, streams // 5)),
            "own": _log_int(rng, 1, 1000)}
    if op == "attn":
        case["window"] = rng.choice((0, 0, 0, 128, _log_int(rng, 1, 4000)))
        if rng.random() < 0.2:
            case.update(streams=rng.randint(1, 8), q=rng.randint(9, 300), alone=0, own=rng.choice((0, 100)), prefix=_log_int(rng, 50, 8000))
    return case


# ---- what a case's plan is (host values that a program has before the call) ---------------------------

def _round64(n):
    return (n + 63) // 64 * 64


def _requests(case):
    """(q_lens, starts, prefix of each sequence or -1, length of each prefix): uneven sequences, the prefixes dealt in turn."""
    rng = random.Random(case["streams"] * 131 + case["q"] * 7 + case["prefix"])
    S, n = case["streams"], case["prefixes"]
    lens = [max(1, case["prefix"] - 37 * i * (case["prefix"] // 500)) for i in range(n)]
    prefix = [-1 if i < case["alone"] else i % n for i in range(S)]
    rng.shuffle(prefix)
    q_lens = [rng.randint(max(1, case["q"] // 2 if case["q"] != 4 else 4), case["q"]) for _ in range(S)]
    starts = [(lens[p] if p >= 0 else 0) + rng.randint(0, case["own"]) for p in prefix]
    return q_lens, starts, prefix, lens


def _slabs(case):
    """(base and cap of the prefixes' slabs, of the sequences' slabs, elements of a pool)."""
    q_lens, _, prefix, lens = _requests(case)
    caps = [_round64(n) for n in lens] + [_round64(case["own"] + case["q"])] * case["streams"]
    bases = [0]
    for c in caps:
        bases.append(bases[-1] + HKV * c * D)
    n = len(lens)
    return (bases[:n], caps[:n]), (bases[n:-1], caps[n:]), bases[-1]


def _row_counts(case):
    """Logits rows of each stream: its drafted tokens and one more."""
    rng = random.Random(case["streams"] * 17 + case["drafts"])
    if case["probs"] == "some":
        return [1 + rng.randint(0, case["drafts"]) for _ in range(case["streams"])]
    return [1 + case["drafts"]] * case["streams"]


def _slots(pos, kind):
    """Element offsets [P, 64] of positions' rows of K or V within a kv head's region."""
    p, d = pos[:, None], torch.arange(D, device=pos.device)[None, :]
    q = p % 64
    block = (p // 64) * 4096
    if kind == "k":
        tile, n = 2 * (q // 32) + (q % 8) // 4, 4 * ((q % 32) // 8) + q % 4
        return block + tile * 1024 + (d // 32) * 512 + (16 * ((d % 32) // 8) + n) * 8 + d % 8
    return block + (q // 32) * 2048 + (d // 16) * 512 + (16 * ((q % 32) // 8) + d % 16) * 8 + q % 8


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _i64(v):
    return torch.tensor(v, dtype=torch.int64, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "verify":
        return _prepare_verify(case, g, s)
    q_lens, starts, prefix, lens = _requests(case)
    (pb, pc), (kb, kc), elems = _slabs(case)
    if case["op"] == "pack":  # other lengths for another seed
        starts = [a + seed % 50 for a in starts]
        kc = [c + 64 for c in kc]
        kb = [HKV * D * 64 * i for i in range(len(kb))]
    s.update(q_lens=_i32(q_lens), starts=_i32(starts), prefix_of=_i32(prefix), prefix_len=_i32(lens), prefix_base=_i64(pb),
             prefix_cap=_i32(pc), kv_base=_i64(kb), kv_cap=_i32(kc), tokens=sum(q_lens))
    if case["op"] == "attn":
        # queries and keys of a spread that gives scores of a few units, so that some keys count far more than others
        s.update(q=(torch.randn(sum(q_lens), HQ, D, device=DEV, generator=g) * 1.5).to(BF16),
                 k=torch.randn(elems, device=DEV, generator=g).to(BF16), v=torch.randn(elems, device=DEV, generator=g).to(BF16),
                 sinks=torch.randn(HQ, device=DEV, generator=g))
    return s


def _prepare_verify(case, g, s):
    V, S = case["vocab"], case["streams"]
    rows = _row_counts(case)
    R = sum(rows)
    cu = [0]
    for n in rows:
        cu.append(cu[-1] + n)
    rng = random.Random(S * 3 + V)
    pick = {"plain": lambda: (1.0, 0, 1.0), "top_p": lambda: (0.8, 0, 0.95),
            "mixed": lambda: rng.choice(((0.0, 0, 1.0), (0.6, 40, 1.0), (0.8, 0, 0.95), (1.0, 0, 1.0), (1.3, 200, 0.9)))}[case["params"]]
    params = [pick() for _ in range(S)]
    # a spread of unlikely tokens and a few dozen likely ones
    x = torch.randn(R, V, device=DEV, generator=g) * 2.0
    likely = torch.randint(0, V, (R, 64), device=DEV, generator=g)
    x.scatter_(1, likely, torch.randn(R, 64, device=DEV, generator=g) * 2.0 + 11.0)
    logits = x.to(BF16)
    # what the drafter thinks, near the target; the drafted token is drawn from it
    temp = torch.tensor([p[0] if p[0] > 0 else 1.0 for p in params], device=DEV).repeat_interleave(_i64(rows))
    x = (logits.float() + torch.randn(R, V, device=DEV, generator=g) * 0.6).div_(temp[:, None])
    drafts = torch.argmax(x - (-torch.rand(R, V, device=DEV, generator=g).clamp_(1e-12, 1 - 1e-7).log_()).log_(), 1)
    best = torch.argmax(logits.float(), 1)
    greedy = torch.tensor([p[0] <= 0 for p in params], device=DEV).repeat_interleave(_i64(rows))
    luck = torch.rand(R, device=DEV, generator=g) < (0.85 if case["probs"] == "none" else 0.0)
    drafts = torch.where(luck | (greedy & (torch.rand(R, device=DEV, generator=g) < 0.7)), best, drafts)
    last = _i64(cu[1:]) - 1
    drafts[last] = -1
    probs_row = torch.arange(R, device=DEV)
    probs_row[last] = -1
    if case["probs"] == "some":  # a third of the streams drafted by lookup
        probs_row[torch.arange(S, device=DEV).repeat_interleave(_i64(rows)) % 3 == 0] = -1
    has = probs_row >= 0
    s.update(logits=logits, cu_rows=_i32(cu), draft=drafts.to(torch.int32), rows=R,
             u=torch.rand(R, dtype=torch.float64, device=DEV, generator=g), u_draw=torch.rand(S, dtype=torch.float64, device=DEV, generator=g),
             temp=torch.tensor([p[0] for p in params], dtype=torch.float32, device=DEV), top_k=_i32([p[1] for p in params]),
             top_p=torch.tensor([p[2] for p in params], dtype=torch.float32, device=DEV), probs=None, probs_row=None)
    if case["probs"] != "none":  # the drafter's distributions, one row after the other
        s["probs"] = torch.softmax(x[has], 1)
        s["probs_row"] = torch.where(has, has.cumsum(0) - 1, -1).to(torch.int32)
    return s


# ---- one pass -----------------------------------------------------------------------------------------

def run(s):
    return {"pack": _pack, "attn": _attn, "verify": _verify}[s["case"]["op"]](s)


def _tokens(s):
    """(cu [S + 1], sequence of each token, place of each token in its sequence)."""
    S = s["q_lens"].numel()
    cu = torch.zeros(S + 1, dtype=torch.int64, device=DEV)
    cu[1:] = s["q_lens"].cumsum(0)
    seq = torch.repeat_interleave(torch.arange(S, device=DEV), s["q_lens"].long(), output_size=s["tokens"])
    return cu, seq, torch.arange(s["tokens"], device=DEV) - cu[seq]


def _pack(s):
    if own:
        from flyai_amd import ops
        b = ops.pack_shared(s["q_lens"], s["starts"], s["kv_base"], s["kv_cap"], s["prefix_of"], s["prefix_len"], D, s["tokens"])
        return tuple(b[n] for n in ("cu_seqlens", "positions", "seq_id", "kv_pos", "kv_slot", "kv_len", "status"))
    cu, seq, i = _tokens(s)
    behind = torch.where(s["prefix_of"] >= 0, s["prefix_len"][s["prefix_of"].clamp_min(0).long()], 0)
    positions = s["starts"][seq] + i
    kv_pos = positions - behind[seq]
    cap = s["kv_cap"][seq]
    fits = (kv_pos >= 0) & (kv_pos < cap)
    kv_slot = torch.where(fits, s["kv_base"][seq] + kv_pos * D, -1)
    kv_len = s["starts"] + s["q_lens"]
    status = (kv_len - behind > s["kv_cap"]).any().int().reshape(1)
    int32 = torch.int32
    return cu.to(int32), positions.to(int32), seq.to(int32), kv_pos.to(int32), kv_slot, kv_len, status


def _attn(s):
    c = s["case"]
    if own:
        from flyai_amd import ops
        plan = ops.attn_shared_plan(s["q_lens"], s["starts"], s["kv_base"], s["kv_cap"], s["prefix_of"], s["prefix_len"],
                                    s["prefix_base"], s["prefix_cap"], HKV, c["window"], s["tokens"], s["k"].numel())
        return ops.attn_shared(s["q"], s["k"], s["v"], s["sinks"], plan)
    T, S, n, window = s["tokens"], c["streams"], c["prefixes"], c["window"] or 2 ** 30
    _, seq, i = _tokens(s)
    mine = s["prefix_of"].long()[seq]                                                            # [T]
    behind = torch.where(mine >= 0, s["prefix_len"].long()[mine.clamp_min(0)], 0)
    at = s["starts"].long()[seq] + i
    q = s["q"].float().reshape(T, HKV, HQ // HKV, D) * D ** -0.5
    heads = torch.arange(HKV, device=DEV)[:, None, None]

    def gather(pool, base, cap, length, kind):  # [slabs, Hkv, length, D]
        off = _slots(torch.arange(length, device=DEV), kind)
        return pool[base[:, None, None, None] + heads * (cap.long() * D)[:, None, None, None] + off].float()

    P = c["prefix"]
    kp, vp = (gather(s[x], s["prefix_base"], s["prefix_cap"], _round64(P), x).transpose(0, 1).reshape(HKV, -1, D) for x in "kv")
    j = torch.arange(_round64(P), device=DEV)
    there = (j < s["prefix_len"][:, None]).reshape(-1)                                           # [n * P]
    owner = torch.arange(n, device=DEV)[:, None].expand(n, _round64(P)).reshape(-1)
    seen = there & (owner == mine[:, None]) & (j.repeat(n) > at[:, None] - window)               # [T, n * P]
    sp = torch.matmul(q.transpose(0, 1).reshape(HKV, -1, D), kp.transpose(1, 2)).reshape(HKV, T, HQ // HKV, -1)
    sp.masked_fill_(~seen[:, None, :], float("-inf"))
    L = int(c["own"] + c["q"])
    ko, vo = (gather(s[x], s["kv_base"], s["kv_cap"], L, x) for x in "kv")                       # [S, Hkv, L, D]
    qo = torch.zeros(S, c["q"], HKV, HQ // HKV, D, device=DEV)
    qo[seq, i] = q
    so = torch.matmul(qo.permute(0, 2, 1, 3, 4).reshape(S, HKV, -1, D), ko.transpose(2, 3)).reshape(S, HKV, c["q"], HQ // HKV, L)
    so = so.permute(0, 2, 1, 3, 4)[seq, i].transpose(0, 1)                                       # [Hkv, T, 8, L]
    p = behind[:, None] + torch.arange(L, device=DEV)
    so = so.masked_fill(~((p <= at[:, None]) & (p > at[:, None] - window))[:, None, :], float("-inf"))
    sink = s["sinks"].reshape(HKV, 1, HQ // HKV, 1)
    m = torch.maximum(torch.maximum(sp.amax(3, keepdim=True), so.amax(3, keepdim=True)), sink)
    sp.sub_(m).exp_()
    so = (so - m).exp()
    total = sp.sum(3, keepdim=True) + so.sum(3, keepdim=True) + (sink - m).exp()
    o = torch.matmul(sp.reshape(HKV, -1, sp.shape[3]), vp).reshape(HKV, T, HQ // HKV, D)
    po = torch.zeros(S, c["q"], HKV, HQ // HKV, L, device=DEV)
    po[seq, i] = so.transpose(0, 1)
    oo = torch.matmul(po.permute(0, 2, 1, 3, 4).reshape(S, HKV, -1, L), vo).reshape(S, HKV, c["q"], HQ // HKV, D)
    o = (o + oo.permute(0, 2, 1, 3, 4)[seq, i].transpose(0, 1)) / total
    return o.transpose(0, 1).reshape(T, HQ, D).to(BF16)


def _verify(s):
    if own:
        from flyai_amd import ops
        return ops.spec_verify(s["logits"], s["cu_rows"], s["draft"], s["u"], s["u_draw"], s["temp"], s["top_k"], s["top_p"],
                               draft_probs=s["probs"], probs_row=s["probs_row"])
    x = s["logits"].float()
    R, V = x.shape
    S = s["cu_rows"].numel() - 1
    cu = s["cu_rows"].long()
    seq = torch.repeat_interleave(torch.arange(S, device=DEV), cu[1:] - cu[:-1], output_size=R)
    rows = torch.arange(R, device=DEV)
    temp, top_k, top_p = s["temp"][seq][:, None], s["top_k"].long()[seq][:, None], s["top_p"].double()[seq][:, None]
    greedy = temp <= 0
    # the filtered weights in descending order of the logits, lower ids first among equals
    z, ids = torch.sort(x / temp.clamp_min(1e-6) + 0.0, dim=1, descending=True, stable=True)
    d = z.double() - z[:, :1].double()
    w = torch.where(d >= -27.75, (d.exp() * ONE).floor(), 0.0).long()
    kth = z.gather(1, torch.where((top_k > 0) & (top_k < V), top_k - 1, V - 1))
    w = w * (z >= kth)
    limit = (top_p * w.sum(1, keepdim=True).double()).floor().long()
    w = w * ((w.cumsum(1) - w <= limit) | (top_p <= 0) | (top_p >= 1))
    best = ids[:, 0]
    w = torch.zeros_like(w).scatter_(1, ids, w)
    W = w.sum(1)
    draft = s["draft"].long()
    there = (draft >= 0) & (draft < V)
    at = draft.clamp(0, V - 1)
    no_probs = s["probs"] is None
    of = torch.full((R,), -1, device=DEV) if no_probs else s["probs_row"].long()
    q_at = torch.ones(R, dtype=torch.float64, device=DEV) if no_probs else torch.where(of >= 0, s["probs"][of.clamp_min(0), at].double(), 1.0)
    accept = torch.where(greedy[:, 0], at == best, s["u"] * q_at * W.double() < w.gather(1, at[:, None])[:, 0].double()) & there
    # the first row of each stream that is not accepted (R: none is left)
    stop = torch.full((S,), R, device=DEV).scatter_reduce_(0, seq, torch.where(accept, R, rows), "amin")
    stops = stop < cu[1:]
    r = stop.clamp_max(R - 1)
    # what is left for the draw there
    left = w[r]
    q_full = torch.zeros(S, V, dtype=torch.float64, device=DEV) if no_probs else s["probs"][of[r].clamp_min(0)].double() * (of[r] >= 0)[:, None]
    taken = (q_full * W[r].double()[:, None]).floor().long()
    lone = there[r] & (of[r] < 0)
    taken = torch.where(torch.arange(V, device=DEV) == at[r][:, None], torch.where(lone, left.amax(1) + 1, taken.gather(1, at[r][:, None])[:, 0])[:, None], taken)
    rest = torch.where(there[r][:, None], (left - taken).clamp_min(0), left)
    run = rest.cumsum(1)
    total = run[:, -1]
    target = torch.minimum((s["u_draw"] * total.double()).long(), (total - 1).clamp_min(0))
    drawn = torch.searchsorted(run, target[:, None], right=True)[:, 0]
    drawn = torch.where(total > 0, drawn, torch.argmax((left == left.amax(1, keepdim=True)).int(), 1))
    drawn = torch.where(greedy[r, 0], best[r], drawn)
    tokens = torch.where(rows < stop[seq], draft, -1)
    tokens = torch.where(rows == stop[seq], drawn[seq], tokens)
    n = torch.where(stops, stop - cu[:-1] + 1, cu[1:] - cu[:-1])
    # the target's probability of each token that comes out
    p = torch.where(greedy[:, 0], 1.0, w.gather(1, tokens.clamp_min(0)[:, None])[:, 0].double() / W.double().clamp_min(1.0))
    return tokens.to(torch.int32), n.to(torch.int32), torch.where(tokens >= 0, p, 0.0).float()


# ---- what a pass cannot do without --------------------------------------------------------------------

def work(case):
    if case["op"] == "verify":
        R, V, S = sum(_row_counts(case)), case["vocab"], case["streams"]
        # every logits row; of the drafter's distributions the row that a stream stops at, and the drafted tokens'
        q = {"none": 0, "some": 2 / 3, "all": 1}[case["probs"]]
        return {"bytes": int(2 * R * V + 4 * S * V * q * 0.8), "flops": R * V}
    q_lens, starts, prefix, lens = _requests(case)
    T, S = sum(q_lens), len(q_lens)
    if case["op"] == "pack":
        return {"bytes": T * 20 + S * (4 + 4 + 4 + 4 + 8 + 4 + 4) + 4 * len(lens), "flops": T}
    window = case["window"] or 2 ** 30
    flops = keys = 0
    first = list(lens)  # of each prefix, the first position that is read
    for ql, st, p in zip(q_lens, starts, prefix):
        P = lens[p] if p >= 0 else 0
        if p >= 0:
            first[p] = min(first[p], max(0, st - window + 1))
        keys += st + ql - max(P, st - window + 1)
        flops += sum(min(window, st + i + 1) for i in range(ql))
    shared = sum(n - f for n, f in zip(lens, first))
    return {"bytes": (keys + shared) * HKV * D * 4 + T * HQ * D * 4, "flops": 4 * HQ * D * flops}


# ---- the definitions, in 64 bits ----------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"pack": _exact_pack, "attn": _exact_attn, "verify": _exact_verify}[case["op"]](case, s)


def _exact_pack(case, s):
    """Token by token, on the host."""
    q_lens, starts, prefix, lens = (s[n].tolist() for n in ("q_lens", "starts", "prefix_of", "prefix_len"))
    base, cap = s["kv_base"].tolist(), s["kv_cap"].tolist()
    cu, pos, sid, kpos, slot, over = [0], [], [], [], [], 0
    for b, n in enumerate(q_lens):
        P = lens[prefix[b]] if prefix[b] >= 0 else 0
        for i in range(n):
            p = starts[b] + i
            pos.append(p)
            sid.append(b)
            kpos.append(p - P)
            slot.append(base[b] + (p - P) * D if 0 <= p - P < cap[b] else -1)
        over |= starts[b] + n - P > cap[b]
        cu.append(cu[-1] + n)
    return tuple(torch.tensor(v) for v in (cu, pos, sid, kpos, slot, [a + n for a, n in zip(starts, q_lens)], [int(over)]))


def _dense(pool, base, cap, kind):
    """A slab's K or V as [kv head, position, dim], by the axes of the blocks: of K [tile pair, tile half, dim half, dim
    eighth, row group, row, dim], where a position of the block is (tile pair, row group, tile half, row); of V [half, dim
    sixteenth, key group, dim, key]."""
    b = pool[base:base + HKV * cap * D]
    if kind == "k":
        b = b.reshape(HKV, cap // 64, 2, 2, 2, 4, 4, 4, 8).permute(0, 1, 2, 6, 3, 7, 4, 5, 8)
    else:
        b = b.reshape(HKV, cap // 64, 2, 4, 4, 16, 8).permute(0, 1, 2, 4, 6, 3, 5)
    return b.reshape(HKV, cap, D).double()


def _exact_attn(case, s):
    """Sequence by sequence over its prefix and its own keys, one after the other."""
    q_lens, starts, prefix, lens = _requests(case)
    (pb, pc), (kb, kc), _ = _slabs(case)
    front = [[_dense(s[x], pb[i], pc[i], x)[:, :lens[i]] for x in "kv"] for i in range(len(lens))]
    sink = s["sinks"].double().reshape(HKV, HQ // HKV, 1, 1)
    out, t = [], 0
    for b, (n, st, p) in enumerate(zip(q_lens, starts, prefix)):
        k, v = (_dense(s[x], kb[b], kc[b], x)[:, :st + n - (lens[p] if p >= 0 else 0)] for x in "kv")
        if p >= 0:
            k, v = torch.cat((front[p][0], k), 1), torch.cat((front[p][1], v), 1)
        q = s["q"][t:t + n].double().permute(1, 0, 2).reshape(HKV, -1, D)
        score = (q @ k.transpose(1, 2) / 8).reshape(HKV, HQ // HKV, n, -1)
        at, j = torch.arange(st, st + n, device=DEV)[:, None], torch.arange(st + n, device=DEV)
        hidden = j > at
        if case["window"]:
            hidden = hidden | (j <= at - case["window"])
        score = torch.cat((score.masked_fill(hidden, float("-inf")), sink.expand(HKV, HQ // HKV, n, 1)), 3)
        w = torch.softmax(score, 3)[..., :-1]
        out.append((w.reshape(HKV, -1, st + n) @ v).reshape(HQ, n, D).transpose(0, 1))
        t += n
    return torch.cat(out)


def _exact_verify(case, s):
    """Stream by stream and row by row, over the distinct values of a row's logits and how often each is there."""
    V = case["vocab"]
    cu, draft, params = s["cu_rows"].tolist(), s["draft"].tolist(), [s[n].tolist() for n in ("temp", "top_k", "top_p")]
    u, u_draw = s["u"].tolist(), s["u_draw"].tolist()
    of = s["probs_row"].tolist() if s["probs"] is not None else [-1] * len(draft)
    tokens, counts, prob = [-1] * len(draft), [], [0.0] * len(draft)
    for b in range(len(cu) - 1):
        temp, k, top_p = (p[b] for p in params)
        n = 0
        for r in range(cu[b], cu[b + 1]):
            n += 1
            d = draft[r]
            if temp <= 0:
                best = int(torch.argmax(s["logits"][r].float()))
                tokens[r], prob[r] = best, 1.0
                if d == best:
                    continue
                break
            values, where, count = torch.unique(-(s["logits"][r].float() / max(temp, 1e-6)), return_inverse=True, return_counts=True)
            weight = torch.floor(torch.exp2(40 + (values[0].double() - values.double()) * (1 / math.log(2)))).long()
            weight[(values[0] - values) < -27.75] = 0
            if 0 < k < V:
                weight[count.cumsum(0) - count >= k] = 0
            kept = count.clone()
            if 0 < top_p < 1:
                limit = math.floor(top_p * float(int((weight * count).sum())))
                above = (weight * count).cumsum(0) - weight * count
                room = torch.where(weight > 0, torch.div(limit - above, weight.clamp_min(1), rounding_mode="floor") + 1, 0)
                kept = torch.where(above > limit, 0, torch.minimum(room, count))
            w = weight[where]
            cut = torch.nonzero((kept > 0) & (kept < count))
            w[kept[where] == 0] = 0
            if cut.numel():
                ties = torch.nonzero(where == cut[0, 0])[:, 0]
                w[ties[int(kept[cut[0, 0]]):]] = 0
            W = int(w.sum())
            q = s["probs"][of[r]].double() if of[r] >= 0 else None
            if d >= 0:
                if u[r] * (float(q[d]) if q is not None else 1.0) * W < int(w[d]):
                    tokens[r], prob[r] = d, int(w[d]) / W
                    continue
                if q is None:
                    rest = w.clone()
                    rest[d] = 0
                else:
                    rest = (w - torch.floor(q * W).long()).clamp_min(0)
            else:
                rest = w
            total = int(rest.sum())
            if total == 0:
                tokens[r] = int(torch.nonzero(w == w.max())[0, 0])
            else:
                tokens[r] = int(torch.nonzero(rest.cumsum(0) > min(int(u_draw[b] * total), total - 1))[0, 0])
            prob[r] = int(w[tokens[r]]) / W if W else 0.0
            break
        counts.append(n)
    return torch.tensor(tokens), torch.tensor(counts), torch.tensor(prob, dtype=torch.float64)
