"""Drafted tokens of a stream verified against the target's filtered weights, with the drafter's distribution or without one.

``Sampler.accept`` (``phase0/specsample.py:79-107``) accepts a deterministic draft d with probability p(d) and draws the first
rejection from p without d; with a drafter's distribution q the rule of speculative sampling accepts with min(1, p(d) / q(d)) and
draws from max(0, p - q), restated here over the sampler's integer weights (``oracle/sampling.py``)."""
import math

import numpy as np

from . import sampling


def _uniform(u):
    return min(u, 1 - 2.0 ** -53) if u >= 0 else 0.0


def _draw(rest, w, u):
    cum = np.cumsum(rest, dtype=np.uint64)
    total = int(cum[-1])
    if total == 0:
        return int(np.argmax(w))
    return int(np.searchsorted(cum, np.uint64(min(int(_uniform(u) * float(total)), total - 1)), side="right"))


def stream(logits, draft, probs, temp, top_k, top_p, u, u_draw):
    """Rows logits[i] judge draft[i] (-1: none), drawn from probs[i] (None: no distribution).  Returns (tokens, p), as many as the stream got."""
    tokens, ps = [], []
    V = logits.shape[1]
    for i, x in enumerate(logits):
        d = draft[i] if 0 <= draft[i] < V else -1
        if temp <= 0:
            best = sampling.greedy(x)
            tokens.append(best)
            ps.append(1.0)
            if d != best:
                break
            continue
        w = sampling.weights(x, temp, top_k, top_p)
        W = int(w.sum(dtype=np.uint64))
        q = probs[i]
        qd = 1.0 if q is None else float(np.fmax(q[d], 0))  # (negative and NaN: 0)
        if d >= 0 and _uniform(u[i]) * qd * float(W) < float(int(w[d])):
            tokens.append(d)
            ps.append(float(int(w[d])) / float(W))
            continue
        rest = w.copy()
        if d >= 0 and q is None:
            rest[d] = 0
        elif d >= 0:
            taken = np.floor(np.fmax(q, 0).astype(np.float64) * float(W))
            rest = np.where(taken >= w.astype(np.float64), 0, w - np.minimum(taken, w.astype(np.float64)).astype(np.uint64)).astype(np.uint64)
        t = _draw(rest, w, u_draw)
        tokens.append(t)
        ps.append(float(int(w[t])) / float(W) if W else 0.0)
        break
    return tokens, ps
