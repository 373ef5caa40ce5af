"""Batches behind shared prefixes for the tests of ops.pack_shared and ops.attn_shared: built on the GPU, mirrored to the oracle."""
import torch

from flyai_amd import kvlayout, ops
from oracle import shared as oracle

DEV = "cuda"


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _round64(n):
    return max(64, (n + 63) // 64 * 64)


class Batch:
    """prefixes: their lengths; seqs: (q_len, positions of the own slab before it, prefix or -1).  Everything outside the
    positions that hold keys is NaN."""

    def __init__(self, prefixes, seqs, Hkv=2, seed=0, spread=1.0, extra_rows=0):
        g = torch.Generator().manual_seed(seed)
        self.prefixes, self.seqs, self.Hkv = prefixes, seqs, Hkv
        self.q_lens = [s[0] for s in seqs]
        self.behind = [prefixes[s[2]] if s[2] >= 0 else 0 for s in seqs]
        self.starts = [b + s[1] for b, s in zip(self.behind, seqs)]
        self.prefix_of = [s[2] for s in seqs]
        lens = [*prefixes, *(s[0] + s[1] for s in seqs)]
        self.caps = [_round64(n) for n in lens]
        self.bases = [0]
        for c in self.caps:
            self.bases.append(self.bases[-1] + Hkv * c * 64)
        self.elems = self.bases[-1]
        self.T = sum(self.q_lens) + extra_rows
        self.keys, self.values = [], []
        self.k = torch.full((self.elems,), float("nan"), dtype=torch.bfloat16)
        self.v = self.k.clone()
        for base, cap, n in zip(self.bases, self.caps, lens):
            k, v = ((torch.randn(Hkv, n, 64, generator=g) * spread).to(torch.bfloat16) for _ in "kv")
            self.keys.append(k)
            self.values.append(v)
            self._write(base, cap, n, k, v)
        self.k, self.v = self.k.to(DEV), self.v.to(DEV)
        self.q = (torch.randn(self.T, 8 * Hkv, 64, generator=g) * spread).to(torch.bfloat16)
        self.sinks = torch.randn(8 * Hkv, generator=g)

    def _write(self, base, cap, n, k, v):
        if n:
            end = base + self.Hkv * cap * 64
            kvlayout.scatter(self.k[base:end], self.Hkv, cap, "k", k, torch.arange(n))
            kvlayout.scatter(self.v[base:end], self.Hkv, cap, "v", v, torch.arange(n))

    def rewrite(self, slab):
        """The pools' copy of keys[slab] and values[slab] again, after a test changed them."""
        k, v = self.k.cpu(), self.v.cpu()
        self.k, self.v = k, v
        self._write(self.bases[slab], self.caps[slab], self.keys[slab].shape[1], self.keys[slab], self.values[slab])
        self.k, self.v = self.k.to(DEV), self.v.to(DEV)

    def lengths(self):
        n = len(self.prefixes)
        return dict(q_lens=_i32(self.q_lens), starts=_i32(self.starts), kv_base=torch.tensor(self.bases[n:-1], dtype=torch.int64, device=DEV),
                    kv_cap=_i32(self.caps[n:]), prefix_of=_i32(self.prefix_of), prefix_len=_i32(self.prefixes))

    def plan(self, window, **change):
        n = len(self.prefixes)
        args = dict(self.lengths(), prefix_base=torch.tensor(self.bases[:n], dtype=torch.int64, device=DEV), prefix_cap=_i32(self.caps[:n]),
                    n_kv_heads=self.Hkv, window=window, n_tokens=self.T, pool_elems=self.elems)
        args.update(change)
        return ops.attn_shared_plan(**args)

    def run(self, window, out=None, **change):
        plan = self.plan(window, **change)
        return ops.attn_shared(self.q.to(DEV), self.k, self.v, self.sinks.to(DEV), plan, out=out), plan

    def expected(self, window):
        """(out, sum of p |v|) fp64 [T, Hq, 64], rows of the sequences alone."""
        n, outs, mags, t = len(self.prefixes), [], [], 0
        for b, (ql, before, p) in enumerate(self.seqs):
            k, v = self.keys[n + b], self.values[n + b]
            if p >= 0:
                k, v = torch.cat((self.keys[p], k), 1), torch.cat((self.values[p], v), 1)
            o, m = oracle.attention(self.q[t:t + ql], k, v, self.starts[b], self.sinks, window)
            outs.append(o)
            mags.append(m)
            t += ql
        return torch.cat(outs), torch.cat(mags)


def check(got, want, mag):
    """P is rounded to bf16 (2^-8 of each at most) before the products and the row sum alike, the result once more: 2^-8 (sum p |v| +
    |out|) and 2^-8 |out|.  Scores, exponentials and sums in fp32 stay below 2^-12 of sum p |v| for the scores of these tests (|s| < 60:
    64 products' sum 64 * 2^-24 of sum |q k| / 8, and 2^-17 in the exponent)."""
    got = got.double().cpu()
    tol = 2.0 ** -8 * (mag + 2 * want.abs()) * 1.01 + 2.0 ** -12 * mag + 1e-30
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float(((got - want).abs() / tol).max()), torch.nonzero(bad)[:4].tolist())
