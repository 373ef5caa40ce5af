// Attention of a batch whose sequences share prefixes.
//
// A prefix's K/V lies in one slab, what follows it in each sequence's own.  Row (t, h) at position p of a sequence behind a
// prefix of P positions sees the prefix's keys [lo, P) and its own slab's [max(lo - P, 0), p - P], lo = max(0, p - window + 1)
// or 0; the softmax runs over both and the head's sink.  The rows of all the prefix's sequences are taken together, so
// its keys are read once per tile of rows, not once per sequence.
//
// Every key range is cut into chunks whose borders go by the slab alone (from its position 0).  A chunk's
// (m, l, O[64]) starts afresh, and a range's total folds its chunks in ascending order (fold below):
//   M' = max(M, m);  O' = O_c 2^(m - M') + O 2^(M - M');  L likewise.
// A work item takes either one chunk or all of them: the items' records are folded by attn_shared_merge_kernel, or the item folds in
// its registers, by the same operations in the same order.  So the work is split where there are few rows
// and not where there are many, and a row's bits depend on neither, nor on the rest of the batch.
//
// The work lists are made on the GPU (attn_shared_plan_kernel), once for a step's layers: the host needs
// no lengths, only bounds, and the grids are sized by those.
#include "attn.h"

namespace flyai {

constexpr int kShRowTokens = 16;      // tokens of a prefix item's tile (4 waves x 2 tiles of 16 rows x 2 tokens)
constexpr int kShWaveTokens = 4;      // tokens of a wave item
constexpr int kShMaxSeqs = 8192, kShMaxPrefixes = 1024;
constexpr int kShChunks = 16;         // a prefix's chunks: at most this many
constexpr int kShMinChunk = 128;
constexpr int kShOwnChunk = 512;
constexpr int kShSpareEntries = 1024;  // list entries beyond one for each tile, for prefixes split by chunks
constexpr int kShSpareWaves = 2048;    // ... and beyond one for each group of a sequence's tokens
constexpr int kShSpareRecs = 8192;     // records beyond two for each token
constexpr int kShGrid = 512;           // workgroups on the chip at once: two a CU

// What an item reads and where it writes.  Its rows are `ntok` tokens: from `first` on in the list of a prefix's tokens (list),
// or token first + i at the slab's position pos0 + i.
struct ShEntry {
  int64_t base;   // of the slab
  int32_t cap;
  int32_t first;
  int32_t ntok;
  int32_t pos0;
  int32_t list;
  int32_t key_lo, key_hi;  // slab positions
  int32_t chunk;           // positions of a chunk
  int32_t rec;             // record of the first token; token i's is rec + i
  int32_t pad;
};

struct ShToken {  // where a token's records lie: n of them, stride apart
  int32_t p_rec, p_n, p_stride;
  int32_t o_rec, o_n, o_stride;
};

struct ShHeader {
  int32_t n_entries, n_waves, n_tokens, status;
  int32_t window, pad[11];
};

// Byte layout of a plan, and how much each list holds at most.
struct ShLayout {
  int32_t T, max_entries, max_waves, max_recs;
  size_t o_entries, o_waves, o_list, o_tokens, bytes;
};

__host__ __device__ inline ShLayout sh_layout(int T, int S, int n_prefix) {
  ShLayout l;
  l.T = T;
  l.max_entries = T / kShRowTokens + (n_prefix < T ? n_prefix : T) + kShSpareEntries;
  // a sequence's groups, and the prefixes whose few tokens go to waves
  l.max_waves = T / kShWaveTokens + (S < T ? S : T) + (n_prefix < T ? n_prefix : T) + kShSpareWaves;
  l.max_recs = 2 * T + kShSpareRecs;
  size_t o = sizeof(ShHeader);
  l.o_entries = o;
  o += (size_t)l.max_entries * sizeof(ShEntry);
  l.o_waves = o;
  o += (size_t)l.max_waves * sizeof(ShEntry);
  l.o_list = o;
  o += (size_t)T * 8;
  l.o_tokens = o;
  o += (size_t)T * sizeof(ShToken);
  l.bytes = (o + 255) & ~(size_t)255;
  return l;
}

// ---- the plan -------------------------------------------------------------------------------------

constexpr int kShPlanThreads = 1024;

template <class T>
__device__ __forceinline__ T sh_excl_scan(T v, T* red, T* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T incl = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T y = __shfl_up(incl, o, 64);
    if (lane >= o) incl += y;
  }
  __syncthreads();  // the last use of red is over
  if (lane == 63) red[wave] = incl;
  __syncthreads();
  T sums = lane < kShPlanThreads / 64 ? red[lane] : (T)0;
#pragma unroll
  for (int o = 1; o < kShPlanThreads / 64; o <<= 1) {
    const T y = __shfl_up(sums, o, 64);
    if (lane >= o) sums += y;
  }
  *total = __shfl(sums, kShPlanThreads / 64 - 1, 64);
  const T base = wave ? __shfl(sums, wave - 1, 64) : (T)0;
  return base + incl - v;
}

__device__ __forceinline__ int sh_prefix_chunk(int P) {
  const int c = ((P + kShChunks - 1) / kShChunks + 63) & ~63;
  return c > kShMinChunk ? c : kShMinChunk;
}

struct ShBatch {
  const int32_t *q_lens, *starts;
  const int64_t* kv_base;
  const int32_t *kv_cap, *prefix_of, *prefix_len;
  const int64_t* prefix_base;
  const int32_t* prefix_cap;
  int S, n_prefix, Hkv, window, T;
  int64_t pool_elems;
};

// Bits of the status word
enum { kShPastSlab = 1, kShPastTokens = 2, kShBeforePrefix = 4, kShBadPrefix = 8, kShBadSequence = 16 };

__device__ __forceinline__ bool sh_slab_ok(int64_t base, int cap, int Hkv, int64_t pool) {
  return cap > 0 && cap % 64 == 0 && base >= 0 && base % 8 == 0 && base <= pool - (int64_t)Hkv * cap * 64;
}

// One workgroup.  Sequences, then prefixes are counted and scanned in LDS, then the lists are written token by token and entry by
// entry.  A prefix's tokens are listed in the order in which its sequences' counts arrive at an LDS counter: which rows share
// a tile may change from launch to launch, a row's result does not (no row's steps depend on its tile mates).
__global__ __launch_bounds__(kShPlanThreads) void attn_shared_plan_kernel(ShBatch b, char* __restrict__ plan) {
  const ShLayout L = sh_layout(b.T, b.S, b.n_prefix);
  ShHeader* hdr = reinterpret_cast<ShHeader*>(plan);
  ShEntry* entries = reinterpret_cast<ShEntry*>(plan + L.o_entries);
  ShEntry* waves = reinterpret_cast<ShEntry*>(plan + L.o_waves);
  int2* list = reinterpret_cast<int2*>(plan + L.o_list);
  ShToken* tokens = reinterpret_cast<ShToken*>(plan + L.o_tokens);
  __shared__ int32_t cu_s[kShMaxSeqs + 1];    // first token of each sequence
  __shared__ int32_t place_s[kShMaxSeqs];     // of its first listed token among its prefix's
  __shared__ int32_t wbase_s[kShMaxSeqs];     // its first wave entry
  __shared__ int32_t pcnt_s[kShMaxPrefixes];  // listed tokens of a prefix
  __shared__ int32_t plo_s[kShMaxPrefixes];   // the first of its positions that any of them sees
  __shared__ int32_t plist_s[kShMaxPrefixes], pent_s[kShMaxPrefixes], prec_s[kShMaxPrefixes];
  __shared__ int64_t red[kShPlanThreads / 64];
  __shared__ int32_t status_s;
  const int tid = threadIdx.x;
  if (tid == 0) status_s = 0;
  for (int p = tid; p < b.n_prefix; p += kShPlanThreads) {
    pcnt_s[p] = 0;
    plo_s[p] = INT32_MAX;
  }
  __syncthreads();
  int32_t status = 0;
  const int per = (b.S + kShPlanThreads - 1) / kShPlanThreads;
  const int s0 = min(b.S, tid * per), s1 = min(b.S, s0 + per);

  int64_t local = 0, total;
#pragma unroll 1
  for (int s = s0; s < s1; ++s) local += max(b.q_lens[s], 0);
  int64_t run = sh_excl_scan(local, red, &total);
  if (total > b.T) status |= kShPastTokens;
  // a sequence as it counts: no tokens where anything about it is out of bounds
  struct Seq {
    int q, P, own0;  // tokens, positions before its own slab's, the first token's slab position
    int p;           // its prefix, if its tokens see any of it
  };
  auto seq_of = [&](int s, int64_t first, int32_t* st) __attribute__((always_inline)) {
    Seq r = {0, 0, 0, -1};
    const int q = b.q_lens[s], start = b.starts[s], p = b.prefix_of[s];
    if (q < 0 || start < 0) *st |= kShBadSequence;
    if (q <= 0 || start < 0 || first + q > b.T) return r;
    int P = 0;
    if (p >= 0) {
      if (p >= b.n_prefix) { *st |= kShBadPrefix; return r; }
      P = b.prefix_len[p];
      if (P < 0 || P > b.prefix_cap[p] || !sh_slab_ok(b.prefix_base[p], b.prefix_cap[p], b.Hkv, b.pool_elems)) { *st |= kShBadPrefix; return r; }
    }
    if (start < P) { *st |= kShBeforePrefix; return r; }
    if (!sh_slab_ok(b.kv_base[s], b.kv_cap[s], b.Hkv, b.pool_elems)) { *st |= kShBadSequence; return r; }
    if ((int64_t)start - P + q > b.kv_cap[s]) { *st |= kShPastSlab; return r; }
    r.q = q;
    r.P = P;
    r.own0 = start - P;
    r.p = p;
    return r;
  };
  // the tokens of a sequence that see its prefix: the first of them, those below P + window - 1
  auto listed = [&](const Seq& r) __attribute__((always_inline)) {
    if (r.p < 0 || r.P == 0) return 0;
    return b.window > 0 ? (int)min((int64_t)r.q, max((int64_t)0, (int64_t)b.window - 1 - r.own0)) : r.q;
  };
  // the first chunk and the number of chunks of its own keys
  auto own_chunks = [&](const Seq& r, int* c0) __attribute__((always_inline)) {
    *c0 = b.window > 0 ? max(0, r.own0 - b.window + 1) / kShOwnChunk : 0;
    return (r.own0 + r.q - 1) / kShOwnChunk + 1 - *c0;
  };
  auto groups_of = [](int q) { return (q + kShWaveTokens - 1) / kShWaveTokens; };

  // groups of tokens; wave entries and records if the sequences' keys are split by chunks
  int64_t my_groups = 0, my_split = 0, my_recs = 0;
#pragma unroll 1
  for (int s = s0; s < s1; ++s) {
    cu_s[s] = (int)min(run, (int64_t)INT32_MAX);
    const Seq r = seq_of(s, run, &status);
    if (r.q > 0) {
      const int n = listed(r);
      if (n > 0) {
        place_s[s] = atomicAdd(&pcnt_s[r.p], n);
        atomicMin(&plo_s[r.p], b.window > 0 ? max(0, r.P + r.own0 - b.window + 1) : 0);
      }
      int c0;
      const int nch = own_chunks(r, &c0);
      my_groups += groups_of(r.q);
      my_split += (int64_t)groups_of(r.q) * nch;
      my_recs += (int64_t)r.q * nch;
    }
    run += max(b.q_lens[s], 0);
  }
  if (s1 == b.S && s0 < s1) cu_s[b.S] = (int)min(run, (int64_t)INT32_MAX);
  int64_t n_groups, split_entries, split_recs;
  sh_excl_scan(my_groups, red, &n_groups);
  sh_excl_scan(my_split, red, &split_entries);
  sh_excl_scan(my_recs, red, &split_recs);  // (its barriers also end the counting)

  // the prefixes: tiles, entries, records
  const int pper = (b.n_prefix + kShPlanThreads - 1) / kShPlanThreads;
  const int p0 = min(b.n_prefix, tid * pper), p1 = min(b.n_prefix, p0 + pper);
  auto chunks_of = [&](int p, int* c0) __attribute__((always_inline)) {
    const int P = b.prefix_len[p], C = sh_prefix_chunk(P);
    *c0 = plo_s[p] / C;
    return (P - 1) / C + 1 - *c0;
  };
  int64_t my_list = 0, my_tiles = 0, my_parts = 0, my_prec = 0, my_few = 0, my_few_parts = 0;
#pragma unroll 1
  for (int p = p0; p < p1; ++p) {
    const int n = pcnt_s[p];
    if (!n) continue;
    int c0;
    const int nch = chunks_of(p, &c0);
    const bool few = n <= kShWaveTokens;
    const int tiles = few ? 1 : (n + kShRowTokens - 1) / kShRowTokens;
    my_list += n;
    (few ? my_few : my_tiles) += tiles;
    (few ? my_few_parts : my_parts) += (int64_t)tiles * nch;
    my_prec += (int64_t)n * nch;
  }
  int64_t n_list, n_tiles, n_parts, n_prec, n_few, n_few_parts;
  const int64_t list0 = sh_excl_scan(my_list, red, &n_list);
  sh_excl_scan(my_tiles, red, &n_tiles);
  sh_excl_scan(my_parts, red, &n_parts);
  sh_excl_scan(my_prec, red, &n_prec);
  sh_excl_scan(my_few, red, &n_few);
  sh_excl_scan(my_few_parts, red, &n_few_parts);
  // Few tiles leave the chip idle: a chunk an item then, as far as the lists and the records hold them.
  const bool psplit = n_tiles * b.Hkv < kShGrid && n_parts <= L.max_entries && n_prec + b.T <= L.max_recs &&
                      n_few_parts + n_groups <= L.max_waves;
  const int64_t precs = psplit ? n_prec : n_list;
  const int64_t few_waves = psplit ? n_few_parts : n_few;
  const bool osplit = split_entries * b.Hkv < 8 * kShGrid && few_waves + split_entries <= L.max_waves &&
                      precs + split_recs <= L.max_recs;
  {
    int64_t e = 0, r = 0, f = 0, tot;
#pragma unroll 1
    for (int p = p0; p < p1; ++p) {
      const int n = pcnt_s[p];
      if (!n) continue;
      int c0;
      const int nch = psplit ? chunks_of(p, &c0) : 1;
      if (n <= kShWaveTokens) f += nch;
      else e += (int64_t)((n + kShRowTokens - 1) / kShRowTokens) * nch;
      r += (int64_t)n * nch;
    }
    int64_t e0 = sh_excl_scan(e, red, &tot), r0 = sh_excl_scan(r, red, &tot), f0 = sh_excl_scan(f, red, &tot), l0 = list0;
#pragma unroll 1
    for (int p = p0; p < p1; ++p) {
      const int n = pcnt_s[p];
      if (!n) continue;
      int c0;
      const int nch = psplit ? chunks_of(p, &c0) : 1;
      const bool few = n <= kShWaveTokens;
      plist_s[p] = (int)l0;
      prec_s[p] = (int)r0;
      pent_s[p] = (int)(few ? f0 : e0);
      l0 += n;
      r0 += (int64_t)n * nch;
      if (few) f0 += nch;
      else e0 += (int64_t)((n + kShRowTokens - 1) / kShRowTokens) * nch;
    }
  }
  // the sequences' wave entries and records
  int64_t my_w = 0, my_r = 0, tot_w, tot_r;
#pragma unroll 1
  for (int s = s0; s < s1; ++s) {
    int32_t ignore = 0;
    const Seq r = seq_of(s, cu_s[s], &ignore);
    if (!r.q) continue;
    int c0;
    const int nch = osplit ? own_chunks(r, &c0) : 1;
    my_w += (int64_t)groups_of(r.q) * nch;
    my_r += (int64_t)r.q * nch;
  }
  int64_t w0 = few_waves + sh_excl_scan(my_w, red, &tot_w), r0 = precs + sh_excl_scan(my_r, red, &tot_r);
  __shared__ int32_t rbase_s[kShMaxSeqs];
#pragma unroll 1
  for (int s = s0; s < s1; ++s) {
    int32_t ignore = 0;
    const Seq r = seq_of(s, cu_s[s], &ignore);
    wbase_s[s] = (int)w0;
    rbase_s[s] = r.q ? (int)r0 : -1;
    if (!r.q) continue;
    int c0;
    const int nch = osplit ? own_chunks(r, &c0) : 1;
    w0 += (int64_t)groups_of(r.q) * nch;
    r0 += (int64_t)r.q * nch;
  }
  if (status) atomicOr(&status_s, status);
  __syncthreads();
  const int Tw = min(cu_s[b.S], b.T);
  if (tid == 0) {
    hdr->n_entries = (int)(psplit ? n_parts : n_tiles);
    hdr->n_waves = (int)(few_waves + tot_w);
    hdr->n_tokens = Tw;
    hdr->status = status_s;
    hdr->window = b.window;
  }
  // a prefix's entries, chunk by chunk: the tiles that read the same keys are neighbours
  for (int p = tid >> 6; p < b.n_prefix; p += kShPlanThreads / 64) {
    const int n = pcnt_s[p];
    if (!n) continue;
    int c0;
    const int P = b.prefix_len[p], C = sh_prefix_chunk(P), nch_all = chunks_of(p, &c0), nch = psplit ? nch_all : 1;
    const bool few = n <= kShWaveTokens;
    const int tiles = few ? 1 : (n + kShRowTokens - 1) / kShRowTokens;
    ShEntry* out = (few ? waves : entries) + pent_s[p];
    for (int i = tid & 63; i < tiles * nch; i += 64) {
      const int c = i / tiles, t = i % tiles;
      ShEntry e;
      e.base = b.prefix_base[p];
      e.cap = b.prefix_cap[p];
      e.first = plist_s[p] + t * kShRowTokens;
      e.ntok = min(kShRowTokens, n - t * kShRowTokens);
      e.pos0 = 0;
      e.list = 1;
      e.key_lo = psplit ? max(plo_s[p], (c0 + c) * C) : plo_s[p];
      e.key_hi = psplit ? min(P, (c0 + c + 1) * C) : P;
      e.chunk = C;
      e.rec = prec_s[p] + c * n + t * kShRowTokens;
      e.pad = 0;
      out[i] = e;
    }
  }
  for (int t = tid; t < Tw; t += kShPlanThreads) {
    int lo = 0, hi = b.S - 1;  // last sequence with cu <= t
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cu_s[mid] <= t) lo = mid; else hi = mid - 1;
    }
    ShToken k = {0, 0, 0, 0, 0, 0};
    int32_t ignore = 0;
    const Seq r = seq_of(lo, cu_s[lo], &ignore);
    const int i = t - cu_s[lo];
    if (r.q) {
      int c0;
      const int nch_all = own_chunks(r, &c0), nch = osplit ? nch_all : 1;
      k.o_rec = rbase_s[lo] + i;
      k.o_n = nch;
      k.o_stride = r.q;
      if (i < listed(r)) {
        int pc0;
        const int n = pcnt_s[r.p], at = place_s[lo] + i;
        k.p_rec = prec_s[r.p] + at;
        k.p_n = psplit ? chunks_of(r.p, &pc0) : 1;
        k.p_stride = n;
        list[plist_s[r.p] + at] = make_int2(t, r.P + r.own0 + i);
      }
      if (i % kShWaveTokens == 0) {  // its group's entries
        for (int c = 0; c < nch; ++c) {
          ShEntry e;
          e.base = b.kv_base[lo];
          e.cap = b.kv_cap[lo];
          e.first = t;
          e.ntok = min(kShWaveTokens, r.q - i);
          e.pos0 = r.own0 + i;
          e.list = 0;
          const int klo = b.window > 0 ? max(0, e.pos0 - b.window + 1) : 0, khi = e.pos0 + e.ntok;
          e.key_lo = osplit ? max(klo, (c0 + c) * kShOwnChunk) : klo;
          e.key_hi = osplit ? min(khi, (c0 + c + 1) * kShOwnChunk) : khi;
          e.chunk = kShOwnChunk;
          e.rec = rbase_s[lo] + c * r.q + i;
          e.pad = 0;
          waves[wbase_s[lo] + (i / kShWaveTokens) * nch + c] = e;
        }
      }
    }
    tokens[t] = k;
  }
}

// ---- the items ------------------------------------------------------------------------------------

// QT tiles of 16 query rows of a wave (row rq = 16 qt + n is token rq / 8, head rq % 8 of the group): the Q^T operand, the slab
// positions that a row sees, the chunk's running softmax (S^T and O^T as in attn.hip) and the range's total.
template <int QT>
struct ShRows {
  bf16x8_t qf[QT][2];
  int lo[QT], hi[QT];
  bool val[QT];
  float m[QT], tm[QT];
  f32x4_t O[QT][4], L[QT], tO[QT][4];
  float tL[QT];  // (every element of L is the row's sum)
};

template <int QT>
__device__ __forceinline__ void sh_fresh(ShRows<QT>& R) {
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    R.m[qt] = -1e30f;
    R.L[qt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) R.O[qt][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
}

// The fold of (m, l, O) into the total (M, L, O): the same operations in the items and in the merge.
struct ShFold {
  float M, a, c;  // the new maximum, what the total and the chunk are multiplied with
};
__device__ __forceinline__ ShFold sh_fold(float M, float m) {
  const float x = M > m ? M : m;
  return {x, __builtin_amdgcn_exp2f(M - x), __builtin_amdgcn_exp2f(m - x)};
}

template <int QT>
__device__ __forceinline__ void sh_fold_chunk(ShRows<QT>& R) {
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const ShFold f = sh_fold(R.tm[qt], R.m[qt]);
    R.tm[qt] = f.M;
    R.tL[qt] = fmaf(R.L[qt][0], f.c, R.tL[qt] * f.a);
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int v = 0; v < 4; ++v) R.tO[qt][dt][v] = fmaf(R.O[qt][dt][v], f.c, R.tO[qt][dt][v] * f.a);
  }
}

// rows of the entry's tokens tok0 .. : in the prefix's list, or behind one another
template <int QT>
__device__ __forceinline__ void sh_rows_init(ShRows<QT>& R, const ShEntry& e, int tok0, const int2* __restrict__ list,
                                             const uint16_t* __restrict__ q, int kv_head, int Hq, int window) {
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int rq = 16 * qt + n, ti = tok0 + (rq >> 3);
    R.val[qt] = ti < e.ntok;
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
    R.lo[qt] = 0;
    R.hi[qt] = INT32_MAX;  // a row that is none sees all (its scores are 0, nothing of it is written)
    if (R.val[qt]) {
      int2 tp = make_int2(e.first + ti, e.pos0 + ti);
      if (e.list) tp = list[e.first + ti];
      R.hi[qt] = tp.y;
      R.lo[qt] = window > 0 ? max(0, tp.y - window + 1) : 0;
      const uint16_t* qp = q + ((size_t)tp.x * Hq + kv_head * 8 + (rq & 7)) * 64 + 8 * g;
      a = *reinterpret_cast<const uint4*>(qp);
      b = *reinterpret_cast<const uint4*>(qp + 32);
    }
    R.qf[qt][0] = as_bf16x8(a);
    R.qf[qt][1] = as_bf16x8(b);
    R.tm[qt] = -1e30f;
    R.tL[qt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) R.tO[qt][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  sh_fresh(R);
}

// the keys that every row of the wave sees: [*lo, *hi]
template <int QT>
__device__ __forceinline__ void sh_interior(const ShRows<QT>& R, int* lo, int* hi) {
  int a = 0, b = INT32_MAX;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    a = max(a, R.lo[qt]);
    b = min(b, R.hi[qt]);
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    a = max(a, __shfl_xor(a, o, 64));
    b = min(b, __shfl_xor(b, o, 64));
  }
  *lo = scalar(a);
  *hi = scalar(b);
}

__device__ __forceinline__ bool bf16_pair_wild(uint32_t w) {
  return (w & 0x7f800000u) == 0x7f800000u || (w & 0x7f80u) == 0x7f80u;
}

// Where a block has keys that some row does not see, their values may be infinite or NaN, and P is 0 there: 0 x inf would be NaN.
// Such values are left out of v, and rows that see one get it by what the products of P with the classes' indicators say.
template <int QT>
__device__ __forceinline__ void sh_wild_values(ShRows<QT>& R, uint4& v0, uint4& v1, int dt, const bf16x8_t (&pt)[QT][2]) {
  uint32_t w[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
  for (int kind = 0; kind < 3; ++kind) {  // +inf, -inf, NaN
    uint32_t f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t o = 0;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t x = (w[i] >> (16 * half)) & 0xffffu;
        const bool is = kind == 0 ? x == 0x7f80u : kind == 1 ? x == 0xff80u : (x & 0x7fffu) > 0x7f80u;
        if (is) o |= 0x3f80u << (16 * half);
      }
      f[i] = o;
    }
    const float add = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : NAN;
    const bf16x8_t f0 = as_bf16x8(make_uint4(f[0], f[1], f[2], f[3])), f1 = as_bf16x8(make_uint4(f[4], f[5], f[6], f[7]));
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      f32x4_t c = mfma16x16x32(f0, pt[qt][0], f32x4_t{0.f, 0.f, 0.f, 0.f});
      c = mfma16x16x32(f1, pt[qt][1], c);
#pragma unroll
      for (int v = 0; v < 4; ++v) R.O[qt][dt][v] += c[v] > 0.f ? add : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if ((w[i] & 0x7f80u) == 0x7f80u) w[i] &= 0xffff0000u;
    if ((w[i] & 0x7f800000u) == 0x7f800000u) w[i] &= 0xffffu;
  }
  v0 = make_uint4(w[0], w[1], w[2], w[3]);
  v1 = make_uint4(w[4], w[5], w[6], w[7]);
}

// One 64-key block against the wave's rows.  k(kt, step) and v(dt, half) give its fragments.  As in attn.hip: scores S^T = K . Q^T,
// P = 2^(s scale - m) rounded to bf16 (2^-9 of each; the row sum takes the rounded values), O^T += V^T . P^T, L += 1 . P^T.
template <int QT, bool MASKED, bool INREG, class KF, class VF, class AF>
__device__ __forceinline__ void sh_block(ShRows<QT>& R, KF&& k, VF&& v, AF&& after_scores, int kb, bool interior, int key_lo, int key_hi) {
  const int g = (threadIdx.x & 63) >> 4;
  const float scale = 0.125f * kLog2e;
  const bf16x8_t ones = as_bf16x8(make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u));
  bf16x8_t pt[QT][2];
  // the row tiles at once where the fragments come from LDS (each is read once), one after the other where they are in
  // registers (half as many scores live)
  constexpr int QN = INREG ? 1 : QT;
#pragma unroll
  for (int q0 = 0; q0 < QT; q0 += QN) {
    f32x4_t s[QN][4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      const bf16x8_t k0 = as_bf16x8(k(kt, 0)), k1 = as_bf16x8(k(kt, 1));
#pragma unroll
      for (int j = 0; j < QN; ++j) {
        s[j][kt] = mfma16x16x32(k0, R.qf[q0 + j][0], f32x4_t{0.f, 0.f, 0.f, 0.f});
        s[j][kt] = mfma16x16x32(k1, R.qf[q0 + j][1], s[j][kt]);
      }
    }
    if (q0 + QN == QT) after_scores();
#pragma unroll
    for (int j = 0; j < QN; ++j) {
      const int qt = q0 + j;
      float bmax = -INFINITY;
      if (MASKED && !interior) {
        const int lo = max(key_lo, R.lo[qt]), hi = min(key_hi - 1, R.hi[qt]);
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = kb + tile_key(kt, 4 * g + i);
            s[j][kt][i] = key >= lo && key <= hi ? s[j][kt][i] : -INFINITY;
          }
      }
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) bmax = fmaxf(bmax, s[j][kt][i]);
      const float m_blk = max_lane_groups(bmax) * scale;
      const bool move = m_blk > R.m[qt] + kMaxSlack;
      if (__ballot(move)) {
        const float m_new = move ? m_blk : R.m[qt];
        const float alpha = __builtin_amdgcn_exp2f(R.m[qt] - m_new);
        R.m[qt] = m_new;
        R.L[qt] *= alpha;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) R.O[qt][dt] *= alpha;
      }
      const float neg_m = -R.m[qt];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          pt[qt][kt >> 1][(kt & 1) * 4 + i] = (__bf16)__builtin_amdgcn_exp2f(fmaf(s[j][kt][i], scale, neg_m));
      R.L[qt] = mfma16x16x32(ones, pt[qt][0], R.L[qt]);
      R.L[qt] = mfma16x16x32(ones, pt[qt][1], R.L[qt]);
    }
  }
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) {
    uint4 v0 = v(dt, 0), v1 = v(dt, 1);
    if (MASKED && !interior) {
      if (kb < key_lo || kb + 64 > key_hi) {  // keys outside the item's range may never have been written
        v0 = mask_keys(v0, kb + 8 * g, key_lo, key_hi);
        v1 = mask_keys(v1, kb + 32 + 8 * g, key_lo, key_hi);
      }
      const bool wild = bf16_pair_wild(v0.x) || bf16_pair_wild(v0.y) || bf16_pair_wild(v0.z) || bf16_pair_wild(v0.w) ||
                        bf16_pair_wild(v1.x) || bf16_pair_wild(v1.y) || bf16_pair_wild(v1.z) || bf16_pair_wild(v1.w);
      if (__ballot(wild)) sh_wild_values(R, v0, v1, dt, pt);
    }
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      R.O[qt][dt] = mfma16x16x32(as_bf16x8(v0), pt[qt][0], R.O[qt][dt]);
      R.O[qt][dt] = mfma16x16x32(as_bf16x8(v1), pt[qt][1], R.O[qt][dt]);
    }
  }
}

// A record: O[64] of (record, kv head, head of the group), and apart from it (m, l).
__device__ __forceinline__ float* sh_rec_o(float* parts, int rec, int Hkv, int g, int h) {
  return parts + (((size_t)rec * Hkv + g) * 8 + h) * 64;
}
__device__ __forceinline__ float* sh_rec_ml(float* parts, int max_recs, int rec, int Hkv, int g, int h) {
  return parts + (size_t)max_recs * Hkv * 512 + (((size_t)rec * Hkv + g) * 8 + h) * 2;
}

template <int QT>
__device__ __forceinline__ void sh_write(const ShRows<QT>& R, const ShEntry& e, int tok0, int kv_head, int Hkv, int max_recs,
                                         float* __restrict__ parts) {
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    if (!R.val[qt]) continue;
    const int rq = 16 * qt + n, rec = e.rec + tok0 + (rq >> 3);
    float* o = sh_rec_o(parts, rec, Hkv, kv_head, rq & 7) + 4 * g;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) *reinterpret_cast<f32x4_t*>(o + 16 * dt) = R.tO[qt][dt];
    if (g == 0) *reinterpret_cast<float2*>(sh_rec_ml(parts, max_recs, rec, Hkv, kv_head, rq & 7)) = make_float2(R.tm[qt], R.tL[qt]);
  }
}

// An item of up to 4 tokens by one wave, K and V straight from the slab.
template <int QT>
__device__ __forceinline__ void sh_wave_item(const ShEntry& e, int kv_head, const int2* __restrict__ list, const uint16_t* __restrict__ q,
                                             const uint16_t* __restrict__ k_pool, const uint16_t* __restrict__ v_pool, int Hq, int Hkv,
                                             int window, int max_recs, float* __restrict__ parts) {
  const int lane = threadIdx.x & 63;
  const int64_t base = e.base + (int64_t)kv_head * e.cap * 64;
  const uint16_t *K = k_pool + base, *V = v_pool + base;
  ShRows<QT> R;
  sh_rows_init(R, e, 0, list, q, kv_head, Hq, window);
  int int_lo, int_hi;
  sh_interior(R, &int_lo, &int_hi);
  int_lo = max(int_lo, e.key_lo);
  int_hi = min(int_hi, e.key_hi - 1);
  uint4 kc[4][2], vc[4][2];
  int kb = e.key_lo & ~63;
  if (kb < e.key_hi) load_k_tile(kc, K, kb, lane);
  int next_fold = (kb / e.chunk + 1) * e.chunk;
  for (; kb < e.key_hi; kb += 64) {
    if (kb == next_fold) {
      sh_fold_chunk(R);
      sh_fresh(R);
      next_fold += e.chunk;
    }
    load_v_tile(vc, V, kb, lane);
    // the next block's K goes into this one's registers once the scores are made
    auto next_k = [&]() __attribute__((always_inline)) {
      if (kb + 64 < e.key_hi) load_k_tile(kc, K, kb + 64, lane);
    };
    auto kf = [&](int kt, int st) __attribute__((always_inline)) { return kc[kt][st]; };
    auto vf = [&](int dt, int h) __attribute__((always_inline)) { return vc[dt][h]; };
    sh_block<QT, true, true>(R, kf, vf, next_k, kb, kb >= int_lo && kb + 63 <= int_hi, e.key_lo, e.key_hi);
  }
  sh_fold_chunk(R);
  sh_write(R, e, 0, kv_head, Hkv, max_recs, parts);
}

// An item of up to 16 tokens by a workgroup of 4 waves, 4 tokens each: a block's K and V go to LDS once for all of them (two
// buffers, the next block's loads in flight while this one computes).
__device__ __forceinline__ void sh_tile_item(const ShEntry& e, int kv_head, const int2* __restrict__ list, const uint16_t* __restrict__ q,
                                             const uint16_t* __restrict__ k_pool, const uint16_t* __restrict__ v_pool, int Hq, int Hkv,
                                             int window, int max_recs, float* __restrict__ parts, uint4 (&buf0)[2][512],
                                             uint4 (&buf1)[2][512]) {
  typedef __attribute__((address_space(3))) void* lds_ptr;
  const int lane = threadIdx.x & 63, wave = scalar((int)threadIdx.x >> 6);
  const int64_t base = e.base + (int64_t)kv_head * e.cap * 64;
  const char *Kb = reinterpret_cast<const char*>(k_pool + base), *Vb = reinterpret_cast<const char*>(v_pool + base);
  auto issue = [&](uint4 (&dst)[2][512], int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int s0 = 256 * j + 64 * wave;
      const char* blk = (s0 < 512 ? Kb : Vb) + ((size_t)kb * 8 + (s0 & 511)) * 16;
      __builtin_amdgcn_global_load_lds((const void*)(blk + (uint32_t)lane * 16u), (lds_ptr)(&dst[0][0] + s0), 16, 0, 0);
    }
  };
  auto landed = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
    lds_barrier();
  };
  const int kb_first = e.key_lo & ~63;
  issue(buf0, kb_first);
  ShRows<2> R;
  sh_rows_init(R, e, 4 * wave, list, q, kv_head, Hq, window);
  int int_lo, int_hi;
  sh_interior(R, &int_lo, &int_hi);
  int_lo = max(int_lo, e.key_lo);
  int_hi = min(int_hi, e.key_hi - 1);
  const bool mine = 4 * wave < e.ntok;
  landed();
  int next_fold = (kb_first / e.chunk + 1) * e.chunk;
  auto step = [&](uint4 (&cur)[2][512], uint4 (&nxt)[2][512], int kb) __attribute__((always_inline)) {
    if (kb + 64 < e.key_hi) issue(nxt, kb + 64);
    if (mine) {
      if (kb == next_fold) {
        sh_fold_chunk(R);
        sh_fresh(R);
        next_fold += e.chunk;
      }
      auto kf = [&](int kt, int st) __attribute__((always_inline)) { return cur[0][kt * 128 + st * 64 + lane]; };
      auto vf = [&](int dt, int h) __attribute__((always_inline)) { return cur[1][h * 256 + dt * 64 + lane]; };
      if (kb >= int_lo && kb + 63 <= int_hi) sh_block<2, false, false>(R, kf, vf, [] {}, kb, true, e.key_lo, e.key_hi);
      else sh_block<2, true, false>(R, kf, vf, [] {}, kb, false, e.key_lo, e.key_hi);
    }
    landed();
  };
  for (int kb = kb_first; kb < e.key_hi; kb += 128) {
    step(buf0, buf1, kb);
    if (kb + 64 < e.key_hi) step(buf1, buf0, kb + 64);
  }
  if (mine) {
    sh_fold_chunk(R);
    sh_write(R, e, 4 * wave, kv_head, Hkv, max_recs, parts);
  }
}

__global__ __launch_bounds__(256, 2) void attn_shared_kernel(const uint16_t* __restrict__ q, const uint16_t* __restrict__ k_pool,
                                                             const uint16_t* __restrict__ v_pool, int Hq, int Hkv, ShLayout L,
                                                             const char* __restrict__ plan, float* __restrict__ parts) {
  __shared__ uint4 buf0[2][512], buf1[2][512];  // [K, V][a 64-key block]
  const ShHeader* hdr = reinterpret_cast<const ShHeader*>(plan);
  const ShEntry* entries = reinterpret_cast<const ShEntry*>(plan + L.o_entries);
  const ShEntry* waves = reinterpret_cast<const ShEntry*>(plan + L.o_waves);
  const int2* list = reinterpret_cast<const int2*>(plan + L.o_list);
  const int n_tile = hdr->n_entries * Hkv, n_wave = hdr->n_waves * Hkv, window = hdr->window;
  const int n = n_tile + (n_wave + 3) / 4;
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    if (i < n_tile) {
      const ShEntry e = entries[i / Hkv];
      sh_tile_item(e, i % Hkv, list, q, k_pool, v_pool, Hq, Hkv, window, L.max_recs, parts, buf0, buf1);
    } else {
      const int w = (i - n_tile) * 4 + scalar((int)threadIdx.x >> 6);
      if (w < n_wave) {
        const ShEntry e = waves[w / Hkv];
        if (e.ntok <= 2) sh_wave_item<1>(e, w % Hkv, list, q, k_pool, v_pool, Hq, Hkv, window, L.max_recs, parts);
        else sh_wave_item<2>(e, w % Hkv, list, q, k_pool, v_pool, Hq, Hkv, window, L.max_recs, parts);
      }
    }
  }
}

// The records of a token's 8 rows of a kv head, folded: the prefix's, the sequence's own, then both and the sink.  Thread (h = tid / 8,
// part = tid % 8) takes 8 dims.  A token without any record (its sequence was refused) gets zeros.
constexpr int kShMergeAhead = 4;

__global__ __launch_bounds__(64) void attn_shared_merge_kernel(const float* __restrict__ parts_in, const char* __restrict__ plan, ShLayout L,
                                                               const float* __restrict__ sinks, int Hq, int Hkv, uint16_t* __restrict__ out) {
  const ShHeader* hdr = reinterpret_cast<const ShHeader*>(plan);
  const int t = blockIdx.x, g = blockIdx.y;
  if (t >= hdr->n_tokens) return;  // behind the last sequence: left as it was
  const ShToken k = reinterpret_cast<const ShToken*>(plan + L.o_tokens)[t];
  float* parts = const_cast<float*>(parts_in);
  const int h = threadIdx.x >> 3, part = threadIdx.x & 7;
  float Mt[2], Lt[2], Ot[2][8];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int rec0 = w ? k.o_rec : k.p_rec, n = w ? k.o_n : k.p_n, stride = w ? k.o_stride : k.p_stride;
    Mt[w] = -1e30f;
    Lt[w] = 0.f;
#pragma unroll
    for (int d = 0; d < 8; ++d) Ot[w][d] = 0.f;
    for (int c0 = 0; c0 < n; c0 += kShMergeAhead) {
      float2 ml[kShMergeAhead];
      float4 o[kShMergeAhead][2];
#pragma unroll
      for (int j = 0; j < kShMergeAhead; ++j) {
        const int rec = rec0 + min(c0 + j, n - 1) * stride;
        ml[j] = *reinterpret_cast<const float2*>(sh_rec_ml(parts, L.max_recs, rec, Hkv, g, h));
        const float4* r = reinterpret_cast<const float4*>(sh_rec_o(parts, rec, Hkv, g, h) + part * 8);
        o[j][0] = r[0];
        o[j][1] = r[1];
      }
#pragma unroll
      for (int j = 0; j < kShMergeAhead; ++j)
        if (c0 + j < n) {
          const ShFold f = sh_fold(Mt[w], ml[j].x);
          Mt[w] = f.M;
          Lt[w] = fmaf(ml[j].y, f.c, Lt[w] * f.a);
          const float v[8] = {o[j][0].x, o[j][0].y, o[j][0].z, o[j][0].w, o[j][1].x, o[j][1].y, o[j][1].z, o[j][1].w};
#pragma unroll
          for (int d = 0; d < 8; ++d) Ot[w][d] = fmaf(v[d], f.c, Ot[w][d] * f.a);
        }
    }
  }
  const int head = g * 8 + h;
  const float sink = sinks[head] * kLog2e;
  const float M = fmaxf(sink, fmaxf(Mt[0], Mt[1]));
  const float a = __builtin_amdgcn_exp2f(Mt[0] - M), c = __builtin_amdgcn_exp2f(Mt[1] - M);
  const float total = fmaf(Lt[1], c, Lt[0] * a) + __builtin_amdgcn_exp2f(sink - M);
  const float inv = k.o_n > 0 ? 1.0f / total : 0.f;
  uint32_t w4[4];
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const float x = fmaf(Ot[1][2 * d], c, Ot[0][2 * d] * a) * inv, y = fmaf(Ot[1][2 * d + 1], c, Ot[0][2 * d + 1] * a) * inv;
    w4[d] = (uint32_t)f2bf(x) | ((uint32_t)f2bf(y) << 16);
  }
  *reinterpret_cast<uint4*>(out + ((size_t)t * Hq + head) * 64 + part * 8) = make_uint4(w4[0], w4[1], w4[2], w4[3]);
}

static int check_shared_shape(const char* what, int T, int S, int n_prefix, int Hkv) {
  FLYAI_REQUIRE(T >= 0 && T <= 65536, "%s: n_tokens %d outside [0, 65536]", what, T);
  FLYAI_REQUIRE(S >= 0 && S <= kShMaxSeqs, "%s: n_seqs %d outside [0, %d]", what, S, kShMaxSeqs);
  FLYAI_REQUIRE(n_prefix >= 0 && n_prefix <= kShMaxPrefixes, "%s: n_prefixes %d outside [0, %d]", what, n_prefix, kShMaxPrefixes);
  FLYAI_REQUIRE(Hkv >= 1 && Hkv <= 64, "%s: n_kv_heads %d outside [1, 64]", what, Hkv);
  return FLYAI_OK;
}

}  // namespace flyai

using namespace flyai;

extern "C" size_t flyai_attn_shared_plan_bytes(int32_t T, int32_t S, int32_t n_prefix) {
  if (T < 0 || T > 65536 || S < 0 || S > kShMaxSeqs || n_prefix < 0 || n_prefix > kShMaxPrefixes) return 0;
  return sh_layout(T, S, n_prefix).bytes;
}

extern "C" size_t flyai_attn_shared_workspace_bytes(int32_t T, int32_t Hkv) {
  if (T < 0 || T > 65536 || Hkv < 1 || Hkv > 64) return 0;
  return (size_t)sh_layout(T, 0, 0).max_recs * Hkv * 8 * (64 + 2) * sizeof(float);
}

extern "C" int flyai_attn_shared_plan(const int32_t* q_lens, const int32_t* starts, const int64_t* kv_base, const int32_t* kv_cap,
                                      const int32_t* prefix_of, const int32_t* prefix_len, const int64_t* prefix_base,
                                      const int32_t* prefix_cap, int32_t S, int32_t n_prefix, int32_t Hkv, int32_t window, int32_t T,
                                      int64_t pool_elems, void* plan, flyai_stream_t stream) {
  const int rc = check_shared_shape("attn_shared_plan", T, S, n_prefix, Hkv);
  if (rc) return rc;
  FLYAI_REQUIRE(window >= 0 && pool_elems >= 0, "attn_shared_plan: window and pool_elems must be >= 0");
  FLYAI_REQUIRE((S == 0 || (q_lens && starts && kv_base && kv_cap && prefix_of)) &&
                    (n_prefix == 0 || (prefix_len && prefix_base && prefix_cap)) && plan && ((uintptr_t)plan & 15) == 0,
                "attn_shared_plan: null pointer, or a plan that is not 16-byte aligned");
  const ShBatch b = {q_lens, starts, kv_base, kv_cap, prefix_of, prefix_len, prefix_base, prefix_cap, S, n_prefix, Hkv, window, T, pool_elems};
  hipLaunchKernelGGL(attn_shared_plan_kernel, dim3(1), dim3(kShPlanThreads), 0, as_stream(stream), b, static_cast<char*>(plan));
  return check_launch("attn_shared_plan");
}

extern "C" int flyai_attn_shared(const uint16_t* q, const uint16_t* k_pool, const uint16_t* v_pool, const float* sinks, int32_t Hq,
                                 int32_t Hkv, int32_t D, int32_t T, int32_t S, int32_t n_prefix, const void* plan, void* workspace,
                                 uint16_t* out, flyai_stream_t stream) {
  const int rc = check_shared_shape("attn_shared", T, S, n_prefix, Hkv);
  if (rc) return rc;
  FLYAI_REQUIRE(D == 64 && Hq == 8 * Hkv, "attn_shared: needs head_dim 64 and 8 query heads per kv head");
  if (T == 0) return FLYAI_OK;
  FLYAI_REQUIRE(q && k_pool && v_pool && sinks && plan && workspace && out, "attn_shared: null pointer");
  FLYAI_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)k_pool & 15) == 0 && ((uintptr_t)v_pool & 15) == 0 &&
                    ((uintptr_t)out & 15) == 0 && ((uintptr_t)workspace & 15) == 0 && ((uintptr_t)plan & 15) == 0,
                "attn_shared: q, the pools, out, plan and workspace must be 16-byte aligned");
  const ShLayout L = sh_layout(T, S, n_prefix);
  hipStream_t s = as_stream(stream);
  const int64_t most = (int64_t)L.max_entries * Hkv + ((int64_t)L.max_waves * Hkv + 3) / 4;
  hipLaunchKernelGGL(attn_shared_kernel, dim3((unsigned)(most < kShGrid ? most : kShGrid)), dim3(256), 0, s, q, k_pool, v_pool, Hq, Hkv, L,
                     static_cast<const char*>(plan), static_cast<float*>(workspace));
  const int rc2 = check_launch("attn_shared");
  if (rc2) return rc2;
  hipLaunchKernelGGL(attn_shared_merge_kernel, dim3(T, Hkv), dim3(64), 0, s, static_cast<const float*>(workspace),
                     static_cast<const char*>(plan), L, sinks, Hq, Hkv, out);
  return check_launch("attn_shared_merge");
}
