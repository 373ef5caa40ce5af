// Drafted tokens of many streams verified against the target's filtered distributions, from given uniforms: the accept rule of
// speculative sampling (Sampler.accept of phase0/specsample.py:79-107, one stream there) for every stream of a batch, with or without the
// drafter's own distribution.
//
// Row r of the logits judges its stream's drafted token d_r; a stream's rows lie behind one another, the last one
// usually without a draft (the bonus token's).  w are the row's integer weights as in sample.hip (temperature, top-k and
// top-p of the stream), W their sum.  A draft is accepted if u_r q_r(d) W < w_d (fp64; q = 1 without a distribution).  The first
// row whose draft is not accepted, or that has none, ends the stream with a draw: the first id whose inclusive prefix
// of w' exceeds floor(u W'), W' the sum of w', where
//   w'_v = w_v                               without a draft,
//   w'_v = w_v but 0 for the draft           rejected, no distribution,
//   w'_v = max(0, w_v - floor(q_v W))        rejected (the product in fp64);
// where nothing is left the first id of maximal w, where every weight is 0 id 0.  A greedy stream (temp <= 0) accepts the first id of
// maximal logit and ends with it.  All sums are of integers: no result depends on the launch.
//
// Three launches: verify_rows_kernel finds each row's filter, W, and whether its draft is accepted; a stream's first row that
// is not is then the only one whose weights are needed one by one: verify_pieces_kernel sums w' over pieces of its ids, and
// verify_draw_kernel finds the piece and the id, and writes what comes out.
//
// With a vocabulary of 201,088 (us): 128 streams' 1,152 rows 159 to 163, of which the rows 118 to 125 (463 MB, 3.9 to 3.7 TB/s; a product of
// two arrays reaches 6.3), the pieces 36, the draw 7; 24 streams' 120 rows 44 (27, 11, 7); one stream's 5 rows 34 (23, 6, 5), where a row is one CU's:
// 12 us of counting in LDS, some 8 of sums over the values.  The rows that many passes over the logits took (ver_row_general's way for all)
// were 1,215 us of 128 streams, 482 of one.  Rows counted in up to eight parts, then added up, made one stream's 32 us and 24 streams' 53;
// a workgroup a CU with the next row's loads ahead 205 of 128 streams' 159.
#include <algorithm>

#include "sample.h"

namespace flyai {

struct VerRow {
  uint64_t W;         // kept weight
  uint64_t tie_keep;  // ties at `edge` that are kept, in id order; ~0: all
  float zmax;
  float lo, edge;     // kept are values from lo (top-k) and edge (top-p) on, -inf: no such bound; values of x, or of z = x / temp (by_z)
  int32_t by_z;
  int32_t accept;
  int32_t arg;        // greedy: the first id of maximal logit
  float p;            // the draft's probability
  int32_t pad;
};

// A piece is kPiece consecutive ids of a stream's last row: 8 for each lane of a wave.
constexpr int kPiece = 512;

struct VerPiece {
  uint64_t above, tie;  // w' of the piece's kept tokens above the edge, of all its ties there
  uint32_t ties, pad;
};

struct VerArgs {
  const uint16_t* logits;
  const int32_t *cu_rows, *draft;
  const double *u, *u_draw;
  const float *temp, *top_p;  // of each stream, or null: the scalars
  const int32_t* top_k;
  float temp1, top_p1;
  int32_t top_k1;
  const float* probs;         // [n_probs, V], or null
  const int32_t* probs_row;   // row of probs for each row, or null: the row itself
  int32_t n_probs, R, V, S, pieces;
};

struct VerParams {
  float temp, tdiv, top_p;
  int top_k;
};

__device__ __forceinline__ VerParams ver_params(const VerArgs& a, int s) {
  VerParams p;
  p.temp = a.temp ? a.temp[s] : a.temp1;
  p.tdiv = fmaxf(p.temp, 1e-6f);
  p.top_p = a.top_p ? a.top_p[s] : a.top_p1;
  p.top_k = a.top_k ? a.top_k[s] : a.top_k1;
  return p;
}

// a stream's rows, within the batch whatever cu_rows holds
__device__ __forceinline__ int2 ver_range(const VerArgs& a, int s) {
  const int r0 = min(max(a.cu_rows[s], 0), a.R);
  return make_int2(r0, max(r0, min(max(a.cu_rows[s + 1], 0), a.R)));
}

// the drafted id, -1 for none
__device__ __forceinline__ int ver_draft(const VerArgs& a, int r) {
  const int d = a.draft[r];
  return d >= 0 && d < a.V ? d : -1;
}

__device__ __forceinline__ const float* ver_probs(const VerArgs& a, int r) {
  if (!a.probs) return nullptr;
  const int i = a.probs_row ? a.probs_row[r] : r;
  return i >= 0 && i < a.n_probs ? a.probs + (size_t)i * a.V : nullptr;
}

__device__ __forceinline__ double ver_uniform(double u) { return u >= 0.0 ? fmin(u, 0x1.fffffffffffffp-1) : 0.0; }

__device__ __forceinline__ bool ver_accepts(const VerArgs& a, int r, int d, uint64_t wd, uint64_t W) {
  if (d < 0) return false;
  const float* q = ver_probs(a, r);
  const double qd = q ? (double)fmaxf(q[d], 0.f) : 1.0;
  return ver_uniform(a.u[r]) * qd * (double)W < (double)wd;
}

// what a rejected draft's distribution leaves of a weight (whole numbers up to 2^40, which doubles hold)
__device__ __forceinline__ double ver_rest(double w, float q, double W) {
  const double left = w - floor((double)fmaxf(q, 0.f) * W);
  return fmax(left, 0.0);
}

// One row by a workgroup, for any logits: every pass reads the row again.
__device__ __forceinline__ void ver_row_general(const VerArgs& a, int row, const VerParams& p, SampShared& sh, VerRow* out) {
  const uint16_t* x = a.logits + (size_t)row * a.V;
  const int tid = threadIdx.x, V = a.V, d = ver_draft(a, row);
  VerRow o = {};
  auto zof = [&](int v) __attribute__((always_inline)) { return __fdiv_rn(bf2f(x[v]), p.tdiv); };
  uint32_t kth = 0;
  if (p.top_k > 0 && p.top_k < V) {
    uint64_t above = 0;
    kth = radix_select(V, [&](int v, uint32_t* k) { *k = f32_key(zof(v)); return true; },
                       [&](int) { return (uint64_t)1; }, (uint64_t)(p.top_k - 1), &above, sh);
  }
  auto kept_k = [&](int v, uint32_t* k) __attribute__((always_inline)) {
    *k = f32_key(zof(v));
    return *k >= kth;
  };
  uint32_t mkey = 0;
  for (int v = tid; v < V; v += kSampThreads) mkey = max(mkey, f32_key(zof(v)));
  mkey = block_max_u32(mkey, sh.red32);
  o.zmax = key_f32(mkey);
  uint64_t sum = 0;
  for (int v = tid; v < V; v += kSampThreads) {
    uint32_t k;
    if (kept_k(v, &k)) sum += samp_weight(zof(v), o.zmax);
  }
  o.W = block_sum(sum, sh.red64);
  o.tie_keep = ~0ull;
  uint32_t pkey = 0;
  if (p.top_p > 0.f && p.top_p < 1.f) {
    const uint64_t T = (uint64_t)floor((double)p.top_p * (double)o.W);
    uint64_t above = 0;
    pkey = radix_select(V, kept_k, [&](int v) { return samp_weight(zof(v), o.zmax); }, T, &above, sh);
    if (pkey) {
      // tie j (0-based, id order) of the boundary value is kept iff above + j * wb <= T (tie 0 always is)
      const uint64_t wb = samp_weight(key_f32(pkey), o.zmax);
      uint32_t ties = 0;
      for (int v = tid; v < V; v += kSampThreads) ties += f32_key(zof(v)) == pkey;
      const uint64_t n = block_sum((uint64_t)ties, sh.red64);
      o.tie_keep = min(n, (T - above) / wb + 1);
      o.W = above + o.tie_keep * wb;
    }
  }
  // the draft's weight; as a boundary tie it counts if its rank among the ties is kept
  uint64_t wd = 0;
  if (d >= 0) {
    const uint32_t k = f32_key(zof(d));
    bool kept = k >= kth && k >= pkey;
    if (kept && pkey && k == pkey) {
      uint32_t before = 0;
      for (int v = tid; v < d; v += kSampThreads) before += f32_key(zof(v)) == pkey;
      kept = block_sum((uint64_t)before, sh.red64) < o.tie_keep;
    }
    if (kept) wd = samp_weight(zof(d), o.zmax);
  }
  if (tid) return;
  // (bounds that are NaN go with a NaN maximum, where nothing has weight)
  o.lo = kth ? key_f32(kth) : -INFINITY;
  o.edge = pkey ? key_f32(pkey) : -INFINITY;
  o.by_z = 1;
  o.p = o.W ? (float)((double)wd / (double)o.W) : 0.f;
  o.accept = ver_accepts(a, row, d, wd, o.W);
  *out = o;
}

// the stream of a row (the last one, should malformed cu_rows name several), -1 behind the last
__device__ __forceinline__ int ver_stream(const VerArgs& a, int row, int* found) {
  if (threadIdx.x == 0) *found = -1;
  __syncthreads();
  for (int s = threadIdx.x; s < a.S; s += blockDim.x)
    if (a.cu_rows[s] <= row && row < a.cu_rows[s + 1]) atomicMax(found, s);
  __syncthreads();
  return *found;
}

// ---- a row, 16 bytes a thread at a time ----
struct __attribute__((packed, aligned(2))) VerVec { u32x4_t v; };  // 16 bytes at any element's address

template <int AHEAD>
struct VerLoaded { u32x4_t w[AHEAD]; };

template <int AHEAD>
__device__ __forceinline__ VerLoaded<AHEAD> ver_load(const uint16_t* __restrict__ x, int v0, int full) {
  VerLoaded<AHEAD> l;
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) {
    const int v = v0 + j * kSampThreads * 8;
    l.w[j] = u32x4_t{0, 0, 0, 0};
    if (v < full) l.w[j] = reinterpret_cast<const VerVec*>(x + v)->v;
  }
  return l;
}

// f(first id, its 8 values) over the thread's vectors of [0, full), the next batch's loads in flight; `l` holds the first batch
template <int AHEAD, class F>
__device__ __forceinline__ void ver_each(const uint16_t* __restrict__ x, int full, VerLoaded<AHEAD> l, F&& f) {
  constexpr int kBatch = AHEAD * kSampThreads * 8;
  for (int v0 = (int)threadIdx.x * 8; v0 < full; v0 += kBatch) {
    const VerLoaded<AHEAD> next = ver_load<AHEAD>(x, v0 + kBatch, full);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int v = v0 + j * kSampThreads * 8;
      if (v < full) f(v, l.w[j]);
    }
    l = next;
  }
}

// ---- a greedy row ----
// Two values of a word at once, in an order that 16-bit integers have: negative ones' magnitude bits turned round.  A thread keeps the
// largest value and the first of its vectors that holds it; -0 orders below +0, so a row whose largest is a zero is looked at
// again for the first zero of either sign.
typedef short s16x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ s16x2_t ver_ordered(uint32_t w) {
  const s16x2_t x = __builtin_bit_cast(s16x2_t, w);
  return x ^ ((x >> 15) & (s16x2_t){0x7fff, 0x7fff});
}

struct VerGreedy {
  uint64_t best[kSampWaves];
  int at;
};

template <int AHEAD>
__device__ __forceinline__ void ver_row_greedy(const VerArgs& a, int row, const VerLoaded<AHEAD>& l, VerGreedy& sh, VerRow* out) {
  const uint16_t* x = a.logits + (size_t)row * a.V;
  const int tid = threadIdx.x, V = a.V, full = V & ~7;
  int best = -0x8001, at = V;  // (a thread without a vector: below every value)
  ver_each(x, full, l, [&](int v, u32x4_t w) {
    const s16x2_t m = __builtin_elementwise_max(__builtin_elementwise_max(ver_ordered(w.x), ver_ordered(w.y)),
                                                __builtin_elementwise_max(ver_ordered(w.z), ver_ordered(w.w)));
    const int top = max((int)m.x, (int)m.y);
    if (top > best) {
      best = top;
      at = v;
    }
  });
  auto one = [&](int v) __attribute__((always_inline)) { return (int)ver_ordered(x[v]).x; };
  if (at < V) {  // the first of the vector
    int i = 0;
    while (i < 7 && one(at + i) != best) ++i;
    at += i;
  }
  if (tid < V - full && one(full + tid) > best) {
    best = one(full + tid);
    at = full + tid;
  }
  // the largest, then the smallest id
  uint64_t key = ((uint64_t)(uint32_t)(best + 0x8001) << 32) | (uint32_t)~at;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const uint64_t y = __shfl_xor(key, o, 64);
    key = y > key ? y : key;
  }
  if ((tid & 63) == 0) sh.best[tid >> 6] = key;
  if (tid == 0) sh.at = V;
  __syncthreads();
  for (int w = 0; w < kSampWaves; ++w) key = sh.best[w] > key ? sh.best[w] : key;
  int arg = (int)~(uint32_t)key;
  if ((int)(key >> 32) == 0x8001) {  // +0 (uniform)
    for (int v = tid; v < V; v += kSampThreads)
      if ((x[v] & 0x7fff) == 0) {
        atomicMin(&sh.at, v);
        break;
      }
    __syncthreads();
    arg = sh.at;
  }
  if (tid) return;
  VerRow o = {};
  o.arg = arg;
  o.accept = ver_draft(a, row) == arg;
  o.p = o.accept ? 1.f : 0.f;
  *out = o;
}

// ---- a row by the counts of its values ----
// A bf16 row has few distinct values: the row is read once, each logit counted in LDS at its value's place, and everything else --
// the maximum, the weights (fp64 exponentials), their sum, top-k, top-p -- runs over the values.  Places: |x| in [2^-40, 2^24)
// of either sign, 8,192 each, and zero.  -inf and lower values than those have no weight wherever the maximum is one of these
// (checked), and are left out; a row with any other value, or whose quotients x / temp are not all normal, is left to
// ver_row_general.
constexpr int kVerHalf = 8192;        // places of a sign
constexpr uint32_t kVerFirst = 0x2b80;  // the bits of 2^-40
constexpr int kVerGroups = 2 * kVerHalf / 16;  // of 16 places in descending order; zero is in front of the first negative group's

struct VerHist {
  uint32_t cnt[2 * kVerHalf];   // by the bits: positive ones, then negative ones, each ascending in |x|
  uint64_t gsum[kVerGroups];    // the groups' weights
  uint32_t gcnt[kVerGroups];    // ... and counts, for top-k
  uint64_t red[kSampWaves];
  uint32_t zeros, bad, low;     // zero's count; a value that has no place; the largest (as f32 key) of the low ones
  int top;                      // the largest value's rank: negative ones from 0 on, zero, positive ones
  int group;                    // what a selection found: the group, the total above it
  uint64_t above, weight;
  float edge;
  uint64_t tie_keep;
  uint32_t before;
};

__device__ __forceinline__ float ver_rank_value(int rank) {
  if (rank == kVerHalf) return 0.f;
  return bf2f((uint16_t)(kVerFirst + (rank > kVerHalf ? rank - kVerHalf - 1 : kVerHalf - 1 - rank + 0x8000)));
}
// place l (0 .. 16, in descending order) of a group: its value, and how often it is there
__device__ __forceinline__ uint32_t ver_group_place(const VerHist& h, int g, int l, float* value) {
  const int zero = g == kVerGroups / 2;
  *value = 0.f;
  if (zero && l == 0) return h.zeros;
  l -= zero;
  if (l < 0 || l >= 16) return 0;
  const int i = g < kVerGroups / 2 ? kVerHalf - 1 - (g * 16 + l) : g * 16 + l;  // index of cnt
  *value = bf2f((uint16_t)(kVerFirst + (i < kVerHalf ? i : i - kVerHalf + 0x8000)));
  return h.cnt[i];
}

template <class T>
__device__ __forceinline__ T wave_total(T v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// the sum of 16 lanes, in the last of them
__device__ __forceinline__ uint32_t row_total(uint32_t v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  return v;
}
__device__ __forceinline__ uint64_t row_total(uint64_t v) {
  auto add = [&](uint32_t lo, uint32_t hi) __attribute__((always_inline)) { v += (uint64_t)hi << 32 | lo; };
#define FLYAI_ROW_STEP(ctrl)                                                            \
  add(__builtin_amdgcn_update_dpp(0, (uint32_t)v, ctrl, 0xf, 0xf, true), \
      __builtin_amdgcn_update_dpp(0, (uint32_t)(v >> 32), ctrl, 0xf, 0xf, true))
  FLYAI_ROW_STEP(0x111);
  FLYAI_ROW_STEP(0x112);
  FLYAI_ROW_STEP(0x114);
  FLYAI_ROW_STEP(0x118);
#undef FLYAI_ROW_STEP
  return v;
}

// The group where the running total of the groups' masses (thread g: group g's, `run` before it) first exceeds limit, to h.group
// (-1: none does) with the total above it.
__device__ __forceinline__ void ver_find_group(VerHist& h, uint64_t run, uint64_t mass, uint64_t limit) {
  if (threadIdx.x == 0) h.group = -1;
  __syncthreads();
  if (run <= limit && limit < run + mass) {
    h.group = threadIdx.x;
    h.above = run;
  }
  __syncthreads();
}

// false: the row is not one for this path (every thread)
template <int AHEAD>
__device__ __forceinline__ bool ver_row_counts(const VerArgs& a, int row, const VerParams& p, const VerLoaded<AHEAD>& l, VerHist& h, VerRow* out) {
  const uint16_t* x = a.logits + (size_t)row * a.V;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = a.V, d = ver_draft(a, row);
  if (!(p.tdiv < 0x1p60f)) return false;
  for (int i = tid; i < 2 * kVerHalf / 4; i += kSampThreads) reinterpret_cast<uint4*>(h.cnt)[i] = make_uint4(0, 0, 0, 0);
  h.gsum[tid] = 0;
  h.gcnt[tid] = 0;
  if (tid == 0) {
    h.zeros = h.bad = h.low = h.before = 0;
    h.top = -1;
  }
  const uint16_t dbits = d >= 0 ? x[d] : 0;
  __syncthreads();
  // (two 16-bit places of a word at once; 0x6000 tells a value without one)
  auto count = [&](uint32_t t) __attribute__((always_inline)) {
    const uint32_t at = ((t << 2) & 0x7ffc7ffcu) | (t & 0x80008000u);  // byte addresses
    char* c = reinterpret_cast<char*>(h.cnt);
    atomicAdd(reinterpret_cast<uint32_t*>(c + (at & 0xffffu)), 1u);
    atomicAdd(reinterpret_cast<uint32_t*>(c + (at >> 16)), 1u);
  };
  // a value that may have no place: one that has no weight is left out (`low` is the largest one's magnitude), another one leaves the
  // row to the general path (low 0)
  uint32_t zeros = 0, low = 0xffffu;
  auto one = [&](uint32_t bits) __attribute__((always_inline)) {
    const uint32_t mag = bits & 0x7fffu, t = mag - kVerFirst;
    const bool none = t >= (uint32_t)kVerHalf, neg = bits & 0x8000u;
    if (!none) atomicAdd(&h.cnt[t + (neg ? kVerHalf : 0)], 1u);
    zeros += mag == 0;
    const bool below = none && neg && mag > kVerFirst;
    low = min(low, below ? mag : none && mag != 0 ? 0u : 0xffffu);
  };
  const int full = V & ~7;
  ver_each(x, full, l, [&](int, u32x4_t w) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    uint32_t t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      t[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(u16x2, (uint32_t)w[i]) - (u16x2){(unsigned short)kVerFirst, (unsigned short)kVerFirst});
    if ((t[0] | t[1] | t[2] | t[3]) & 0x60006000u) {
#pragma unroll
      for (int i = 0; i < 8; ++i) one((i & 1 ? w[i >> 1] >> 16 : w[i >> 1]) & 0xffffu);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) count(t[i]);
    }
  });
  if (tid < V - full) one(x[full + tid]);
  if (zeros) atomicAdd(&h.zeros, zeros);
  if (low == 0) h.bad = 1;
  else if (low != 0xffffu) atomicMax(&h.low, f32_key(bf2f((uint16_t)(low | 0x8000u))));
  __syncthreads();
  // the values that are there: the largest, then their weights and counts by group
  constexpr int kPer = 2 * kVerHalf / kSampThreads;
  uint32_t n[kPer];
  int top = -1;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int i = j * kSampThreads + tid;
    n[j] = h.cnt[i];
    if (n[j]) top = max(top, i < kVerHalf ? kVerHalf + 1 + i : 2 * kVerHalf - 1 - i);
  }
  if (tid == 0 && h.zeros) top = max(top, kVerHalf);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) top = max(top, __shfl_xor(top, o, 64));
  if (lane == 0) atomicMax(&h.top, top);
  __syncthreads();
  if (h.bad || h.top < 0) return false;
  const float zmax = __fdiv_rn(ver_rank_value(h.top), p.tdiv);
  // (a row whose maximum is so low that a low value has weight; key 0: there was none)
  if (h.low && samp_weight(__fdiv_rn(key_f32(h.low), p.tdiv), zmax) != 0) return false;
  const bool use_k = p.top_k > 0 && p.top_k < V, use_p = p.top_p > 0.f && p.top_p < 1.f;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (!__ballot(n[j])) continue;
    const int i = j * kSampThreads + tid;
    const float v = bf2f((uint16_t)(kVerFirst + (i < kVerHalf ? i : i - kVerHalf + 0x8000)));
    uint64_t m = n[j] ? n[j] * samp_weight(__fdiv_rn(v, p.tdiv), zmax) : 0;
    // 16 lanes are a group: their sum to the last one
    const int g = i < kVerHalf ? (kVerHalf - 1 - i) >> 4 : i >> 4;
    m = row_total(m);
    if ((lane & 15) == 15) h.gsum[g] = m;
    if (use_k) {
      const uint32_t c = row_total(n[j]);
      if ((lane & 15) == 15) h.gcnt[g] = c;
    }
  }
  const bool zero_too = tid == kVerGroups / 2 && h.zeros;  // that group's: zero's besides
  __syncthreads();
  uint64_t mass = h.gsum[tid] + (zero_too ? h.zeros * samp_weight(0.f, zmax) : 0), W;
  const uint64_t run = block_excl_scan<kSampThreads>(mass, h.red, &W);
  VerRow o = {};
  o.zmax = zmax;
  o.lo = o.edge = -INFINITY;
  o.tie_keep = ~0ull;
  if (use_k) {  // the border's group, then its place, by the first wave's lanes
    uint64_t all;
    const uint64_t c = h.gcnt[tid] + (zero_too ? h.zeros : 0), before = block_excl_scan<kSampThreads>(c, h.red, &all);
    ver_find_group(h, before, c, (uint64_t)(p.top_k - 1));
    const int g = h.group;
    if (g >= 0) {
      if (wave == 0) {
        float v;
        const uint32_t m = ver_group_place(h, g, lane, &v);
        const uint64_t incl = wave_incl_scan((uint64_t)m);
        const int k = __ffsll((unsigned long long)__ballot(h.above + incl > (uint64_t)(p.top_k - 1))) - 1;
        const uint64_t kept = wave_total(m && lane <= k ? m * samp_weight(__fdiv_rn(v, p.tdiv), zmax) : 0);
        if (lane == k) {
          h.edge = v;
          h.weight = kept;
        }
      }
      __syncthreads();
      o.lo = h.edge;
      if (tid > g) mass = 0;
      if (tid == g) {
        mass = h.weight;
        h.above = run + mass;
      }
      __syncthreads();
      W = h.above;
    }
  }
  if (use_p) {
    const uint64_t T = (uint64_t)floor((double)p.top_p * (double)W);
    ver_find_group(h, run, mass, T);
    const int g = h.group;
    if (g >= 0) {
      if (wave == 0) {
        float v;
        const uint32_t m = ver_group_place(h, g, lane, &v);
        const uint64_t w = m && v >= o.lo ? samp_weight(__fdiv_rn(v, p.tdiv), zmax) : 0;
        const uint64_t incl = h.above + wave_incl_scan(m * w);
        const int k = __ffsll((unsigned long long)__ballot(incl > T)) - 1;
        if (lane == k) {
          const uint64_t above = incl - m * w;
          h.edge = v;
          const uint64_t keep = min((uint64_t)m, (T - above) / w + 1);
          h.tie_keep = keep == m ? ~0ull : keep;
          h.weight = above + keep * w;
        }
      }
      __syncthreads();
      o.edge = h.edge;
      o.tie_keep = h.tie_keep;
      W = h.weight;
    }
  }
  o.W = W;
  uint64_t wd = 0;
  if (d >= 0) {
    const float v = bf2f(dbits);
    bool in = v >= o.lo && v >= o.edge;
    if (in && use_p && v == o.edge && o.tie_keep != ~0ull) {  // a tie at the border: its rank in id order (uniform)
      // (the ids before it as the row is read; two values of a word at once, -0 the same as +0)
      uint32_t c = 0;
      const int whole = d & ~7;
      const uint32_t one = (dbits & 0x7fff) ? 0xffff : 0x7fff, mask = one | one << 16, want = (dbits | (uint32_t)dbits << 16) & mask;
      auto count = [&](uint32_t w) __attribute__((always_inline)) {
        const uint32_t t = (w & mask) ^ want;
        c += ((t & 0xffffu) == 0) + (t >> 16 == 0);
      };
      ver_each(x, whole, ver_load<AHEAD>(x, tid * 8, whole), [&](int, u32x4_t w) {
        count(w.x);
        count(w.y);
        count(w.z);
        count(w.w);
      });
      if (whole + tid < d) c += bf2f(x[whole + tid]) == v;
      c = wave_total(c);
      if (lane == 0 && c) atomicAdd(&h.before, c);
      __syncthreads();
      in = h.before < o.tie_keep;
    }
    if (in) wd = samp_weight(__fdiv_rn(v, p.tdiv), zmax);
  }
  if (tid == 0) {
    o.p = (float)((double)wd / (double)W);
    o.accept = ver_accepts(a, row, d, wd, W);
    *out = o;
  }
  return true;
}

// A row a workgroup.  With more rows than CUs two workgroups a CU, so that one's counting hides part of the other's sums (1,152 rows 118
// us; one a CU with twice the loads ahead 122); otherwise one, which has the registers for that (120 rows 26 us for 30).
template <int PER_CU, int AHEAD>
__global__ __launch_bounds__(kSampThreads, 4 * PER_CU) void verify_rows_kernel(VerArgs a, VerRow* __restrict__ rows) {
  __shared__ union { VerHist hist; VerGreedy greedy; SampShared gen; } sh;
  __shared__ int found;
  const int row = blockIdx.x;
  const VerLoaded<AHEAD> l = ver_load<AHEAD>(a.logits + (size_t)row * a.V, (int)threadIdx.x * 8, a.V & ~7);  // while the stream is looked up
  const int s = ver_stream(a, row, &found);
  if (s < 0) return;
  const VerParams p = ver_params(a, s);
  if (!(p.temp > 0.f)) {
    ver_row_greedy(a, row, l, sh.greedy, rows + row);
    return;
  }
  if (ver_row_counts(a, row, p, l, sh.hist, rows + row)) return;
  __syncthreads();  // every thread has read the union's other side
  ver_row_general(a, row, p, sh.gen, rows + row);
}

// the first of a stream's rows that ends it (its end: none does); every thread gets it
__device__ __forceinline__ int ver_stop(const VerArgs& a, const VerRow* __restrict__ rows, int2 range, int* red) {
  if (threadIdx.x == 0) *red = range.y;
  __syncthreads();
  for (int r = range.x + (int)threadIdx.x; r < range.y; r += blockDim.x)
    if (!rows[r].accept) atomicMin(red, r);
  __syncthreads();
  return *red;
}

// w' of one id, but for a tie's rank: 0 below the filter's bounds; *tie: it is a boundary tie
struct VerWeights {
  const uint16_t* x;
  const float* q;
  float tdiv, zmax, lo, edge;
  bool by_z;
  double W;
  int d;  // the rejected draft, where no distribution goes with it (else -1)

  __device__ __forceinline__ double kept(uint32_t bits, bool* tie) const {
    const float v = bf2f((uint16_t)bits), y = by_z ? __fdiv_rn(v, tdiv) : v;
    *tie = y == edge;
    if (!(y >= lo && y >= edge)) return 0.0;
    return samp_weight_f64(by_z ? y : __fdiv_rn(v, tdiv), zmax);
  }
  __device__ __forceinline__ double rest(int v, double w) const { return v == d ? 0.0 : q ? ver_rest(w, q[v], W) : w; }
};

__device__ __forceinline__ VerWeights ver_weights(const VerArgs& a, int s, int row, const VerRow& r) {
  const int d = ver_draft(a, row);
  const float* q = d >= 0 ? ver_probs(a, row) : nullptr;
  return {a.logits + (size_t)row * a.V, q, ver_params(a, s).tdiv, r.zmax, r.lo, r.edge, r.by_z != 0, (double)r.W, q ? -1 : d};
}

// w' of the stop row's pieces, a wave each at a time, the next one's loads in flight.  A piece's sums stay below 2^49 and are exact in
// doubles.  Without a filter nearly every token has weight: a workgroup with many pieces makes the weights of the common values once
// (|x| in [2^-24, 2^8)) and looks them up; the others are made one by one.  128 streams 35 us with the tables (one of 1,024 threads a
// CU; 47 with four of 256 threads, which make it four times), 73 without; the unfiltered ones among 24 streams 11 and 17.
constexpr int kVerTable = 32 * 128;      // values of a sign
constexpr uint32_t kVerTableFirst = 0x3380;  // the bits of 2^-24
constexpr int kPieceThreads = 1024;
constexpr int kTablePieces = 32;  // of a workgroup, for a table: twice as many tokens as it has values

struct __attribute__((packed, aligned(4))) VerVec4 { f32x4_t v; };

__global__ __launch_bounds__(kPieceThreads, 4) void verify_pieces_kernel(VerArgs a, const VerRow* __restrict__ rows,
                                                                         VerPiece* __restrict__ pieces) {
  __shared__ double table[2 * kVerTable + 1];  // the last one: 0
  __shared__ int stop_s;
  const int s = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int2 range = ver_range(a, s);
  const int stop = ver_stop(a, rows, range, &stop_s);
  if (stop >= range.y) return;
  if (!(ver_params(a, s).temp > 0.f)) return;
  const VerRow r = rows[stop];
  const VerWeights w = ver_weights(a, s, stop, r);
  struct Loaded {
    uint32_t x[4];
    f32x4_t q[2];
  };
  const int last = a.V >= 8 ? a.V - 8 : 0;
  // 8 ids a lane; where the row ends within them, the row's last 8 (those before the lane's ids are taken out below)
  auto load = [&](int c) __attribute__((always_inline)) {
    Loaded l = {};
    const int v = min(c * kPiece + lane * 8, last);
    if (a.V >= 8) {
      const u32x4_t x = reinterpret_cast<const VerVec*>(w.x + v)->v;
#pragma unroll
      for (int j = 0; j < 4; ++j) l.x[j] = x[j];
      if (w.q) {
        l.q[0] = reinterpret_cast<const VerVec4*>(w.q + v)->v;
        l.q[1] = reinterpret_cast<const VerVec4*>(w.q + v + 4)->v;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (j < a.V) {
          l.x[j >> 1] |= (uint32_t)w.x[j] << (16 * (j & 1));
          if (w.q) l.q[j >> 2][j & 3] = w.q[j];
        }
    }
    return l;
  };
  const int step = gridDim.x * (kPieceThreads / 64);
  int c = blockIdx.x * (kPieceThreads / 64) + wave;
  Loaded next = {};
  if (c < a.pieces) next = load(c);
  const bool look_up = r.lo == -INFINITY && r.edge == -INFINITY && a.pieces >= kTablePieces * (int)gridDim.x;
  if (look_up) {
    for (int i = threadIdx.x; i < 2 * kVerTable; i += kPieceThreads) {
      const uint32_t bits = kVerTableFirst + (i < kVerTable ? i : i - kVerTable + 0x8000u);
      const float z = __fdiv_rn(bf2f((uint16_t)bits), w.tdiv);
      table[i] = z <= w.zmax ? samp_weight_f64(z, w.zmax) : 0.0;  // (no value of the row lies above)
    }
    if (threadIdx.x == 0) table[2 * kVerTable] = 0.0;
    __syncthreads();
  }
  const float down = (w.zmax - 28.f) * w.tdiv, least = down - fabsf(down) * 0x1p-20f;  // below it there is no weight (that starts 27.75 down)
  for (; c < a.pieces; c += step) {
    Loaded l = next;
    if (c + step < a.pieces) next = load(c + step);
    const int first = c * kPiece + lane * 8, v0 = min(first, last);
    const int no = look_up ? w.d : -1;  // (a filter counts the draft among its ties)
    if ((c + 1) * kPiece > a.V || (no >= 0 && no / kPiece == c)) {  // ids that are others' or none, and the draft: -inf has no weight
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int v = v0 + j;
        if (v < first || v >= a.V || v == no) l.x[j >> 1] = j & 1 ? (l.x[j >> 1] & 0xffffu) | 0xff800000u : (l.x[j >> 1] & 0xffff0000u) | 0xff80u;
      }
    }
    double above = 0, tie = 0;
    uint32_t ties = 0;
    if (look_up) {
      typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
      uint32_t at[4], odd = 0;  // byte addresses of a word's two values; the bits that tell values outside the table
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u16x2 t2 = __builtin_bit_cast(u16x2, l.x[i]);
        t2 -= (u16x2){(unsigned short)kVerTableFirst, (unsigned short)kVerTableFirst};
        const uint32_t t = __builtin_bit_cast(uint32_t, t2);
        at[i] = ((t << 3) & 0x7ff87ff8u) | (t & 0x80008000u);
        odd |= ((t & 0x70000000u) ? 2u : 0u) << (2 * i) | ((t & 0x7000u) ? 1u : 0u) << (2 * i);
      }
      const char* tab = reinterpret_cast<const char*>(table);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t b = j & 1 ? at[j >> 1] >> 16 : at[j >> 1] & 0xffffu;
        if (odd >> j & 1) b = 2 * kVerTable * 8;
        double k = *reinterpret_cast<const double*>(tab + b);
        if (w.q) k = ver_rest(k, l.q[j >> 2][j & 3], w.W);
        above += k;
      }
      if (odd) {  // (masked ids and the like have no weight)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (bf2f((uint16_t)(j & 1 ? l.x[j >> 1] >> 16 : l.x[j >> 1])) < least) odd &= ~(1u << j);
      }
      while (odd) {  // a lane's next value that has no entry
        const int v = v0 + __ffs(odd) - 1;
        odd &= odd - 1;
        bool none;
        if (v >= first && v < a.V && v != w.d) above += w.rest(v, w.kept(w.x[v], &none));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        bool is_tie;
        double k = w.kept(j & 1 ? l.x[j >> 1] >> 16 : l.x[j >> 1] & 0xffffu, &is_tie);
        if (w.q) k = ver_rest(k, l.q[j >> 2][j & 3], w.W);
        if (v0 + j == w.d) k = 0.0;
        if (is_tie) {
          tie += k;
          ++ties;
        } else {
          above += k;
        }
      }
    }
    const bool apart = r.tie_keep != ~0ull;  // some ties are kept and some are not (uniform)
    above = wave_total(apart ? above : above + tie);
    if (apart) {
      tie = wave_total(tie);
      ties = wave_total(ties);
    } else {
      tie = 0;
      ties = 0;
    }
    if (lane == 0) pieces[(size_t)s * a.pieces + c] = {(uint64_t)above, (uint64_t)tie, ties, 0};
  }
}

// A stream a workgroup: two sums over its pieces, one over the ids of the piece that is hit, and of the one whose ties are kept in part;
// a chain of round trips (5 to 8 us).
__global__ __launch_bounds__(kPiece) void verify_draw_kernel(VerArgs a, const VerRow* __restrict__ rows,
                                                             const VerPiece* __restrict__ pieces, int32_t* __restrict__ tokens,
                                                             int32_t* __restrict__ counts, float* __restrict__ p_out) {
  __shared__ uint64_t red[kPiece / 64];
  __shared__ int stop_s, hit_s, part_s, first_s;
  __shared__ uint64_t left_s, part_before_s, hit_before_s, part_sum_s;
  const int s = blockIdx.x, tid = threadIdx.x;
  const int2 range = ver_range(a, s);
  const int stop = ver_stop(a, rows, range, &stop_s);
  for (int r = range.x + tid; r < range.y; r += kPiece) {
    if (r == stop) continue;
    tokens[r] = r < stop ? a.draft[r] : -1;
    p_out[r] = r < stop ? rows[r].p : 0.f;
  }
  if (tid == 0) {
    counts[s] = min(stop + 1, range.y) - range.x;
    part_s = hit_s = -1;
    first_s = INT32_MAX;
  }
  if (stop >= range.y) return;
  const VerRow r = rows[stop];
  if (!(ver_params(a, s).temp > 0.f)) {
    if (tid == 0) {
      tokens[stop] = r.arg;
      p_out[stop] = 1.f;
    }
    return;
  }
  const VerWeights w = ver_weights(a, s, stop, r);
  // one id of a piece a thread: its w' and kept weight, with `before` ties in the pieces before
  auto one = [&](int c, uint64_t before, double* kept) __attribute__((always_inline)) -> uint64_t {
    const int v = c * kPiece + tid;
    bool tie = false;
    double k = v < a.V ? w.kept(w.x[v], &tie) : 0.0;
    if (r.tie_keep != ~0ull) {  // uniform
      uint64_t n;
      const uint64_t rank = before + block_excl_scan<kPiece>((uint64_t)tie, red, &n);
      if (tie && rank >= r.tie_keep) k = 0.0;
    }
    *kept = k;
    return v < a.V ? (uint64_t)w.rest(v, k) : 0;
  };
  // a run of consecutive pieces a thread; the one whose ties are kept in part is summed anew
  const VerPiece* mine = pieces + (size_t)s * a.pieces;
  const int per = (a.pieces + kPiece - 1) / kPiece, c0 = min(a.pieces, tid * per), c1 = min(a.pieces, c0 + per);
  uint64_t ties = 0, all;
  for (int c = c0; c < c1; ++c) ties += mine[c].ties;
  const uint64_t ties0 = r.tie_keep != ~0ull ? block_excl_scan<kPiece>(ties, red, &all) : 0;
  uint64_t t = ties0;
  __syncthreads();
  for (int c = c0; c < c1; ++c) {
    const uint64_t n = mine[c].ties;
    if (t < r.tie_keep && t + n > r.tie_keep) {
      part_s = c;
      part_before_s = t;
    }
    t += n;
  }
  __syncthreads();
  if (part_s >= 0) {  // uniform
    double kept;
    uint64_t total;
    const uint64_t k = one(part_s, part_before_s, &kept);
    block_excl_scan<kPiece>(k, red, &total);
    if (tid == 0) part_sum_s = total;
    __syncthreads();
  }
  auto sum_of = [&](int c, uint64_t before) __attribute__((always_inline)) {
    const VerPiece m = mine[c];
    return c == part_s ? part_sum_s : m.above + (before + m.ties <= r.tie_keep ? m.tie : 0);
  };
  uint64_t sum = 0, total;
  t = ties0;
  for (int c = c0; c < c1; ++c) {
    sum += sum_of(c, t);
    t += mine[c].ties;
  }
  uint64_t run = block_excl_scan<kPiece>(sum, red, &total);
  uint64_t target = (uint64_t)(ver_uniform(a.u_draw[s]) * (double)total);
  target = total && target >= total ? total - 1 : target;
  if (target >= run && target < run + sum) {  // one thread, unless nothing is left
    t = ties0;
    for (int c = c0; c < c1; ++c) {
      const uint64_t n = sum_of(c, t);
      if (target >= run && target < run + n) {
        hit_s = c;
        left_s = target - run;
        hit_before_s = t;
      }
      run += n;
      t += mine[c].ties;
    }
  }
  __syncthreads();
  if (hit_s >= 0) {
    double kept;
    const uint64_t k = one(hit_s, hit_before_s, &kept);
    run = block_excl_scan<kPiece>(k, red, &all);
    if (left_s >= run && left_s < run + k) {
      tokens[stop] = hit_s * kPiece + tid;
      p_out[stop] = (float)(kept / (double)r.W);
    }
    return;
  }
  // nothing is left: the first id of maximal weight (the ties at the filter's border keep its first, which is the only one that counts here).
  // It has a place of its own: waves that come late still read hit_s above, and no barrier lies between.
  uint64_t best = 0;
  int at = INT32_MAX;
  for (int v = tid; v < a.V; v += kPiece) {
    bool tie;
    const uint64_t k = (uint64_t)w.kept(w.x[v], &tie);
    if (k > best) {
      best = k;
      at = v;
    }
  }
  uint64_t top = best;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const uint64_t y = __shfl_xor(top, o, 64);
    top = y > top ? y : top;
  }
  if ((tid & 63) == 0) red[tid >> 6] = top;
  __syncthreads();
  for (int i = 0; i < kPiece / 64; ++i) top = red[i] > top ? red[i] : top;
  if (best == top) atomicMin(&first_s, at);
  __syncthreads();
  if (tid == 0) {
    tokens[stop] = top ? first_s : 0;
    p_out[stop] = top ? (float)((double)top / (double)r.W) : 0.f;
  }
}

}  // namespace flyai

using namespace flyai;

extern "C" size_t flyai_spec_verify_workspace_bytes(int32_t R, int32_t V, int32_t S) {
  if (R < 0 || V < 1 || V > (1 << 22) || S < 0) return 0;
  return (size_t)R * sizeof(VerRow) + (size_t)S * ceil_div(V, kPiece) * sizeof(VerPiece);
}

extern "C" int flyai_spec_verify(const uint16_t* logits, int32_t R, int32_t V, const int32_t* cu_rows, int32_t S, const int32_t* draft,
                                 const double* u, const double* u_draw, const float* temps, const int32_t* top_ks, const float* top_ps,
                                 float temp, int32_t top_k, float top_p, const float* draft_probs, int32_t n_probs,
                                 const int32_t* probs_row, int32_t* tokens, int32_t* counts, float* p, void* workspace,
                                 flyai_stream_t stream) {
  FLYAI_REQUIRE(R >= 0 && S >= 0 && V >= 1 && V <= (1 << 22), "spec_verify: needs R, S >= 0 and V in [1, 2^22]");
  FLYAI_REQUIRE(R < (1 << 22), "spec_verify: %d rows, a launch takes 2^22 - 1 workgroups of 1,024 threads", R);
  FLYAI_REQUIRE(S <= 65535, "spec_verify: n_streams %d above 65535", S);
  if (S == 0) return FLYAI_OK;
  FLYAI_REQUIRE(cu_rows && counts && u_draw && (R == 0 || (logits && draft && u && tokens && p && workspace)), "spec_verify: null pointer");
  FLYAI_REQUIRE(!draft_probs || n_probs >= 0, "spec_verify: bad n_probs");
  FLYAI_REQUIRE(!draft_probs || probs_row || n_probs == R, "spec_verify: draft_probs of other rows need probs_row");
  FLYAI_REQUIRE(top_k >= 0, "spec_verify: top_k must be >= 0");
  FLYAI_REQUIRE(((uintptr_t)workspace & 7) == 0, "spec_verify: the workspace must be 8-byte aligned");
  const VerArgs a = {logits, cu_rows, draft, u, u_draw, temps, top_ps, top_ks, temp, top_p, top_k, draft_probs, probs_row, n_probs, R, V, S,
                     ceil_div(V, kPiece)};
  VerRow* rows = static_cast<VerRow*>(workspace);
  VerPiece* pieces = reinterpret_cast<VerPiece*>(rows + R);
  hipStream_t s = as_stream(stream);
  if (R > 0) {
    if (R > device_cus())
      hipLaunchKernelGGL((verify_rows_kernel<2, 2>), dim3(R), dim3(kSampThreads), 0, s, a, rows);
    else
      hipLaunchKernelGGL((verify_rows_kernel<1, 4>), dim3(R), dim3(kSampThreads), 0, s, a, rows);
    // a workgroup a CU, a piece a wave at least
    const int wgs = std::max(1, std::min(ceil_div(a.pieces, kPieceThreads / 64), device_cus() / S));
    hipLaunchKernelGGL(verify_pieces_kernel, dim3(wgs, S), dim3(kPieceThreads), 0, s, a, rows, pieces);
  }
  hipLaunchKernelGGL(verify_draw_kernel, dim3(S), dim3(kPiece), 0, s, a, rows, pieces, tokens, counts, p);
  return check_launch("spec_verify");
}
