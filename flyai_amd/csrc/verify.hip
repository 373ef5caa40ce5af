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
// is not is then the only one whose weights are needed one by one: verify_chunks_kernel sums w' over chunks of its ids, and
// verify_draw_kernel finds the chunk and the id, and writes what comes out.
#include <algorithm>

#include "sample.h"

namespace flyai {

struct VerRow {
  uint64_t W;         // kept weight
  uint64_t tie_keep;  // ties at pkey that are kept, in id order
  float zmax;
  uint32_t kkey, pkey;  // f32 keys: z >= kkey and above pkey (0: no such bound) are kept
  int32_t accept;
  int32_t arg;        // greedy: the first id of maximal logit
  float p;            // the draft's probability
};

struct VerChunk {
  uint64_t above, tie;  // w' of the chunk's kept tokens above pkey, of all its ties at pkey
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
  int32_t n_probs, R, V, S, chunk, n_chunks;
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

// what a rejected draft's distribution takes from a weight
__device__ __forceinline__ uint64_t ver_rest(uint64_t w, float q, uint64_t W) {
  const double t = floor((double)fmaxf(q, 0.f) * (double)W);
  return t >= (double)w ? 0 : w - (uint64_t)t;
}

// One row by a workgroup, for any logits: every pass reads the row again.
__device__ __forceinline__ void ver_row_general(const VerArgs& a, int row, const VerParams& p, SampShared& sh, VerRow* out) {
  const uint16_t* x = a.logits + (size_t)row * a.V;
  const int tid = threadIdx.x, V = a.V, d = ver_draft(a, row);
  VerRow o = {};
  if (!(p.temp > 0.f)) {
    uint64_t best = 0;
    for (int v = tid; v < V; v += kSampThreads) {
      const uint64_t k = ((uint64_t)f32_key(bf2f(x[v])) << 32) | (uint32_t)~v;
      best = k > best ? k : best;
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
      const uint64_t y = __shfl_xor(best, off, 64);
      best = y > best ? y : best;
    }
    __syncthreads();
    if ((tid & 63) == 0) sh.red64[tid >> 6] = best;
    __syncthreads();
    for (int w = 0; w < kSampWaves; ++w) best = sh.red64[w] > best ? sh.red64[w] : best;
    o.arg = (int)~(uint32_t)best;
    o.accept = d == o.arg;
    o.p = d == o.arg ? 1.f : 0.f;
    if (tid == 0) *out = o;
    return;
  }
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
  o.kkey = kth;
  uint64_t sum = 0;
  for (int v = tid; v < V; v += kSampThreads) {
    uint32_t k;
    if (kept_k(v, &k)) sum += samp_weight(zof(v), o.zmax);
  }
  o.W = block_sum(sum, sh.red64);
  o.tie_keep = ~0ull;
  if (p.top_p > 0.f && p.top_p < 1.f) {
    const uint64_t T = (uint64_t)floor((double)p.top_p * (double)o.W);
    uint64_t above = 0;
    o.pkey = radix_select(V, kept_k, [&](int v) { return samp_weight(zof(v), o.zmax); }, T, &above, sh);
    if (o.pkey) {
      // tie j (0-based, id order) of the boundary value is kept iff above + j * wb <= T (tie 0 always is)
      const uint64_t wb = samp_weight(key_f32(o.pkey), o.zmax);
      uint32_t ties = 0;
      for (int v = tid; v < V; v += kSampThreads) ties += f32_key(zof(v)) == o.pkey;
      const uint64_t n = block_sum((uint64_t)ties, sh.red64);
      o.tie_keep = wb == 0 ? n : min(n, (T - above) / wb + 1);
      o.W = above + o.tie_keep * wb;
    }
  }
  // the draft's weight; as a boundary tie it counts if its rank among the ties is kept
  uint64_t wd = 0;
  if (d >= 0) {
    const uint32_t k = f32_key(zof(d));
    bool kept = k >= kth && k >= o.pkey;
    if (kept && o.pkey && k == o.pkey) {
      uint32_t before = 0;
      for (int v = tid; v < d; v += kSampThreads) before += f32_key(zof(v)) == o.pkey;
      kept = block_sum((uint64_t)before, sh.red64) < o.tie_keep;
    }
    if (kept) wd = samp_weight(zof(d), o.zmax);
  }
  if (tid) return;
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

__global__ __launch_bounds__(kSampThreads) void verify_rows_kernel(VerArgs a, VerRow* __restrict__ rows) {
  __shared__ SampShared sh;
  __shared__ int found;
  const int row = blockIdx.x, s = ver_stream(a, row, &found);
  if (s < 0) return;
  ver_row_general(a, row, ver_params(a, s), sh, rows + row);
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
  float tdiv, zmax;
  uint32_t kkey, pkey;
  uint64_t W;
  int d;  // the rejected draft, where no distribution goes with it (else -1)

  __device__ __forceinline__ uint64_t kept(uint16_t bits, bool* tie) const {
    const float z = __fdiv_rn(bf2f(bits), tdiv);
    const uint32_t k = f32_key(z);
    *tie = false;
    if (k < kkey || k < pkey) return 0;
    *tie = pkey != 0 && k == pkey;
    return samp_weight(z, zmax);
  }
  __device__ __forceinline__ uint64_t rest(int v, uint64_t w) const { return v == d ? 0 : q && w ? ver_rest(w, q[v], W) : w; }
};

__device__ __forceinline__ VerWeights ver_weights(const VerArgs& a, int s, int row, const VerRow& r) {
  const int d = ver_draft(a, row);
  const float* q = d >= 0 ? ver_probs(a, row) : nullptr;
  return {a.logits + (size_t)row * a.V, q, ver_params(a, s).tdiv, r.zmax, r.kkey, r.pkey, r.W, q ? -1 : d};
}

__global__ __launch_bounds__(kChunkThreads) void verify_chunks_kernel(VerArgs a, const VerRow* __restrict__ rows,
                                                                      VerChunk* __restrict__ chunks) {
  __shared__ uint64_t red[kChunkThreads / 64];
  __shared__ int stop_s;
  const int c = blockIdx.x, s = blockIdx.y;
  const int2 range = ver_range(a, s);
  const int stop = ver_stop(a, rows, range, &stop_s);
  if (stop >= range.y) return;
  if (!(ver_params(a, s).temp > 0.f)) return;
  const VerRow r = rows[stop];
  const VerWeights w = ver_weights(a, s, stop, r);
  uint64_t above = 0, tie = 0, total;
  uint32_t ties = 0;
  for_chunk(w.x, c * a.chunk, min(a.V, (c + 1) * a.chunk), a.V % 8 == 0 && ((uintptr_t)a.logits & 15) == 0, [&](int v, uint16_t bits) {
    bool is_tie;
    const uint64_t k = w.rest(v, w.kept(bits, &is_tie));
    if (is_tie) {
      tie += k;
      ++ties;
    } else {
      above += k;
    }
  });
  VerChunk o;
  block_excl_scan<kChunkThreads>(above, red, &total);
  o.above = total;
  block_excl_scan<kChunkThreads>(tie, red, &total);
  o.tie = total;
  block_excl_scan<kChunkThreads>((uint64_t)ties, red, &total);
  o.ties = (uint32_t)total;
  o.pad = 0;
  if (threadIdx.x == 0) chunks[(size_t)s * a.n_chunks + c] = o;
}

// The ids of chunk c of which thread t has a run of consecutive ones, their ties ranked from `rank` on: f(id, w') in order.
template <class F>
__device__ __forceinline__ void ver_walk(const VerArgs& a, const VerWeights& w, int v0, int v1, uint64_t rank, uint64_t tie_keep, F&& f) {
  for (int v = v0; v < v1; ++v) {
    bool tie;
    uint64_t k = w.kept(w.x[v], &tie);
    if (tie && rank++ >= tie_keep) k = 0;
    f(v, w.rest(v, k), k);
  }
}

__global__ __launch_bounds__(kSampThreads) void verify_draw_kernel(VerArgs a, const VerRow* __restrict__ rows,
                                                                   const VerChunk* __restrict__ chunks, int32_t* __restrict__ tokens,
                                                                   int32_t* __restrict__ counts, float* __restrict__ p_out) {
  __shared__ uint64_t red[kSampWaves];
  __shared__ uint64_t sum_s[kMaxChunks], tie_s[kMaxChunks];
  __shared__ int stop_s, hit_s, part_s;
  __shared__ uint64_t left_s;
  const int s = blockIdx.x, tid = threadIdx.x;
  const int2 range = ver_range(a, s);
  const int stop = ver_stop(a, rows, range, &stop_s);
  for (int r = range.x + tid; r < range.y; r += kSampThreads) {
    if (r == stop) continue;
    tokens[r] = r < stop ? a.draft[r] : -1;
    p_out[r] = r < stop ? rows[r].p : 0.f;
  }
  if (tid == 0) counts[s] = min(stop + 1, range.y) - range.x;
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
  auto run_of = [&](int c, int* v0, int* v1) __attribute__((always_inline)) {
    const int c0 = c * a.chunk, c1 = min(a.V, c0 + a.chunk), per = (c1 - c0 + kSampThreads - 1) / kSampThreads;
    *v0 = min(c1, c0 + tid * per);
    *v1 = min(c1, *v0 + per);
  };
  // the rank of a thread's first tie
  auto rank_of = [&](int c, int v0, int v1) __attribute__((always_inline)) {
    uint64_t n = 0, all;
    for (int v = v0; v < v1; ++v) {
      bool tie;
      w.kept(w.x[v], &tie);
      n += tie;
    }
    return tie_s[c] + block_excl_scan<kSampThreads>(n, red, &all);
  };
  // every chunk's w', and the one whose ties are kept in part
  if (tid == 0) part_s = -1;
  __syncthreads();
  if (tid < 64) {
    VerChunk c = {0, 0, 0, 0};
    if (tid < a.n_chunks) c = chunks[(size_t)s * a.n_chunks + tid];
    const uint64_t before = wave_incl_scan((uint64_t)c.ties) - c.ties;
    tie_s[tid] = before;
    sum_s[tid] = c.above + (before + c.ties <= r.tie_keep ? c.tie : 0);
    if (before < r.tie_keep && before + c.ties > r.tie_keep) part_s = tid;
  }
  __syncthreads();
  if (part_s >= 0) {  // uniform
    int v0, v1;
    run_of(part_s, &v0, &v1);
    uint64_t mine = 0, total;
    const uint64_t rank = rank_of(part_s, v0, v1);
    ver_walk(a, w, v0, v1, rank, r.tie_keep, [&](int, uint64_t k, uint64_t) { mine += k; });
    block_excl_scan<kSampThreads>(mine, red, &total);
    if (tid == 0) sum_s[part_s] = total;
    __syncthreads();
  }
  if (tid < 64) {
    const uint64_t n = sum_s[tid], incl = wave_incl_scan(n), total = __shfl(incl, 63, 64);
    if (tid == 0) hit_s = -1;
    uint64_t target = (uint64_t)(ver_uniform(a.u_draw[s]) * (double)total);
    target = total && target >= total ? total - 1 : target;
    if (target >= incl - n && target < incl) {
      hit_s = tid;
      left_s = target - (incl - n);
    }
  }
  __syncthreads();
  const int c = hit_s;
  if (c >= 0) {
    int v0, v1;
    run_of(c, &v0, &v1);
    const uint64_t rank = rank_of(c, v0, v1);
    uint64_t mine = 0, total;
    ver_walk(a, w, v0, v1, rank, r.tie_keep, [&](int, uint64_t k, uint64_t) { mine += k; });
    uint64_t run = block_excl_scan<kSampThreads>(mine, red, &total);
    if (left_s >= run && left_s < run + mine) {
      bool done = false;
      ver_walk(a, w, v0, v1, rank, r.tie_keep, [&](int v, uint64_t k, uint64_t full) {
        run += k;
        if (!done && run > left_s) {
          done = true;
          tokens[stop] = v;
          p_out[stop] = (float)((double)full / (double)r.W);
        }
      });
    }
    return;
  }
  // nothing is left: the first id of maximal weight (the ties at the filter's border keep its first, which is the only one that counts here)
  uint64_t best = 0;
  int at = 0x7fffffff;
  for (int v = tid; v < a.V; v += kSampThreads) {
    bool tie;
    const uint64_t k = w.kept(w.x[v], &tie);
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
  if (tid == 0) hit_s = 0x7fffffff;
  __syncthreads();
  for (int i = 0; i < kSampWaves; ++i) top = red[i] > top ? red[i] : top;
  if (best == top) atomicMin(&hit_s, at);
  __syncthreads();
  if (tid == 0) {
    tokens[stop] = top ? hit_s : 0;
    p_out[stop] = top ? (float)((double)top / (double)r.W) : 0.f;
  }
}

static void verify_chunks(int V, int* chunk, int* n_chunks) {
  const int steps = (int)(((int64_t)V + (int64_t)kMaxChunks * kChunkStep - 1) / ((int64_t)kMaxChunks * kChunkStep));
  *chunk = std::max(kMinChunk, steps * kChunkStep);
  *n_chunks = ceil_div(V, *chunk);
}

}  // namespace flyai

using namespace flyai;

extern "C" size_t flyai_spec_verify_workspace_bytes(int32_t R, int32_t V, int32_t S) {
  if (R < 0 || V < 1 || V > (1 << 22) || S < 0) return 0;
  int chunk, n;
  verify_chunks(V, &chunk, &n);
  return (size_t)R * sizeof(VerRow) + (size_t)S * n * sizeof(VerChunk);
}

extern "C" int flyai_spec_verify(const uint16_t* logits, int32_t R, int32_t V, const int32_t* cu_rows, int32_t S, const int32_t* draft,
                                 const double* u, const double* u_draw, const float* temps, const int32_t* top_ks, const float* top_ps,
                                 float temp, int32_t top_k, float top_p, const float* draft_probs, int32_t n_probs,
                                 const int32_t* probs_row, int32_t* tokens, int32_t* counts, float* p, void* workspace,
                                 flyai_stream_t stream) {
  FLYAI_REQUIRE(R >= 0 && S >= 0 && V >= 1 && V <= (1 << 22), "spec_verify: needs R, S >= 0 and V in [1, 2^22]");
  FLYAI_REQUIRE(S <= 65535, "spec_verify: n_streams %d above 65535", S);
  if (S == 0) return FLYAI_OK;
  FLYAI_REQUIRE(cu_rows && counts && u_draw && (R == 0 || (logits && draft && u && tokens && p && workspace)), "spec_verify: null pointer");
  FLYAI_REQUIRE(!draft_probs || n_probs >= 0, "spec_verify: bad n_probs");
  FLYAI_REQUIRE(!draft_probs || probs_row || n_probs == R, "spec_verify: draft_probs of other rows need probs_row");
  FLYAI_REQUIRE(top_k >= 0, "spec_verify: top_k must be >= 0");
  FLYAI_REQUIRE(((uintptr_t)workspace & 7) == 0, "spec_verify: the workspace must be 8-byte aligned");
  VerArgs a = {logits, cu_rows, draft, u, u_draw, temps, top_ps, top_ks, temp, top_p, top_k, draft_probs, probs_row, n_probs, R, V, S, 0, 0};
  verify_chunks(V, &a.chunk, &a.n_chunks);
  VerRow* rows = static_cast<VerRow*>(workspace);
  VerChunk* chunks = reinterpret_cast<VerChunk*>(rows + R);
  hipStream_t s = as_stream(stream);
  if (R > 0) {
    hipLaunchKernelGGL(verify_rows_kernel, dim3(R), dim3(kSampThreads), 0, s, a, rows);
    hipLaunchKernelGGL(verify_chunks_kernel, dim3(a.n_chunks, S), dim3(kChunkThreads), 0, s, a, rows, chunks);
  }
  hipLaunchKernelGGL(verify_draw_kernel, dim3(S), dim3(kSampThreads), 0, s, a, rows, chunks, tokens, counts, p);
  return check_launch("spec_verify");
}
