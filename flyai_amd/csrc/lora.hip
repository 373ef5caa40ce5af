// Low-rank adapters of many requests at once beside a shared projection.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "gemm.h"

namespace flyai {

int launch_gemm(const uint16_t* x, const uint16_t* W, int M, int N, int K, float* part, int* slices, hipStream_t s);
int launch_gemm_tiled_lora(const uint16_t* x, const uint16_t* W, const uint16_t* b, int M, int N, int K, float* out, uint16_t* y,
                           uint16_t* residual, const LoraArgs& a, hipStream_t s);
int launch_gemm_tall_lora(const uint16_t* x, const uint16_t* W, const uint16_t* b, int M, int N, int K, float* out, uint16_t* y,
                          uint16_t* residual, const LoraArgs& a, hipStream_t s);
bool gemm_tall_pays(int M, int N);
bool gemm_tiled_lora_fits(int M, int K, const LoraArgs& a);
bool gemm_is_tiled(int M);
int gemm_planes(int M, int K);

// The down product by itself, for batches whose projection takes the tiled kernel (smaller ones have it in the
// projection's launch, gemm_splitk_bf16_kernel).
constexpr int kDownTiles = 64, kDownWindow = 2;

__global__ __launch_bounds__(64 * kDownParts) void lora_down_kernel(const uint16_t* __restrict__ x, int M, int K, LoraArgs a) {
  __shared__ LoraDownLds<kDownParts, kDownTiles, kDownWindow> lds;
  lora_down<kDownParts, kDownTiles, kDownWindow>(x, M, K, a, blockIdx.x, gridDim.x, lds);
}

// ---- up, and the projection's finalize ---------------------------------------------------------------------------
// y = bf16(sum of the projection's planes + h B^T + bias); or, without planes, h B^T as a plane of its own for another
// finalize to add (-0 where a row has no adapter: x + -0 is x).
// A wave takes 16 rows x 16 features and all of the rows' adapters, one after the other, the next one's columns on their way
// under the products: it multiplies the whole tile with an adapter, and the adapter's rows keep the result.  h and B come in
// whole 128-byte runs and are turned round in the wave's own LDS (the tiled GEMM's swizzle; as MFMA operands from memory, 16
// rows of 64 bytes an instruction, they were half of the time).  Nothing is shared, so there is no barrier.  Lane (r, g) holds
// features 4g .. +3 of row r from the planes to the result.
// 5,120 features, R = 64: 4.0 us for 1 row, 7.5 for 48 rows of 12 adapters, 8.6 for 200 rows (8 KB a row); what bounds it is a
// chain of three round trips at few rows, the planes' bytes at many.  The four waves of a workgroup sharing 16 features'
// adapters took 4.2, 8.0 and 16.4.
template <bool PLANE>
__global__ __launch_bounds__(256) void lora_finalize_kernel(const float* __restrict__ part, int slices, int M, int N,
                                                                 LoraArgs a, const uint16_t* __restrict__ b,
                                                                 uint16_t* __restrict__ y, uint16_t* __restrict__ residual,
                                                                 float* __restrict__ plane_out) {
  __shared__ __align__(1024) char stage[4][3 * 2048];  // a wave's h (high terms, low terms), an adapter's columns
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int f0 = (blockIdx.x * 4 + wave) * 16, m0 = blockIdx.y * 16;
  if (f0 >= N) return;
  char* l = stage[wave];
  const int cols = lora_cols(a.R), seg = lora_segment(a, f0), row = m0 + r;
  const int2 who = a.meta[min(row, M - 1)];
  u32x4_t hv[4];  // 8 rows an instruction
#pragma unroll
  for (int k = 0; k < 4; ++k)
    hv[k] = *reinterpret_cast<const u32x4_t*>(a.h + ((size_t)min(m0 + 8 * (k & 1) + (lane >> 3), M - 1) * a.n_seg + seg) * 2 * cols +
                                              (k & 2 ? cols : 0) + lora_chunk(8 * (k & 1), 0, cols));
  const size_t idx = (size_t)min(row, M - 1) * N + f0 + 4 * g, plane = (size_t)M * N;
  f32x4_dw p[8];
  u16x4_h bias, res;
  if constexpr (!PLANE) {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = *reinterpret_cast<const f32x4_dw*>(part + min(i, slices - 1) * plane + idx);
    // no load under a branch: its wait would be for everything before it
    bias = *reinterpret_cast<const u16x4_h*>(b ? b + f0 + 4 * g : a.B);
    res = *reinterpret_cast<const u16x4_h*>(residual ? residual + idx : a.B);
  }
  const int key = row < M && who.y > 0 ? who.x : -1;
  uint64_t todo = __ballot(key >= 0) & 0xffff;
  f32x4_t d = {-0.f, -0.f, -0.f, -0.f};
  if (todo) {
    int ad = -1, rank = 0;
    u32x4_t nb[2];
    uint32_t off[2];  // of the lane's chunks in an adapter's rows from f0 on
#pragma unroll
    for (int i = 0; i < 2; ++i) off[i] = (8 * i + (lane >> 3)) * a.R + lora_chunk(8 * i, 0, a.R);
    auto next = [&]() __attribute__((always_inline)) {
      ad = -1;
      if (!todo) return;
      const int first = __builtin_ctzll(todo);
      ad = __builtin_amdgcn_readlane(key, first), rank = __builtin_amdgcn_readlane(who.y, first);
      todo &= ~__ballot(key == ad);
      const uint16_t* B = a.B + ((size_t)ad * N + f0) * a.R;
#pragma unroll
      for (int i = 0; i < 2; ++i) nb[i] = *reinterpret_cast<const u32x4_t*>(B + off[i]);
    };
    next();
#pragma unroll
    for (int k = 0; k < 4; ++k) *reinterpret_cast<u32x4_t*>(l + 1024 * k + 16 * lane) = hv[k];
    const int frag = r * 128 + ((g ^ ((r >> 1) & 7)) << 4);
    while (ad >= 0) {
      const int now = ad, cur = rank;
      asm volatile("" ::: "memory");  // a wave's LDS operations complete in order
#pragma unroll
      for (int i = 0; i < 2; ++i) *reinterpret_cast<u32x4_t*>(l + 4096 + 1024 * i + 16 * lane) = nb[i];
      asm volatile("" ::: "memory");
      next();
      f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
      for (int c = 0; kLoraCols * c < cur; ++c) {
        const int left = cur - kLoraCols * c;
        uint4 raw, hi, lo;
        if (c < 2) {
          raw = *reinterpret_cast<const uint4*>(l + 4096 + (frag ^ (c << 6)));
          hi = *reinterpret_cast<const uint4*>(l + (frag ^ (c << 6)));
          lo = *reinterpret_cast<const uint4*>(l + 2048 + (frag ^ (c << 6)));
        } else {  // ranks past 64: straight from memory
          const uint16_t* hr = a.h + ((size_t)min(row, M - 1) * a.n_seg + seg) * 2 * cols + kLoraCols * c + 8 * g;
          raw = *reinterpret_cast<const uint4*>(a.B + ((size_t)now * N + f0 + r) * a.R + lora_col(a.R, c, g));
          hi = *reinterpret_cast<const uint4*>(hr), lo = *reinterpret_cast<const uint4*>(hr + cols);
        }
        const bf16x8_t w = left < kLoraCols ? lora_within(raw, left - 8 * g) : as_bf16x8(raw);
        acc = mfma16x16x32(w, as_bf16x8(hi), acc);
        acc = mfma16x16x32(w, as_bf16x8(lo), acc);
      }
      if (key == now) d = acc;
    }
  }
  if (row >= M) return;
  if constexpr (PLANE) {
    *reinterpret_cast<f32x4_t*>(plane_out + idx) = d;
  } else {
    f32x4_dw o = p[0];
#pragma unroll
    for (int i = 1; i < 8; ++i)
      if (i < slices) o += p[i];
    for (int i = 8; i < slices; ++i) o += *reinterpret_cast<const f32x4_dw*>(part + i * plane + idx);
    u16x4_h out;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float q = bf16_round(o[c] + d[c] + (b ? bf2f(bias[c]) : 0.f));
      out[c] = residual ? f2bf(bf2f(res[c]) + q) : f2bf(q);
    }
    *reinterpret_cast<u16x4_h*>((residual ? residual : y) + idx) = out;
  }
}

static int launch_lora_finalize(const float* part, int slices, int M, int N, const LoraArgs& a, const uint16_t* b, uint16_t* y,
                                uint16_t* residual, float* plane_out, hipStream_t s) {
  const auto kernel = plane_out ? lora_finalize_kernel<true> : lora_finalize_kernel<false>;
  hipLaunchKernelGGL(kernel, dim3(ceil_div(N, 64), ceil_div(M, 16)), dim3(256), 0, s, part, slices, M, N, a, b, y, residual, plane_out);
  return check_launch("lora_finalize");
}

static size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

static size_t partial_bytes(int M, int N, int K) { return (size_t)gemm_planes(M, K) * M * N * sizeof(float); }

// No more workgroups than items there can be: a window has at most as many adapters as rows, or as the bank, and one more
// item for every 64 rows.
static int down_wgs(const LoraArgs& a, int M, int span, int split, int wgs) {
  const int64_t pairs = (int64_t)ceil_div(M, span) * std::min({span, M, a.n}) + (M - 1) / kDownRows;
  return (int)std::min<int64_t>(wgs, pairs * lora_down_groups(a) * split);
}

int launch_lora_down(const uint16_t* x, int M, int K, const LoraArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(lora_down_kernel, dim3(down_wgs(a, M, kDownRows * kDownWindow, 4, device_cus())), dim3(64 * kDownParts), 0, s, x, M, K, a);
  return check_launch("lora_down");
}

// The projection's planes and h: one launch below the tiled kernel's rows, of the split-K kernel with four waves (with eight
// the down product's registers would not fit), the down product's own before the tiled kernel.
static int launch_gemm_lora(const uint16_t* x, const uint16_t* W, int M, int N, int K, float* part, int* slices, const LoraArgs& a,
                            hipStream_t s) {
  if (gemm_is_tiled(M)) {
    const int rc = launch_lora_down(x, M, K, a, s);
    return rc ? rc : launch_gemm(x, W, M, N, K, part, slices, s);
  }
  *slices = gemm_slices(K);
  // not split: the workgroups share the CUs with the projection's, which want all of them (200 rows of one adapter, 5,120 x
  // 2,880: 22.2 us with 12 workgroups for h, 26.3 with 48); and for more than two tiles of rows, where the projection's own
  // workgroups take long, at most one for every other CU.  24 adapters of 192 rank columns, 5,120 x 2,880, up to one a CU / half
  // of that: 30 rows 14.3 / 20.1 us, 64 rows 14.8 / 20.0, 100 rows 20.6 / 27.4, 200 rows 30.7 / 28.8
  const int wgs = down_wgs(a, M, kTiledMinRows, 1, M <= 2 * kDownRows ? device_cus() : device_cus() / 2);
  const int bxs = ceil_div(N, 64);
  hipLaunchKernelGGL((gemm_splitk_bf16_kernel<4, true>), dim3(wgs + bxs * *slices), dim3(256), 0, s, x, W, M, N, K, part, a, wgs, bxs);
  return check_launch("gemm_splitk_lora");
}

int launch_gemm_lora_planes(const uint16_t* x, const uint16_t* W, int M, int N, int K, float* part, int* slices, const LoraArgs& a,
                            hipStream_t s) {
  if (gemm_is_tiled(M)) {
    // a stage's K and segments are multiples of 64 (flyai_stage_create), and it keeps room for one plane from here on
    FLYAI_REQUIRE(gemm_tiled_lora_fits(M, K, a), "lora: planes of %d rows need K and segments in multiples of 64", M);
    *slices = 1;
    const int rc = launch_lora_down(x, M, K, a, s);
    if (rc) return rc;
    return (gemm_tall_pays(M, N) ? launch_gemm_tall_lora : launch_gemm_tiled_lora)(x, W, nullptr, M, N, K, part, nullptr, nullptr, a, s);
  }
  const int rc = launch_gemm_lora(x, W, M, N, K, part, slices, a, s);
  if (rc) return rc;
  return launch_lora_finalize(part, 0, M, N, a, nullptr, nullptr, nullptr, part + (size_t)(*slices)++ * M * N, s);
}

size_t lora_h_bytes(int M, int R, int n_seg) { return align256((size_t)M * n_seg * lora_cols(R) * 4) + align256((size_t)M * sizeof(int2)); }

void lora_bind(LoraArgs* a, char* ws, int M) {
  a->h = reinterpret_cast<uint16_t*>(ws);
  a->meta = reinterpret_cast<int2*>(ws + align256((size_t)M * a->n_seg * lora_cols(a->R) * 4));
}

int launch_linear_lora(const uint16_t* x, const uint16_t* W, const uint16_t* b, int M, int N, int K, LoraArgs a, uint16_t* y,
                       uint16_t* residual, char* ws, hipStream_t s) {
  float* part = reinterpret_cast<float*>(ws);
  const bool ends = gemm_tiled_lora_fits(M, K, a);  // the tiled kernel ends the projection: no planes
  lora_bind(&a, ws + (ends ? 0 : align256(partial_bytes(M, N, K))), M);
  int slices = 0, rc;
  if (ends) {
    rc = launch_lora_down(x, M, K, a, s);
    if (rc) return rc;
    return (gemm_tall_pays(M, N) ? launch_gemm_tall_lora : launch_gemm_tiled_lora)(x, W, b, M, N, K, nullptr, y, residual, a, s);
  }
  rc = launch_gemm_lora(x, W, M, N, K, part, &slices, a, s);
  if (rc) return rc;
  return launch_lora_finalize(part, slices, M, N, a, b, y, residual, nullptr, s);
}

int make_lora_args(LoraArgs* out, const uint16_t* A, const uint16_t* B, const float* scale, const int32_t* ranks, int n, int R,
                   const int32_t* segments, int n_seg, int N, const int32_t* adapter, const int32_t* row_seq, int n_seqs) {
  FLYAI_REQUIRE(n >= 1 && R >= 16 && R <= 128 && R % 16 == 0, "lora: needs adapters, and R in 16, 32, ..., 128");
  FLYAI_REQUIRE(segments && n_seg >= 1 && n_seg <= 4, "lora: 1 to 4 segments");
  FLYAI_REQUIRE(A && B && scale && ranks && adapter, "lora: null pointer");
  FLYAI_REQUIRE(((uintptr_t)A | (uintptr_t)B) % 16 == 0, "lora: A and B must be 16-byte aligned");
  FLYAI_REQUIRE(!row_seq || n_seqs >= 1, "lora: row_seq needs n_seqs >= 1");
  int64_t sum = 0;
  LoraArgs a{A, B, scale, ranks, adapter, row_seq, n, R, n_seg, n_seqs, {0, 0, 0}, nullptr, nullptr};
  for (int i = 0; i < n_seg; ++i) {
    FLYAI_REQUIRE(segments[i] > 0 && segments[i] % 16 == 0, "lora: segment %d of %d features: a multiple of 16", i, segments[i]);
    sum += segments[i];
    if (i < 3) a.seg_end[i] = (int)std::min<int64_t>(sum, INT32_MAX);
  }
  FLYAI_REQUIRE(sum == N, "lora: the segments' %lld features are not the projection's %d", (long long)sum, N);
  *out = a;
  return FLYAI_OK;
}

}  // namespace flyai

using namespace flyai;

extern "C" size_t flyai_linear_lora_workspace_bytes(int32_t M, int32_t N, int32_t K, int32_t R, int32_t n_segments) {
  if (M <= 0 || N <= 0 || K <= 0 || R <= 0 || n_segments <= 0) return 0;
  // of several segments the widths are not known here: they may straddle a wave's features
  const bool ends = gemm_is_tiled(M) && K % 64 == 0 && n_segments == 1;
  return (ends ? 0 : align256(partial_bytes(M, N, K))) + lora_h_bytes(M, R, n_segments);
}

extern "C" int flyai_linear_lora_bf16(const uint16_t* x, const uint16_t* w, const uint16_t* b, int32_t M, int32_t N,
                                      int32_t K, const uint16_t* lora_a, const uint16_t* lora_b, const float* scale,
                                      const int32_t* ranks, int32_t n_adapters, int32_t R, const int32_t* segments_host,
                                      int32_t n_segments, const int32_t* adapter, const int32_t* row_seq, int32_t n_seqs,
                                      uint16_t* y, uint16_t* residual, void* workspace, flyai_stream_t stream) {
  FLYAI_REQUIRE(M >= 0 && M <= (1 << 19) && N > 0 && K > 0 && N % 16 == 0 && K % 32 == 0 && K <= 8192,
                "linear_lora: need M <= %d, N %% 16 == 0, K %% 32 == 0, K <= 8192", 1 << 19);
  if (M == 0) return FLYAI_OK;  // an empty tensor has no address
  FLYAI_REQUIRE(x && w && (y || residual) && workspace, "linear_lora: null pointer");
  FLYAI_REQUIRE(((uintptr_t)x | (uintptr_t)w | (uintptr_t)y | (uintptr_t)residual | (uintptr_t)workspace) % 16 == 0,
                "linear_lora: x, w, y, residual and workspace must be 16-byte aligned");
  LoraArgs a;
  const int rc = make_lora_args(&a, lora_a, lora_b, scale, ranks, n_adapters, R, segments_host, n_segments, N, adapter, row_seq,
                                n_seqs);
  if (rc) return rc;
  // other workgroups read x while one writes its result
  const char *xb = reinterpret_cast<const char*>(x), *yb = reinterpret_cast<const char*>(residual ? residual : y);
  FLYAI_REQUIRE(xb + (size_t)M * K * 2 <= yb || yb + (size_t)M * N * 2 <= xb, "linear_lora: the result overlaps x");
  return launch_linear_lora(x, w, b, M, N, K, a, y, residual, static_cast<char*>(workspace), as_stream(stream));
}
