// Low-rank adapters of many requests at once beside a shared projection.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "gemm.h"

namespace flyai {

int launch_gemm(const uint16_t* x, const uint16_t* W, int M, int N, int K, float* part, int* slices, hipStream_t s);
int launch_gemm_tiled_lora(const uint16_t* x, const uint16_t* W, const uint16_t* b, int M, int N, int K, float* out, uint16_t* y,
                           uint16_t* residual, const LoraArgs& a, hipStream_t s);
bool gemm_tiled_lora_fits(int M, int K, const LoraArgs& a);
bool gemm_is_tiled(int M);
int gemm_planes(int M, int K);

// The down product by itself, for batches whose projection takes the tiled kernel (smaller ones have it in the
// projection's launch, gemm_splitk_bf16_kernel).
constexpr int kDownTiles = 64;

__global__ __launch_bounds__(64 * kDownParts) void lora_down_kernel(const uint16_t* __restrict__ x, int M, int K, LoraArgs a) {
  __shared__ LoraDownLds<kDownParts, kDownTiles> lds;
  lora_down<kDownParts, kDownTiles>(x, M, K, a, blockIdx.x, gridDim.x, lds);
}

// ---- up, and the projection's finalize ---------------------------------------------------------------------------
// y = bf16(sum of the projection's planes + h B^T + bias); or, without planes, h B^T as a plane of its own for another
// finalize to add (-0 where a row has no adapter: x + -0 is x).
// A workgroup takes 16 rows x 16 features.  Its four waves share the adapters among the rows: each multiplies the whole
// tile with its own, and the adapter's rows keep the result.  h and B come in whole 128-byte runs and are turned round in
// LDS (the tiled GEMM's swizzle): as MFMA operands from memory, 16 rows of 64 bytes an instruction, they took 5 of the
// 10 us at 48 rows of 12 adapters.
constexpr int kUpCols = 64;  // rank columns a pass
constexpr int kUpMine = 4;   // adapters a wave: 16 rows have at most 16

struct LoraUpLds {
  char h[2][16 * 128];               // high and low terms: 16 rows of 64 columns
  char b[4][kUpMine][16 * 128];      // a wave's adapters: 16 features of 64 columns
  float d[16][17];
};

template <bool PLANE>
__global__ __launch_bounds__(256, 4) void lora_finalize_kernel(const float* __restrict__ part, int slices, int M, int N,
                                                            LoraArgs a, const uint16_t* __restrict__ b,
                                                            uint16_t* __restrict__ y, uint16_t* __restrict__ residual,
                                                            float* __restrict__ plane_out) {
  __shared__ __align__(1024) LoraUpLds l;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int f0 = blockIdx.x * 16, m0 = blockIdx.y * 16;
  const int cols = lora_cols(a.R), seg = lora_segment(a, f0);
  int2 who = a.meta[min(m0 + r, M - 1)];
  // h: the wave's four rows, 16 lanes each, 8 chunks of the high terms and 8 of the low ones
  const int hq = 4 * wave + (lane >> 4), hc = (lane & 7) ^ ((hq >> 1) & 7);
  const uint16_t* hp = a.h + ((size_t)min(m0 + hq, M - 1) * a.n_seg + seg) * 2 * cols + (lane & 8 ? cols : 0);
  u32x4_t hv = *reinterpret_cast<const u32x4_t*>(hp + min(8 * hc, cols - 8));
  // this thread's output: row 4 * wave + lane / 16, feature lane % 16
  const int mine = 4 * wave + (lane >> 4), row = m0 + mine;
  const size_t idx = (size_t)min(row, M - 1) * N + f0 + r, plane = (size_t)M * N;
  float p[8];
  uint16_t bias = 0, res = 0;
  if constexpr (!PLANE) {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = part[min(i, slices - 1) * plane + idx];
    // no load under a branch: its wait would be for everything before it
    bias = *(b ? b + f0 + r : a.B);
    res = *(residual ? residual + idx : a.B);
  }
  if (m0 + r >= M) who.y = 0;
  const bool has = __builtin_amdgcn_ds_bpermute(4 * mine, who.y) > 0;
  const int key = who.y > 0 ? who.x : -1;
  bool fresh = key >= 0;  // the first of its adapter's rows
#pragma unroll
  for (int i = 0; i < 15; ++i) fresh &= i >= r || __builtin_amdgcn_readlane(key, i) != key;
  uint64_t firsts = __ballot(fresh) & 0xffff;
  const int n = __builtin_popcountll(firsts);
  if (n > 0) {
    // the wave's adapters: every fourth
    for (int i = 0; i < wave; ++i) firsts &= firsts - 1;
    int ads[kUpMine], ranks[kUpMine];
#pragma unroll
    for (int s = 0; s < kUpMine; ++s) {
      const int at = __builtin_ctzll(firsts | 1ull << 63);
      ads[s] = firsts ? __builtin_amdgcn_readlane(who.x, at & 15) : -1;
      ranks[s] = firsts ? __builtin_amdgcn_readlane(who.y, at & 15) : 0;
      for (int i = 0; i < 4; ++i) firsts &= firsts - 1;
    }
    f32x4_t acc[kUpMine];
#pragma unroll
    for (int s = 0; s < kUpMine; ++s) acc[s] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    int top = who.y;  // the largest rank of the tile: the same in every wave
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) top = max(top, __shfl_xor(top, off, 64));
    top = __builtin_amdgcn_readfirstlane(top);
    const int frag = r * 128 + ((g ^ ((r >> 1) & 7)) << 4);
    for (int c0 = 0; c0 < top; c0 += kUpCols) {
      if (c0) {
        __syncthreads();
        hv = *reinterpret_cast<const u32x4_t*>(hp + min(c0 + 8 * hc, cols - 8));
      }
      u32x4_t bv[kUpMine][2];
#pragma unroll
      for (int s = 0; s < kUpMine; ++s)
        if (c0 < ranks[s]) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {  // 8 features an instruction
            const int q = 8 * i + (lane >> 3), c = (lane & 7) ^ ((q >> 1) & 7);
            bv[s][i] = *reinterpret_cast<const u32x4_t*>(a.B + ((size_t)ads[s] * N + f0 + q) * a.R + min(c0 + 8 * c, a.R - 8));
          }
        }
      *reinterpret_cast<u32x4_t*>(l.h[lane >> 3 & 1] + hq * 128 + 16 * (lane & 7)) = hv;
#pragma unroll
      for (int s = 0; s < kUpMine; ++s)
        if (c0 < ranks[s]) {
#pragma unroll
          for (int i = 0; i < 2; ++i) *reinterpret_cast<u32x4_t*>(l.b[wave][s] + 1024 * i + 16 * lane) = bv[s][i];
        }
      __syncthreads();
#pragma unroll
      for (int c = 0; c < kUpCols / kLoraCols; ++c) {
        const bf16x8_t hi = as_bf16x8(*reinterpret_cast<const uint4*>(l.h[0] + (frag ^ (c << 6))));
        const bf16x8_t lo = as_bf16x8(*reinterpret_cast<const uint4*>(l.h[1] + (frag ^ (c << 6))));
#pragma unroll
        for (int s = 0; s < kUpMine; ++s)
          if (c0 + kLoraCols * c < ranks[s]) {
            const bf16x8_t w = lora_within(*reinterpret_cast<const uint4*>(l.b[wave][s] + (frag ^ (c << 6))),
                                           ranks[s] - c0 - kLoraCols * c - 8 * g);
            acc[s] = mfma16x16x32(w, hi, acc[s]);
            acc[s] = mfma16x16x32(w, lo, acc[s]);
          }
      }
    }
    // lane (r, g): features 4g .. +3 of row r
#pragma unroll
    for (int s = 0; s < kUpMine; ++s)
      if (key >= 0 && key == ads[s]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) l.d[r][4 * g + i] = acc[s][i];
      }
    __syncthreads();
  }
  if (row >= M) return;
  const float up = has ? l.d[mine][r] : -0.f;
  if constexpr (PLANE) {
    plane_out[idx] = up;
  } else {
    float o = p[0];
#pragma unroll
    for (int i = 1; i < 8; ++i)
      if (i < slices) o += p[i];
    for (int i = 8; i < slices; ++i) o += part[i * plane + idx];
    const float q = bf16_round(o + up + (b ? bf2f(bias) : 0.f));
    if (residual) residual[idx] = f2bf(bf2f(res) + q);
    else y[idx] = f2bf(q);
  }
}

static size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

static size_t partial_bytes(int M, int N, int K) { return (size_t)gemm_planes(M, K) * M * N * sizeof(float); }

// No more workgroups than items there can be: a tile has at most as many adapters as rows, or as the bank.
static int down_wgs(const LoraArgs& a, int M, int split, int wgs) {
  return (int)std::min<int64_t>(wgs, (int64_t)ceil_div(M, kDownRows) * std::min({kDownRows, M, a.n}) * lora_down_groups(a) * split);
}

int launch_lora_down(const uint16_t* x, int M, int K, const LoraArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(lora_down_kernel, dim3(down_wgs(a, M, 4, device_cus())), dim3(64 * kDownParts), 0, s, x, M, K, a);
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
  // 2,880: 21.9 us with 12 workgroups for h, 26.7 with 48)
  const int wgs = down_wgs(a, M, 1, device_cus() / 2);
  const int bxs = ceil_div(N, 64);
  hipLaunchKernelGGL((gemm_splitk_bf16_kernel<4, true>), dim3(wgs + bxs * *slices), dim3(256), 0, s, x, W, M, N, K, part, a, wgs, bxs);
  return check_launch("gemm_splitk_lora");
}

int launch_gemm_lora_planes(const uint16_t* x, const uint16_t* W, int M, int N, int K, float* part, int* slices, const LoraArgs& a,
                            hipStream_t s) {
  if (gemm_tiled_lora_fits(M, K, a)) {
    *slices = 1;
    const int rc = launch_lora_down(x, M, K, a, s);
    return rc ? rc : launch_gemm_tiled_lora(x, W, nullptr, M, N, K, part, nullptr, nullptr, a, s);
  }
  const int rc = launch_gemm_lora(x, W, M, N, K, part, slices, a, s);
  if (rc) return rc;
  hipLaunchKernelGGL(lora_finalize_kernel<true>, dim3(N / 16, ceil_div(M, 16)), dim3(256), 0, s, part, 0, M, N, a, nullptr, nullptr,
                     nullptr, part + (size_t)*slices * M * N);
  ++*slices;
  return check_launch("lora_plane");
}

size_t lora_h_bytes(int M, int R, int n_seg) { return align256((size_t)M * n_seg * lora_cols(R) * 4) + align256((size_t)M * sizeof(int2)); }

void lora_bind(LoraArgs* a, char* ws, int M) {
  a->h = reinterpret_cast<uint16_t*>(ws);
  a->meta = reinterpret_cast<int2*>(ws + align256((size_t)M * a->n_seg * lora_cols(a->R) * 4));
}

int launch_linear_lora(const uint16_t* x, const uint16_t* W, const uint16_t* b, int M, int N, int K, LoraArgs a, uint16_t* y,
                       uint16_t* residual, char* ws, hipStream_t s) {
  float* part = reinterpret_cast<float*>(ws);
  lora_bind(&a, ws + align256(partial_bytes(M, N, K)), M);
  int slices = 0, rc;
  if (gemm_tiled_lora_fits(M, K, a)) {
    rc = launch_lora_down(x, M, K, a, s);
    return rc ? rc : launch_gemm_tiled_lora(x, W, b, M, N, K, nullptr, y, residual, a, s);
  }
  rc = launch_gemm_lora(x, W, M, N, K, part, &slices, a, s);
  if (rc) return rc;
  hipLaunchKernelGGL(lora_finalize_kernel<false>, dim3(N / 16, ceil_div(M, 16)), dim3(256), 0, s, part, slices, M, N, a, b, y, residual,
                     nullptr);
  return check_launch("lora_finalize");
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
  return align256(partial_bytes(M, N, K)) + lora_h_bytes(M, R, n_segments);
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
  return launch_linear_lora(x, w, b, M, N, K, a, y, residual, static_cast<char*>(workspace), as_stream(stream));
}
