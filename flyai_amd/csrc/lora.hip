// Low-rank adapters of many requests at once beside a shared projection.
#include <algorithm>

#include "common.h"
#include "lora.h"

namespace flyai {

int launch_gemm(const uint16_t* x, const uint16_t* W, int M, int N, int K, float* part, int* slices, hipStream_t s);
int gemm_planes(int M, int K);

// ---- down: h = scale (x A^T) of each row's adapter ---------------------------------------------------------------
// A workgroup takes 16 rows and one chunk of 16 rank columns of one segment; its waves split K and their sums are added
// in wave order through LDS, so a row's h does not depend on its tile.  Lane (r, g) of an MFMA holds row r in both
// operands, so a row's products never meet another row's: for each adapter among the 16 rows the whole tile is
// multiplied and only its own rows keep the result.
// h is kept as two bf16 terms, the value and what its rounding left out, side by side as the 32 values of one MFMA's K:
// [row][segment][chunk][16 high | 16 low].  Against the up matrix's 16 columns, taken twice, one MFMA gives the
// product with an h of 16 significant bits (2^-17 of d at most), for the bytes of one fp32 value.
constexpr int kDownWaves = 8;

__global__ __launch_bounds__(64 * kDownWaves) void lora_down_kernel(const uint16_t* __restrict__ x, int M, int K,
                                                                    LoraArgs a, uint16_t* __restrict__ h) {
  __shared__ float red[kDownWaves][16][20];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int m0 = blockIdx.x * 16, chunks = a.R / 16;
  const int sc = blockIdx.y, seg = sc / chunks, c = sc % chunks;
  const int mine = m0 + r < M ? lora_of_row(a, m0 + r) : -1;
  const int steps = K / 32, s0 = steps * wave / kDownWaves, s1 = steps * (wave + 1) / kDownWaves;
  const uint16_t* xr = x + (size_t)min(m0 + r, M - 1) * K + 8 * g;
  uint64_t todo = __ballot(mine >= 0) & 0xffff;
  for (; todo;) {
    const int ad = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
    const uint64_t rows = __ballot(mine == ad) & 0xffff;
    todo &= ~rows;
    const int rank = lora_rank(a, ad);
    const bool live = 16 * c < rank;  // a chunk past the adapter's rank is never read
    if (live) {
      const uint16_t* ar = a.A + ((size_t)ad * a.n_seg * a.R + (size_t)seg * a.R + 16 * c + r) * K + 8 * g;
      f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
      for (int s = s0; s < s1; ++s)
        acc = mfma16x16x32(as_bf16x8(*reinterpret_cast<const uint4*>(ar + 32 * s)),
                           as_bf16x8(*reinterpret_cast<const uint4*>(xr + 32 * s)), acc);
      // lane (r, g): rank columns 4g .. +3 of row r
      if (mine == ad) *reinterpret_cast<f32x4_t*>(&red[wave][r][4 * g]) = acc;
    }
  }
  __syncthreads();
  const int row = threadIdx.x >> 4, j = threadIdx.x & 15;
  if (row < 16 && m0 + row < M) {
    const int ad = lora_of_row(a, m0 + row);
    const int rank = ad >= 0 ? lora_rank(a, ad) : 0;
    if (16 * c < rank) {
      float v = red[0][row][j];
#pragma unroll
      for (int w = 1; w < kDownWaves; ++w) v += red[w][row][j];
      v = 16 * c + j < rank ? v * a.scale[ad] : 0.f;
      const uint16_t hi = f2bf(v);
      // a value past bf16's range keeps its infinity: inf - inf would make it NaN
      const float rest = v - bf2f(hi);
      uint16_t* o = h + (((size_t)(m0 + row) * a.n_seg + seg) * chunks + c) * 32 + j;
      o[0] = hi;
      o[16] = rest == rest ? f2bf(rest) : 0;
    }
  }
}

// ---- up: y = bf16(sum of the projection's planes + h B^T + bias) -------------------------------------------------
// A wave takes 16 rows x 16 features: lane (r, g) holds features 4g .. +3 of row r.
__global__ __launch_bounds__(256) void lora_finalize_kernel(const float* __restrict__ part, int slices, int M, int N,
                                                            LoraArgs a, const uint16_t* __restrict__ h,
                                                            const uint16_t* __restrict__ b, uint16_t* __restrict__ y,
                                                            uint16_t* __restrict__ residual) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int f0 = (blockIdx.x * 4 + wave) * 16, m0 = blockIdx.y * 16;
  if (f0 >= N) return;
  const int row = m0 + r;
  const size_t idx = (size_t)min(row, M - 1) * N + f0 + 4 * g;
  const int mine = row < M ? lora_of_row(a, row) : -1;
  f32x4_t d = {0.f, 0.f, 0.f, 0.f};
  lora_up_tile(a, h, M, N, m0, f0, mine, d);
  const size_t plane = (size_t)M * N;
  f32x4_t o = *reinterpret_cast<const f32x4_t*>(part + idx);
  for (int i = 1; i < slices; ++i) o += *reinterpret_cast<const f32x4_t*>(part + i * plane + idx);
  if (row >= M) return;
  ushort4 bv = make_ushort4(0, 0, 0, 0), rv = bv, out;
  if (b) bv = *reinterpret_cast<const ushort4*>(b + f0 + 4 * g);
  if (residual) rv = *reinterpret_cast<const ushort4*>(residual + idx);
  const uint16_t bb[4] = {bv.x, bv.y, bv.z, bv.w}, rr[4] = {rv.x, rv.y, rv.z, rv.w};
  uint16_t oo[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float v = mine >= 0 ? o[i] + d[i] : o[i];
    const float q = bf16_round(v + (b ? bf2f(bb[i]) : 0.f));
    oo[i] = residual ? f2bf(bf2f(rr[i]) + q) : f2bf(q);
  }
  out = make_ushort4(oo[0], oo[1], oo[2], oo[3]);
  *reinterpret_cast<ushort4*>((residual ? residual : y) + idx) = out;
}

static size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

static size_t partial_bytes(int M, int N, int K) { return (size_t)gemm_planes(M, K) * M * N * sizeof(float); }

int launch_linear_lora(const uint16_t* x, const uint16_t* W, const uint16_t* b, int M, int N, int K, const LoraArgs& a,
                       uint16_t* y, uint16_t* residual, char* ws, hipStream_t s) {
  float* part = reinterpret_cast<float*>(ws);
  uint16_t* h = reinterpret_cast<uint16_t*>(ws + align256(partial_bytes(M, N, K)));
  hipLaunchKernelGGL(lora_down_kernel, dim3(ceil_div(M, 16), a.n_seg * a.R / 16), dim3(64 * kDownWaves), 0, s, x, M, K, a, h);
  int rc = check_launch("lora_down");
  if (rc) return rc;
  int slices = 0;
  rc = launch_gemm(x, W, M, N, K, part, &slices, s);
  if (rc) return rc;
  hipLaunchKernelGGL(lora_finalize_kernel, dim3(ceil_div(N, 64), ceil_div(M, 16)), dim3(256), 0, s, part, slices, M, N, a, h,
                     b, y, residual);
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
  LoraArgs a{A, B, scale, ranks, adapter, row_seq, n, R, n_seg, n_seqs, {0, 0, 0}};
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
  return align256(partial_bytes(M, N, K)) + (size_t)M * n_segments * R * 4;
}

extern "C" int flyai_linear_lora_bf16(const uint16_t* x, const uint16_t* w, const uint16_t* b, int32_t M, int32_t N,
                                      int32_t K, const uint16_t* lora_a, const uint16_t* lora_b, const float* scale,
                                      const int32_t* ranks, int32_t n_adapters, int32_t R, const int32_t* segments_host,
                                      int32_t n_segments, const int32_t* adapter, const int32_t* row_seq, int32_t n_seqs,
                                      uint16_t* y, uint16_t* residual, void* workspace, flyai_stream_t stream) {
  FLYAI_REQUIRE(M >= 0 && M <= (1 << 20) && N > 0 && K > 0 && N % 16 == 0 && K % 32 == 0 && K <= 8192,
                "linear_lora: need M <= %d, N %% 16 == 0, K %% 32 == 0, K <= 8192", 1 << 20);
  if (M == 0) return FLYAI_OK;  // an empty tensor has no address
  FLYAI_REQUIRE(x && w && (y || residual) && workspace, "linear_lora: null pointer");
  FLYAI_REQUIRE(((uintptr_t)x | (uintptr_t)w | (uintptr_t)b | (uintptr_t)y | (uintptr_t)residual | (uintptr_t)workspace) % 16 == 0,
                "linear_lora: pointers must be 16-byte aligned");
  LoraArgs a;
  const int rc = make_lora_args(&a, lora_a, lora_b, scale, ranks, n_adapters, R, segments_host, n_segments, N, adapter, row_seq,
                                n_seqs);
  if (rc) return rc;
  return launch_linear_lora(x, w, b, M, N, K, a, y, residual, static_cast<char*>(workspace), as_stream(stream));
}
