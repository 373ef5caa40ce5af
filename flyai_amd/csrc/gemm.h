// The split-K projection kernel, for the plain projection (linear.hip) and the one with adapters (lora.hip).
#pragma once
#include <type_traits>

#include "common.h"
#include "lora.h"

namespace flyai {

// gemm_splitk: workgroup = 4 or 8 waves on as many consecutive 16-feature tiles and one K slice of kKQW groups
// of 128.  MFMA step j of group q takes, in lane (r, g), K = 128q + 32j + 8g .. +7 for both operands
// (any K order shared by the two operands is valid), so each weight load instruction reads one
// whole 64-byte run of each of its 16 rows.  The activation slice (64 rows x 512 K, bf16) is staged once in LDS; each wave issues all
// of its weight loads for the slice before its first MFMA (a single HBM round trip per wave) and
// writes fp32 partial sums part[slice][row][feature].  A finalize kernel adds the slices in slice
// order (so the result is independent of timing), the bias, and the fused epilogue.
typedef float f32x4_dw __attribute__((ext_vector_type(4), aligned(4)));  // partials are 4-byte aligned,
typedef uint16_t u16x4_h __attribute__((ext_vector_type(4), aligned(2)));  // bf16 tensors 2-byte
constexpr int kKQW = 4;       // K groups of 128 per slice
constexpr int kGemmRows = 64; // activation rows per pass
constexpr int kTiledMinRows = 256;  // batches of at least this many rows take the tiled kernel

// More rows than a pass: the weights stay in registers over the passes of 64 rows, and the next pass's activations
// are loaded into registers under the current pass's MFMAs (one barrier pair a pass, on LDS only: the loads stay in
// flight).  A pass used to be staged behind a barrier that drained every load, by workgroups of 64 features: the
// two projections of 5,120 x 2,880 and 2,880 x 4,096 took 19.2 and 18.5 us at 137 rows, now 16.3 and 15.6; 24.9 and
// 24.3 at 255, now 22.5 and 22.2.  Eight waves and 128 features read the activations half as often from L2, where
// that grid still gives most CUs a workgroup (launch_gemm_splitk); wider waves (two feature tiles each) made no
// difference.  What is left past the weights' 5 us is the partial planes' way out, about 4 us per 64 rows.
// No load sits under a lane's branch: rows past M and features past N read a clamped one (their sums are not
// stored), K past the row's end is replaced by zero in both operands.  With the loads predicated the weights' waited
// for the activations' to return: 7.7 us for 1 row of either projection, 8.1 for 16; now 7.2 and 7.5.  The weights'
// are under no branch at all (a slice of fewer groups reads its last steps again): with one per group of 128 the
// compiler could not count them, and the LDS stores waited for all but three of them: kernel and finalize at 64 rows
// 14.4 us for 5,120 x 2,880, now 14.0, 14.0 for 2,880 x 4,096, now 13.6.
// LORA: the adapters' down product is in the launch, in its first `wgs` workgroups, beside the stream of the weights; the
// grid has one axis then.
template <int WAVES, bool LORA>
__global__ __launch_bounds__(64 * WAVES, LORA ? 2 : 1) void gemm_splitk_bf16_kernel(
    const uint16_t* __restrict__ x, const uint16_t* __restrict__ W, int M, int N, int K,
    float* __restrict__ part, LoraArgs lo, int wgs, int bxs) {
  typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
  __shared__ u32x4 as[kGemmRows][kKQW * 16 + 1];  // 64 rows x 512 bf16, +16 B per row vs bank conflicts
  if constexpr (LORA) {
    constexpr int kTiles = kTiledMinRows / kDownRows;
    typedef LoraDownLds<WAVES, kTiles, kTiles> down_lds;
    static_assert(sizeof(as) >= sizeof(down_lds), "the down product's LDS");
    if ((int)blockIdx.x < wgs) {
      lora_down<WAVES, kTiles, kTiles>(x, M, K, lo, blockIdx.x, wgs, *reinterpret_cast<down_lds*>(as));
      return;
    }
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int nt = (LORA ? ((int)blockIdx.x - wgs) % bxs : (int)blockIdx.x) * WAVES + wave;
  const int slice = LORA ? ((int)blockIdx.x - wgs) / bxs : (int)blockIdx.y;
  const int KQ = (K + 127) / 128;
  const int kq0 = slice * kKQW;
  const int nkq = min(kKQW, KQ - kq0);
  const int feat = nt * 16 + r;
  // a wave loads whole rows of the slice (64 lanes x 16 bytes): row WAVES j + wave of the pass in load j
  constexpr int kPer = kGemmRows / WAVES, kPerTile = 16 / WAVES;
  static_assert(kKQW * 16 == 64, "one row of a slice is one wave load");
  const int k = 128 * kq0 + 8 * lane;
  const bool kval = k < K;
  const uint16_t* xk = x + min(k, K - 8);
  u32x4 av[kPer];
  auto load_rows = [&](int m0) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < kGemmRows / 16; ++t)
      if (m0 + 16 * t < M) {
#pragma unroll
        for (int j = t * kPerTile; j < (t + 1) * kPerTile; ++j)
          av[j] = *reinterpret_cast<const u32x4*>(xk + (size_t)min(m0 + WAVES * j + wave, M - 1) * K);
      }
  };
  auto store_rows = [&](int m0) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < kGemmRows / 16; ++t)
      if (m0 + 16 * t < M) {
#pragma unroll
        for (int j = t * kPerTile; j < (t + 1) * kPerTile; ++j)
          as[WAVES * j + wave][lane] = kval ? av[j] : u32x4{0u, 0u, 0u, 0u};
      }
  };
  // The activation slice's loads go out first, then the weights, so the LDS stores wait only for the activations
  // (loads complete in issue order) and the L2 round trip for them overlaps the HBM fetch of the weights.
  load_rows(0);
  const uint16_t* wrow = W + (size_t)min(feat, N - 1) * K + 8 * g;
  u32x4 wv[kKQW][4];
#pragma unroll
  for (int q = 0; q < kKQW; ++q)
#pragma unroll
    for (int j = 0; j < 4; ++j)  // step j reads K kb + 32j .. +31 (K % 32 == 0)
      wv[q][j] = *reinterpret_cast<const u32x4*>(wrow + min(128 * (kq0 + q) + 32 * j, K - 32));
  float* pp = part + (size_t)slice * M * N;
  for (int m0 = 0; m0 < M; m0 += kGemmRows) {
    if (m0) lds_barrier();  // every wave has read the previous pass's rows
    store_rows(m0);
    if (m0 + kGemmRows < M) load_rows(m0 + kGemmRows);
    lds_barrier();
    // the row tiles of the pass as a constant: without branches between them their MFMA chains interleave
    const auto pass = [&](auto tiles) __attribute__((always_inline)) {
      constexpr int MT = decltype(tiles)::value;
      f32x4_t acc[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < kKQW; ++q) {
        if (q >= nkq) break;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x4 w = 128 * (kq0 + q) + 32 * j < K ? wv[q][j] : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
          for (int m = 0; m < MT; ++m)
            acc[m] = mfma16x16x32(__builtin_bit_cast(bf16x8_t, w),
                                  __builtin_bit_cast(bf16x8_t, as[16 * m + r][q * 16 + 4 * j + g]), acc[m]);
        }
      }
      // weights as the first operand: lane (r, g) holds features 4g .. +3 of row 16m + r, one 16-byte store
      if (nt * 16 >= N) return;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int row = m0 + 16 * m + r;
        if (row >= M) continue;
        auto* o = reinterpret_cast<f32x4_dw*>(pp + (size_t)row * N + nt * 16 + 4 * g);
        if (WAVES == 8) __builtin_nontemporal_store(acc[m], o);  // planes beyond L2: 137 rows 18.3 -> 16.6 us
        else *o = acc[m];
      }
    };
    const int mt_count = (min(kGemmRows, M - m0) + 15) / 16;
    if (mt_count == 4) pass(std::integral_constant<int, 4>{});
    else if (mt_count == 3) pass(std::integral_constant<int, 3>{});
    else if (mt_count == 2) pass(std::integral_constant<int, 2>{});
    else pass(std::integral_constant<int, 1>{});
  }
}

int gemm_slices(int K);

}  // namespace flyai
