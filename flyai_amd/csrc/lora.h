// The low-rank adapters' arguments and their up product, for the kernels that add it to a projection.
#pragma once
#include "common.h"

namespace flyai {

struct LoraArgs {
  const uint16_t* A;       // [n][n_seg * R][K]
  const uint16_t* B;       // [n][N][R]
  const float* scale;      // [n]
  const int32_t* ranks;    // [n]
  const int32_t* adapter;  // of a row, or of a row's sequence
  const int32_t* row_seq;  // null: adapter is per row
  int n, R, n_seg, n_seqs;
  int seg_end[3];  // first feature past segments 0, 1, 2
};

// The adapter of row t, -1 for none (an id or a sequence out of range is none).
__device__ __forceinline__ int lora_of_row(const LoraArgs& a, int t) {
  int i = t;
  if (a.row_seq) {
    i = a.row_seq[t];
    if ((unsigned)i >= (unsigned)a.n_seqs) return -1;
  }
  const int ad = a.adapter[i];
  return (unsigned)ad < (unsigned)a.n ? ad : -1;
}

__device__ __forceinline__ int lora_rank(const LoraArgs& a, int ad) { return min(max(a.ranks[ad], 0), a.R); }

// The segment of feature f (wave-uniform when f is).
__device__ __forceinline__ int lora_segment(const LoraArgs& a, int f) {
  int seg = 0;
#pragma unroll
  for (int i = 0; i < 3; ++i) seg += i + 1 < a.n_seg && f >= a.seg_end[i];
  return seg;
}

// d += h B^T on a tile of 16 rows from m0 and 16 features from f0 (one segment, a multiple of 16): lane (r, g) gets
// features f0 + 4g .. +3 of row m0 + r, whose adapter is `mine` (-1: none).  One product per adapter among the rows, from
// zero over its rank's chunks in order, kept by its own rows alone: what another row's adapter holds, an infinity or a
// NaN among it, never reaches this one, and the sum does not depend on the tile.
__device__ __forceinline__ void lora_up_tile(const LoraArgs& a, const uint16_t* __restrict__ h, int M, int N, int m0, int f0,
                                             int mine, f32x4_t& d) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int chunks = a.R / 16, seg = lora_segment(a, f0);
  const uint16_t* hr = h + ((size_t)min(m0 + r, M - 1) * a.n_seg + seg) * chunks * 32 + 8 * g;
  uint64_t todo = __ballot(mine >= 0) & 0xffff;
  for (; todo;) {
    const int ad = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
    todo &= ~__ballot(mine == ad);
    const int rank = lora_rank(a, ad);
    const uint16_t* br = a.B + ((size_t)ad * N + f0 + r) * a.R + 8 * (g & 1);
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    for (int c = 0; 16 * c < rank; ++c) {
      uint4 bw = *reinterpret_cast<const uint4*>(br + 16 * c);
      const int left = rank - 16 * c - 8 * (g & 1);  // columns of this lane's eight within the rank
      if (left < 8) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&bw);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = 2 * i + 1 < left ? w[i] : 2 * i < left ? w[i] & 0xffffu : 0u;
      }
      acc = mfma16x16x32(as_bf16x8(bw), as_bf16x8(*reinterpret_cast<const uint4*>(hr + 32 * c)), acc);
    }
    if (mine == ad) d = acc;
  }
}

}  // namespace flyai
