// What the attention kernels share: a 64-key block's fragments, its masks, the running maximum's rule.
#pragma once
#include "common.h"

namespace flyai {

constexpr float kLog2e = 1.4426950408889634f;

// A running max m (base-2 units) moves only when a block's max exceeds it by more than kMaxSlack.
constexpr float kMaxSlack = 8.f;
constexpr float kMaxSentinel = -1e29f;  // a running max at or below this is the initial -1e30 (no key yet)

__device__ __forceinline__ uint4 mask_keys(uint4 v, int key0, int lo, int hi) {
  // zero the bf16 elements whose key (key0 + element index) lies outside [lo, hi)
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int key = key0 + i;
    if (key < lo || key >= hi) w[i >> 1] &= (i & 1) ? 0x0000ffffu : 0xffff0000u;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ int tile_key(int kt, int m) {
  return 32 * (kt >> 1) + 8 * (m >> 2) + 4 * (kt & 1) + (m & 3);
}

// Every 64-key block starts at a multiple of 64 below key_hi <= cap (cap % 64 == 0), so all 64 keys
// are inside the slab: the loads below are unconditional (no branch between loads).  The slab is
// tiled (kv_k_off / kv_v_off in common.h): a 64-key block is 4096 contiguous elements, and each of
// these 16-byte-per-lane loads reads one contiguous KiB of it.
// KV is read once per step, so the loads are nontemporal (streamed, as the expert weights are).
typedef unsigned int attn_u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint4 ld_kv(const uint16_t* p) {
  const attn_u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const attn_u32x4*>(p));
  return make_uint4(v.x, v.y, v.z, v.w);
}

__device__ __forceinline__ void load_k_tile(uint4 (&k)[4][2], const uint16_t* __restrict__ K, int kb,
                                            int lane) {
  const uint16_t* blk = K + (size_t)kb * 64 + lane * 8;
#pragma unroll
  for (int kt = 0; kt < 4; ++kt) {
    k[kt][0] = ld_kv(blk + kt * 1024);
    k[kt][1] = ld_kv(blk + kt * 1024 + 512);
  }
}

__device__ __forceinline__ void load_v_tile(uint4 (&v)[4][2], const uint16_t* __restrict__ Vt, int kb,
                                            int lane) {
  const uint16_t* blk = Vt + (size_t)kb * 64 + lane * 8;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) v[dt][h] = ld_kv(blk + h * 2048 + dt * 512);
}

// Max over the four lanes n, n+16, n+32, n+48 (one query row's lane groups), with gfx950's
// v_permlane32_swap / v_permlane16_swap (VALU lane swaps, no LDS round trip).  Swapping a register
// with a copy of itself leaves lane i's value and its partner's in the two results.  (A compare and
// select: fmaxf on the swapped values is three instructions, since the compiler quiets possible
// signalling NaNs in both operands first.)
__device__ __forceinline__ float max_lane_groups(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const float x0 = __uint_as_float(a[0]), x1 = __uint_as_float(a[1]);
  v = x0 > x1 ? x0 : x1;
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const float y0 = __uint_as_float(b[0]), y1 = __uint_as_float(b[1]);
  return y0 > y1 ? y0 : y1;
}

}  // namespace flyai
