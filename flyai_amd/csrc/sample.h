// What the samplers share: keys in value order, the exact integer weights, selections and scans of a workgroup.
#pragma once
#include <math.h>

#include "common.h"

namespace flyai {

constexpr int kSampThreads = 1024;
constexpr int kSampWaves = kSampThreads / 64;

// order-preserving key of a finite fp32 value: larger value <=> larger key (-0 keyed as +0)
__device__ __forceinline__ uint32_t f32_key(float z) {
  const uint32_t u = z == 0.f ? 0u : __float_as_uint(z);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ float key_f32(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// floor(2^40 * e^d) for d <= 0, by Cody-Waite range reduction (d = k ln2 + r, |r| <= ln2 / 2, ln2 split
// into a 32-bit head, so k * head is exact, and a tail) and the degree-13 Taylor polynomial of e^r
// (truncation error below 5e-18), each fp64 operation rounded on its own (no fused multiply-add):
// within one unit of the exact floor.  d below -27.75 gives 0 (2^40 e^d < 1 there).
__device__ __forceinline__ double samp_weight_f64(float z, float zmax) {  // (a double holds it: it is at most 2^40)
#pragma clang fp contract(off)
  const double d = (double)z - (double)zmax;
  if (!(d >= -27.75)) return 0.0;
  const double k = rint(d * 0x1.71547652b82fep+0);
  const double r = (d - k * 0x1.62e42feep-1) - k * 0x1.a39ef35793c76p-33;
  double p = 0x1.6124613a86d09p-33;
  p = p * r + 0x1.1eed8eff8d898p-29;
  p = p * r + 0x1.ae64567f544e4p-26;
  p = p * r + 0x1.27e4fb7789f5cp-22;
  p = p * r + 0x1.71de3a556c734p-19;
  p = p * r + 0x1.a01a01a01a01ap-16;
  p = p * r + 0x1.a01a01a01a01ap-13;
  p = p * r + 0x1.6c16c16c16c17p-10;
  p = p * r + 0x1.1111111111111p-7;
  p = p * r + 0x1.5555555555555p-5;
  p = p * r + 0x1.5555555555555p-3;
  p = p * r + 0x1p-1;
  p = p * r + 1.0;
  p = p * r + 1.0;
  return floor(ldexp(p, (int)k + 40));
}

__device__ __forceinline__ uint64_t samp_weight(float z, float zmax) { return (uint64_t)samp_weight_f64(z, zmax); }

// block sums over the 1024 threads through LDS (one slot per wave)
template <class T>
__device__ __forceinline__ T block_sum(T v, T* red) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();
  if (lane == 0) red[wave] = v;
  __syncthreads();
  T s = 0;
#pragma unroll
  for (int w = 0; w < kSampWaves; ++w) s += red[w];
  return s;
}

__device__ __forceinline__ uint32_t block_max_u32(uint32_t v, uint32_t* red) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();
  if (lane == 0) red[wave] = v;
  __syncthreads();
  uint32_t m = 0;
#pragma unroll
  for (int w = 0; w < kSampWaves; ++w) m = max(m, red[w]);
  return m;
}

struct SampShared {
  uint64_t hist[256];
  uint64_t red64[kSampWaves];
  uint32_t red32[kSampWaves];
  uint64_t scan[kSampThreads];
  uint64_t sel_above;  // weight (or count) above the selected bin
  uint32_t sel_prefix;
  int sel_found;
};

// Radix selection over the 32-bit keys of the kept tokens, 8 bits per pass from the top: the key of
// the token where the running total of `mass` (counts for top-k, weights for top-p), taken in
// descending key order, first exceeds `limit`.  Returns the key; *above gets the total mass of the
// kept tokens with larger keys.  If the total never exceeds limit, returns 0 with *above = total.
template <class KeyOf, class MassOf>
__device__ uint32_t radix_select(int V, KeyOf key_of, MassOf mass_of, uint64_t limit, uint64_t* above, SampShared& sh) {
  uint32_t prefix = 0;
  uint64_t run = 0;  // mass of tokens above the current prefix's range
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int b = threadIdx.x; b < 256; b += kSampThreads) sh.hist[b] = 0;
    __syncthreads();
    const uint32_t hi_mask = shift == 24 ? 0u : (0xffffffffu << (shift + 8));
    for (int v = threadIdx.x; v < V; v += kSampThreads) {
      uint32_t k;
      uint64_t m;
      if (!key_of(v, &k)) continue;
      if ((k & hi_mask) != (prefix & hi_mask)) continue;
      m = mass_of(v);
      if (m) atomicAdd((unsigned long long*)&sh.hist[(k >> shift) & 0xff], (unsigned long long)m);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int found = -1;
      uint64_t r = run;
      for (int b = 255; b >= 0; --b) {
        if (r + sh.hist[b] > limit) {
          found = b;
          break;
        }
        r += sh.hist[b];
      }
      sh.sel_found = found;
      sh.sel_above = r;
      sh.sel_prefix = found >= 0 ? (prefix | ((uint32_t)found << shift)) : 0u;
    }
    __syncthreads();
    if (sh.sel_found < 0) {
      *above = sh.sel_above;
      return 0u;
    }
    prefix = sh.sel_prefix;
    run = sh.sel_above;
  }
  *above = run;
  return prefix;
}

// ---- a row in chunks of consecutive ids ----
constexpr int kChunkThreads = 256;
constexpr int kMaxChunks = 64;
constexpr int kChunkStep = kChunkThreads * 8;  // ids of one iteration of a chunk's loop
constexpr int kMinChunk = 2 * kChunkStep;      // two iterations: less, and the launch outweighs the loads

// the 16 bits of a bf16 in value order (-0 as +0), and back
__device__ __forceinline__ uint32_t bf_key(uint16_t b) {
  return (b & 0x8000u) ? (b == 0x8000u ? 0x8000u : (~(uint32_t)b & 0xffffu)) : (b | 0x8000u);
}
__device__ __forceinline__ float key_bf(uint32_t k) {
  return bf2f((uint16_t)((k & 0x8000u) ? (k & 0x7fffu) : (~k & 0xffffu)));
}
__device__ __forceinline__ uint64_t key_weight(uint32_t k, float tdiv, float zmax) {
  return samp_weight(__fdiv_rn(key_bf(k), tdiv), zmax);
}

template <class T>
__device__ __forceinline__ T wave_incl_scan(T v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T y = __shfl_up(v, o, 64);
    if (lane >= o) v += y;
  }
  return v;
}

// exclusive prefix over the workgroup's NT threads; *total gets the sum
template <int NT, class T>
__device__ __forceinline__ T block_excl_scan(T v, T* red, T* total) {
  const T incl = wave_incl_scan(v);
  const int wave = threadIdx.x >> 6;
  __syncthreads();  // the last use of red is over
  if ((threadIdx.x & 63) == 63) red[wave] = incl;
  __syncthreads();
  T base = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    base += w < wave ? red[w] : (T)0;
    sum += red[w];
  }
  *total = sum;
  return base + incl - v;
}

// f(id, bits) for the thread's ids of [c0, c1), in steps of 8 consecutive ids a thread
template <class F>
__device__ __forceinline__ void for_chunk(const uint16_t* __restrict__ x, int c0, int c1, int vec, F&& f) {
  for (int b = c0 + (int)threadIdx.x * 8; b < c1; b += kChunkStep) {
    if (vec && b + 8 <= c1) {
      const uint4 q = *reinterpret_cast<const uint4*>(x + b);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) f(b + j, (uint16_t)((j & 1) ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu));
    } else {
      const int n = min(8, c1 - b);
      for (int j = 0; j < n; ++j) f(b + j, x[b + j]);
    }
  }
}

}  // namespace flyai
