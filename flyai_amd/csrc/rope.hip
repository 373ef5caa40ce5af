// Rotary positions on rows of any head count and head size: half and interleaved layouts, part of the head,
// scaled frequencies, and the inverse rotation (which is the gradient).
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace flyai {

// angle(t, i) = positions[t] * inv_freq[i]; the pair (u, v) of index i becomes
//   (s (u cos - v sin), s (v cos + u sin)),  sin negated for the inverse,
// with u, v = x[i], x[i + rot/2] (half) or x[2i], x[2i + 1] (interleaved).  Dims from rot on are copied.
//
// The angle is a 64-bit product (32 bits are 0.06 rad off at position 10^6), reduced to [-pi/4, pi/4] there, and only
// then rounded to 32 bits.  Near position 2^31 the product's own rounding is up to 2^-23 (two steps of an fp32 cosine), so
// what it left out is added to the reduced angle.  That angle's rounding is at most 2^-25, the sums below add as much again
// and the Taylor terms left out 2e-9: cos and sin are off by less than 3 * 2^-25 at any int32 position (1.8 * 2^-25 at most over
// 1,536 pairs of the farthest positions and frequencies of 0.5 to 1; 4.4 without the product's rest).  Products and sums are
// fp32, rounded once to the output's type.
__device__ __forceinline__ void sincos_reduced(int position, double frequency, float& s, float& c) {
  const double kTwoOverPi = 0.63661977236758134308, kPio2Hi = 1.57079632679489655800, kPio2Lo = 6.12323399573676603587e-17;
  const double angle = position * frequency, left = fma((double)position, frequency, -angle);
  const double q = rint(angle * kTwoOverPi);
  // q * kPio2Hi leaves the fma unrounded until the difference is taken; kPio2Lo is pi/2 minus kPio2Hi
  const float r = (float)(fma(-q, kPio2Lo, fma(-q, kPio2Hi, angle)) + left);
  const float z = r * r;
  // sin r = r - r^3/3! + r^5/5! - r^7/7! + r^9/9!,  cos r = 1 - r^2/2! + ... - r^10/10!
  const float sp = fmaf(r * z, fmaf(z, fmaf(z, fmaf(z, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), r);
  const float cp = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
  // the quadrant: q mod 4 (|q| < 2^53 is an exact integer; only its two low bits matter)
  const int quad = (int)((long long)q & 3);
  s = (quad & 1) ? cp : sp;
  c = (quad & 1) ? sp : cp;
  s = (quad & 2) ? -s : s;
  c = (quad == 1 || quad == 2) ? -c : c;
}

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(uint16_t v) { return bf2f(v); }
template <> __device__ __forceinline__ float to_f(_Float16 v) { return (float)v; }
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ uint16_t from_f(float v) { return f2bf(v); }
template <> __device__ __forceinline__ _Float16 from_f(float v) { return (_Float16)v; }
template <> __device__ __forceinline__ float from_f(float v) { return v; }

struct RopeArgs {
  const void* x;
  void* out;
  const int32_t* positions;
  const double* inv_freq;
  int64_t x_token, x_head, o_token, o_head;  // strides in elements; the last dim is contiguous
  float scaling;
  int T, H, D, rot, inverse;
  int upr, uph;       // units of a head that rotate, units of a head
  int tokens, units;  // per workgroup: tokens, and units of each of them
};

constexpr int kRopeThreads = 256;
constexpr int kRopePairs = 1024;  // (cos, sin) pairs a workgroup keeps in LDS: 8 KiB

// A workgroup takes `tokens` tokens and, of each, `units` of its H * uph units (blockIdx.y picks which): it computes the
// tokens' cos and sin once into LDS, then every thread moves units.  A unit is V elements and their partners (half
// layout), V / 2 pairs (interleaved) or V elements to copy, V * sizeof(T) = 16 or 8 bytes where sizes, strides and
// addresses allow, one element (one pair) otherwise.  A unit is read whole before it is written, by the same thread,
// so x and out may be the same tensor.
// What bounds it is the bytes: 8,192 tokens of 64 heads of 128 in fp32, 537 MB, take 96 us (5.6 TB/s), 3,001 of 32 heads of 192
// in fp16, a third of each turned, 74 MB, 13.4 us (5.5 TB/s); 24 tokens of 72 heads of 64, 2.9 us, are a launch and two round
// trips.
template <typename T, int V, bool HALF>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeArgs a) {
  __shared__ float2 cs[kRopePairs];
  typedef T vec_t __attribute__((ext_vector_type(V)));
  constexpr int N = HALF ? V : (V > 1 ? V : 2);  // elements of a rotating unit's first (half) or only load
  const int P = a.rot / 2;
  const int t0 = blockIdx.x * a.tokens, nt = min(a.tokens, a.T - t0);
  for (int i = threadIdx.x; i < nt * P; i += kRopeThreads) {
    float s, c;
    sincos_reduced(a.positions[t0 + i / P], a.inv_freq[i % P], s, c);
    cs[i] = make_float2(c * a.scaling, (a.inverse ? -s : s) * a.scaling);
  }
  __syncthreads();
  const int per = a.H * a.uph, u0 = blockIdx.y * a.units, nu = min(a.units, per - u0);
  const T* x = static_cast<const T*>(a.x);
  T* out = static_cast<T*>(a.out);
  auto load = [](const T* p, T (&v)[N], auto count) __attribute__((always_inline)) {
    if constexpr (V > 1) {
      const vec_t w = *reinterpret_cast<const vec_t*>(p);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = w[i];
    } else {
#pragma unroll
      for (int i = 0; i < decltype(count)::value; ++i) v[i] = p[i];
    }
  };
  auto store = [](T* p, const T (&v)[N], auto count) __attribute__((always_inline)) {
    if constexpr (V > 1) {
      vec_t w;
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = v[i];
      *reinterpret_cast<vec_t*>(p) = w;
    } else {
#pragma unroll
      for (int i = 0; i < decltype(count)::value; ++i) p[i] = v[i];
    }
  };
  using One = std::integral_constant<int, 1>;
  using All = std::integral_constant<int, N>;
  for (int i = threadIdx.x; i < nt * nu; i += kRopeThreads) {
    const int tl = i / nu, u = u0 + i % nu;
    const int h = u / a.uph, c = u % a.uph;
    const int64_t xr = (int64_t)(t0 + tl) * a.x_token + (int64_t)h * a.x_head;
    const int64_t orow = (int64_t)(t0 + tl) * a.o_token + (int64_t)h * a.o_head;
    const float2* tab = cs + tl * P;
    if (c >= a.upr) {
      const int d = a.rot + (c - a.upr) * V;
      T v[N];
      load(x + xr + d, v, One{});
      store(out + orow + d, v, One{});
    } else if constexpr (HALF) {
      const int d = c * V;
      T u1[N], v1[N];
      load(x + xr + d, u1, All{});
      load(x + xr + d + P, v1, All{});
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float2 w = tab[d + j];
        const float uf = to_f(u1[j]), vf = to_f(v1[j]);
        u1[j] = from_f<T>(fmaf(uf, w.x, -(vf * w.y)));
        v1[j] = from_f<T>(fmaf(vf, w.x, uf * w.y));
      }
      store(out + orow + d, u1, All{});
      store(out + orow + d + P, v1, All{});
    } else {
      const int d = c * N;
      T v[N];
      load(x + xr + d, v, All{});
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        const float2 w = tab[(d + j) / 2];
        const float uf = to_f(v[j]), vf = to_f(v[j + 1]);
        v[j] = from_f<T>(fmaf(uf, w.x, -(vf * w.y)));
        v[j + 1] = from_f<T>(fmaf(vf, w.x, uf * w.y));
      }
      store(out + orow + d, v, All{});
    }
  }
}

template <typename T>
static void rope_go(RopeArgs& a, bool half, int bytes, hipStream_t s) {
  constexpr int E = (int)sizeof(T);
  const int V = bytes > E ? bytes / E : 1;
  const int pair = half ? V : (V > 1 ? V : 2);  // of a unit: rotating elements (half: of its first half)
  a.upr = (half ? a.rot / 2 : a.rot) / pair;
  a.uph = a.upr + (a.D - a.rot) / V;
  const int per = a.H * a.uph;
  // Units of a workgroup: four a thread, one while that leaves most of the chip without a workgroup.  One / four a thread, 72
  // heads of 64 bf16: 24 tokens 2.9 / 4.1 us, 300 tokens 3.6 / 4.5, 1,000 tokens 5.1 / 6.3; 3,001 tokens of 32 heads of 192 fp16
  // 14.7 / 13.3; 8,192 of 64 heads of 128 fp32 100 / 96.
  const int64_t total = (int64_t)a.T * per;
  const int want = total >= (int64_t)4 * kRopeThreads * 2 * device_cus() ? 4 * kRopeThreads : kRopeThreads;
  const int most = a.rot > 0 ? kRopePairs / (a.rot / 2) : want;
  a.tokens = std::max(1, std::min(want / per, most));
  a.units = std::min(per, want);
  const dim3 grid(ceil_div(a.T, a.tokens), ceil_div(per, a.units));
  auto run = [&](auto v, auto h) {
    hipLaunchKernelGGL((rope_kernel<T, decltype(v)::value, decltype(h)::value>), grid, dim3(kRopeThreads), 0, s, a);
  };
  using Half = std::true_type;
  using Inter = std::false_type;
  using V16 = std::integral_constant<int, 16 / E>;
  using V8 = std::integral_constant<int, 8 / E>;
  using V1 = std::integral_constant<int, 1>;
  if (bytes == 16) half ? run(V16{}, Half{}) : run(V16{}, Inter{});
  else if (bytes == 8) half ? run(V8{}, Half{}) : run(V8{}, Inter{});
  else half ? run(V1{}, Half{}) : run(V1{}, Inter{});
}

}  // namespace flyai

using namespace flyai;

extern "C" int flyai_rope(const void* x, int64_t x_token, int64_t x_head, const int32_t* positions,
                          const double* inv_freq, float scaling, int32_t T, int32_t H, int32_t D, int32_t rot,
                          int32_t dtype, int32_t interleaved, int32_t inverse, void* out, int64_t o_token,
                          int64_t o_head, flyai_stream_t stream) {
  FLYAI_REQUIRE(T >= 0 && H > 0 && D > 0, "rope: bad shape");
  FLYAI_REQUIRE(rot > 0 && rot % 2 == 0 && rot <= D && rot <= 2 * kRopePairs,
                "rope: the rotated part must be even, in [2, min(D, %d)]", 2 * kRopePairs);
  FLYAI_REQUIRE(T <= (1 << 22) && (int64_t)H * D <= (1 << 22), "rope: T and H * D at most %d", 1 << 22);
  FLYAI_REQUIRE(dtype >= FLYAI_BF16 && dtype <= FLYAI_F32, "rope: unknown dtype %d", dtype);
  FLYAI_REQUIRE(x_token >= 0 && x_head >= 0 && o_token >= 0 && o_head >= 0, "rope: negative stride");
  if (T == 0) return FLYAI_OK;
  FLYAI_REQUIRE(x && out && positions && inv_freq, "rope: null pointer");
  // two output rows that share elements would race
  const bool heads_inner = H == 1 || T == 1 || o_token >= o_head;
  const int64_t inner = heads_inner ? o_head : o_token, outer = heads_inner ? o_token : o_head;
  const int64_t n_in = heads_inner ? H : T, n_out = heads_inner ? T : H;
  FLYAI_REQUIRE((n_in == 1 || inner >= D) && (n_out == 1 || outer >= (n_in - 1) * inner + D),
                "rope: output rows overlap");
  // x is read and out written row by row, in no order: they are the same rows or lie apart
  const int64_t E = dtype == FLYAI_F32 ? 4 : 2;
  const char *xb = static_cast<const char*>(x), *ob = static_cast<const char*>(out);
  const char* xe = xb + ((T - 1) * x_token + (H - 1) * x_head + D) * E;
  const char* oe = ob + ((T - 1) * o_token + (H - 1) * o_head + D) * E;
  FLYAI_REQUIRE(xe <= ob || oe <= xb || (x == out && (T == 1 || x_token == o_token) && (H == 1 || x_head == o_head)),
                "rope: out overlaps x and is not x");
  RopeArgs a{x, out, positions, inv_freq, x_token, x_head, o_token, o_head, scaling, T, H, D, rot, inverse != 0, 0, 0, 0, 0};
  // The widest load that every row start, the partner's distance and the copied part allow: 16 bytes, 8 or one element took
  // 13.3, 17.5 and 38.5 us for 3,001 tokens of 32 heads of 192 fp16, 5.2, 5.9 and 9.1 for 1,000 of 72 heads of 64 bf16.
  auto fits = [&](int bytes) {
    const int64_t v = bytes / E, rotated = interleaved ? rot : rot / 2;
    return ((uintptr_t)x | (uintptr_t)out) % bytes == 0 && rotated % v == 0 && (D - rot) % v == 0 &&
           (T == 1 || (x_token % v == 0 && o_token % v == 0)) && (H == 1 || (x_head % v == 0 && o_head % v == 0)) &&
           (D == rot || rot % v == 0);
  };
  const int bytes = fits(16) ? 16 : fits(8) ? 8 : (int)E;
  hipStream_t s = as_stream(stream);
  if (dtype == FLYAI_BF16) rope_go<uint16_t>(a, !interleaved, bytes, s);
  else if (dtype == FLYAI_F16) rope_go<_Float16>(a, !interleaved, bytes, s);
  else rope_go<float>(a, !interleaved, bytes, s);
  return check_launch("rope");
}
