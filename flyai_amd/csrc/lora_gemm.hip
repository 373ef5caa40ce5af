// The projection with adapters for large batches: 192 rows x 128 features a workgroup.
#include "common.h"
#include "gemm.h"

namespace flyai {

typedef uint16_t u16x4_t __attribute__((ext_vector_type(4)));

// gemm_tiled_lds_kernel's arithmetic (linear.hip) with 48 rows x 64 features a wave: 7 KiB of operands from LDS for 12 MFMAs where
// waves of 32 x 64 read 6 for 8, which is what bounds those (835 clocks a 64-K group of 128 x 128, 512 of them MFMA).  The
// same MFMAs in the same K order, each 512-K slice from zero and the slices added in order, so a row's bits do not depend
// on which of the two kernels a batch takes.  W is the first operand: a lane then holds four features of a row, which go out
// (and a row's adapter is chosen) together.  The products of a group's first half are kept before its barrier; scheduled
// behind it, the reads' time was all waiting (2,096 rows 89 -> 82.6 us).  Operands go global -> LDS in whole 128-byte runs through three stages of one
// 64-K group each, a group's loads issued two groups ahead; a row's eight 16-byte chunks are swizzled by row.  Rows and
// features past M / N load clamped ones and are never stored.
constexpr int kTallM = 192, kTallN = 128, kTallTiles = 3;  // 4 x 2 waves of 3 row tiles
constexpr int kTallStages = 3, kTallLoads = 5;             // load instructions a wave and group: 24 for x, 16 for W
constexpr int kTallA = kTallM * 128, kTallB = kTallN * 128;  // bytes a stage

template <bool PLANE>
__global__ __launch_bounds__(512) void gemm_tall_lora_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ W,
                                                             const uint16_t* __restrict__ bias, int M, int N, int K,
                                                             float* __restrict__ out, uint16_t* __restrict__ y,
                                                             uint16_t* __restrict__ residual, LoraArgs lo) {
  typedef __attribute__((address_space(3))) void* lds_ptr;
  __shared__ __align__(1024) char sa0[kTallA], sa1[kTallA], sa2[kTallA];
  __shared__ __align__(1024) char sb0[kTallB], sb1[kTallB], sb2[kTallB];
  __shared__ __align__(1024) char held_b[kTallN * 128];  // one adapter's columns
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int gm = (M + kTallM - 1) / kTallM, tile = lora_tile(blockIdx.x, gm, (N + kTallN - 1) / kTallN);
  if (tile < 0) return;
  const int m0 = (tile % gm) * kTallM, n0 = (tile / gm) * kTallN;
  const int wm = wave >> 1, wn = wave & 1, mw = m0 + 48 * wm, nw = n0 + 64 * wn;  // the wave's 48 x 64 block
  const int KG = K / 64;
  // instruction u = 5 wave + i fills half a 16-row tile, 8 rows: u < 24 of x, the others of W
  const uint16_t* src[kTallLoads];
#pragma unroll
  for (int i = 0; i < kTallLoads; ++i) {
    const int u = kTallLoads * wave + i, ub = u < 24 ? u : u - 24;
    const int q = 8 * ub + (lane >> 3), chunk = (lane & 7) ^ ((q >> 1) & 7);
    src[i] = (u < 24 ? x + (size_t)min(m0 + q, M - 1) * K : W + (size_t)min(n0 + q, N - 1) * K) + 8 * chunk;
  }
  auto issue = [&](char* sa, char* sb, int q) __attribute__((always_inline)) {
    const size_t k = (size_t)min(q, KG - 1) * 64;
#pragma unroll
    for (int i = 0; i < kTallLoads; ++i) {
      const int u = kTallLoads * wave + i;
      char* to = u < 24 ? sa + 1024 * u : sb + 1024 * (u - 24);
      __builtin_amdgcn_global_load_lds((const void*)(src[i] + k), (lds_ptr)to, 16, 0, 0);
    }
  };
  // tot starts at -0: -0 + x is x, so the first fold copies the first slice's sums
  f32x4_t acc[kTallTiles][4], tot[kTallTiles][4];
#pragma unroll
  for (int a = 0; a < kTallTiles; ++a)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      acc[a][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      tot[a][b] = f32x4_t{-0.f, -0.f, -0.f, -0.f};
    }
  const int frag = r * 128 + ((g ^ ((r >> 1) & 7)) << 4);
  bf16x8_t a0[kTallTiles], a1[kTallTiles], b0[4], b1[4];
  auto read_ab = [&](bf16x8_t (&af)[kTallTiles], bf16x8_t (&bw)[4], const char* sa, const char* sb, int j) __attribute__((always_inline)) {
    const int fo = frag ^ (j << 6);
#pragma unroll
    for (int t = 0; t < kTallTiles; ++t) af[t] = as_bf16x8(*reinterpret_cast<const uint4*>(sa + (kTallTiles * wm + t) * 2048 + fo));
#pragma unroll
    for (int t = 0; t < 4; ++t) bw[t] = as_bf16x8(*reinterpret_cast<const uint4*>(sb + (4 * wn + t) * 2048 + fo));
  };
  auto mfma_step = [&](const bf16x8_t (&af)[kTallTiles], const bf16x8_t (&bw)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < kTallTiles; ++a)
#pragma unroll
      for (int b = 0; b < 4; ++b) acc[a][b] = mfma16x16x32(bw[b], af[a], acc[a][b]);
  };
  // group q from stage (ca, cb) (its step-0 operands already in a0 / b0); hands over to (na, nb), refills (ca, cb) with q + 3
  auto group = [&](char* ca, char* cb, const char* na, const char* nb, int q) __attribute__((always_inline)) {
    read_ab(a1, b1, ca, cb, 1);
    mfma_step(a0, b0);
    __builtin_amdgcn_sched_barrier(0);  // the products go out under the reads, not behind the barrier
    __builtin_amdgcn_s_waitcnt(waitcnt_vm((kTallStages - 2) * kTallLoads));  // this wave's part of the next stage landed
    lds_barrier();  // every wave's part of the next stage is in LDS; every wave is done reading this one
    read_ab(a0, b0, na, nb, 0);
    issue(ca, cb, q + kTallStages);
    mfma_step(a1, b1);
    __builtin_amdgcn_sched_barrier(0);
    if ((q & 7) == 7 || q == KG - 1) {  // the end of a 512-K slice
#pragma unroll
      for (int a = 0; a < kTallTiles; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          tot[a][b] += acc[a][b];
          acc[a][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
    }
  };
  // what the up products need is fetched under the GEMM, as in gemm_tiled_lds_kernel
  int2 held = lo.meta[min(m0 + kTallM / 2, M - 1)];
  const int2 who = lo.meta[min(mw + lane, M - 1)];
  u16x4_h bv[4];  // N % 16 == 0
  if constexpr (!PLANE) {
#pragma unroll
    for (int b = 0; b < 4; ++b) bv[b] = *reinterpret_cast<const u16x4_h*>(bias ? bias + min(nw + 16 * b, N - 16) + 4 * g : lo.B);
  }
  // the stage waits count loads per group in issue order: no load may move across a group
  asm volatile("" ::: "memory");
  issue(sa0, sb0, 0);
  asm volatile("" ::: "memory");
  issue(sa1, sb1, 1);
  asm volatile("" ::: "memory");
  issue(sa2, sb2, 2);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(waitcnt_vm((kTallStages - 1) * kTallLoads));
  lds_barrier();  // stage 0 is in LDS
  held.x = __builtin_amdgcn_readfirstlane(held.y) > 0 ? __builtin_amdgcn_readfirstlane(held.x) : -1;
  if (held.x >= 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      __builtin_amdgcn_global_load_lds((const void*)(lo.B + ((size_t)held.x * N + min(n0 + 16 * wave + 8 * i + (lane >> 3), N - 1)) * lo.R +
                                                     lora_chunk(8 * i, 0, lo.R)),
                                       (lds_ptr)(held_b + 2048 * wave + 1024 * i), 16, 0, 0);
  }
  u32x4_t hv[4 * kTallTiles];
  lora_fetch_h<kTallTiles>(lo, M, mw, min(nw, N - 1), hv);
  asm volatile("" ::: "memory");
  read_ab(a0, b0, sa0, sb0, 0);
  int q = 0;
  for (; q + 3 <= KG; q += 3) {
    group(sa0, sb0, sa1, sb1, q);
    group(sa1, sb1, sa2, sb2, q + 1);
    group(sa2, sb2, sa0, sb0, q + 2);
  }
  if (q < KG) group(sa0, sb0, sa1, sb1, q);
  if (q + 1 < KG) group(sa1, sb1, sa2, sb2, q + 1);
  __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));  // the loads issued past the end have landed
  lds_barrier();  // every wave is done with the stages; every wave's part of the held columns has landed
  // 12 KiB of the stages for each wave: its h, which become operands in registers, then another adapter's columns, its results
  static_assert(kTallA == 24576 && kTallB >= 12288, "two waves to an A stage, one to a B stage");
  char* const own = wave < 6 ? (wave < 2 ? sa0 : wave < 4 ? sa1 : sa2) + 12288 * (wave & 1) : wave == 6 ? sb0 : sb1;
#pragma unroll
  for (int k = 0; k < 4 * kTallTiles; ++k) *reinterpret_cast<u32x4_t*>(own + 1024 * k + 16 * lane) = hv[k];
  bf16x8_t h[kTallTiles][2][2];
#pragma unroll
  for (int t = 0; t < kTallTiles; ++t)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int k = 0; k < 2; ++k) h[t][c][k] = as_bf16x8(*reinterpret_cast<const uint4*>(own + 4096 * t + 2048 * k + (frag ^ (c << 6))));
  asm volatile("" ::: "memory");
  if (nw < N)
    lora_up_block<kTallTiles, true>(lo, M, N, mw, nw, who, [&](int t, int c, int k) __attribute__((always_inline)) { return h[t][c][k]; }, held.x,
                              held_b + 8192 * wn, own, tot);
  // lane (r, g) holds features 16 b + 4g .. +3 of row 16 a + r of the wave's block
  if constexpr (PLANE) {
#pragma unroll
    for (int a = 0; a < kTallTiles; ++a)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (mw + 16 * a + r < M && nw + 16 * b < N)
          *reinterpret_cast<f32x4_dw*>(out + (size_t)(mw + 16 * a + r) * N + nw + 16 * b + 4 * g) = tot[a][b];
  } else {
    // a row's 128 bytes go out together, by way of LDS: 16-byte chunk c of row q sits at position c ^ q % 8
    asm volatile("" ::: "memory");
#pragma unroll
    for (int a = 0; a < kTallTiles; ++a)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        u16x4_t w;
#pragma unroll
        for (int v = 0; v < 4; ++v) w[v] = f2bf(tot[a][b][v] + (bias ? bf2f(bv[b][v]) : 0.f));
        *reinterpret_cast<u16x4_t*>(own + (16 * a + r) * 128 + (((2 * b + (g >> 1)) ^ (r & 7)) << 4) + 8 * (g & 1)) = w;
      }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
    asm volatile("" ::: "memory");
#pragma unroll
    for (int j = 0; j < 2 * kTallTiles; ++j) {
      const int row = 8 * j + (lane >> 3), c = lane & 7, feat = nw + 8 * c;
      u32x4_t w = *reinterpret_cast<const u32x4_t*>(own + row * 128 + ((c ^ (row & 7)) << 4));
      if (mw + row >= M || feat >= N) continue;
      const size_t at = (size_t)(mw + row) * N + feat;
      if (residual) {
        const u32x4_t old = *reinterpret_cast<const u32x4_t*>(residual + at);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = f2bf(__uint_as_float(old[i] << 16) + __uint_as_float(w[i] << 16)) |
                 (uint32_t)f2bf(__uint_as_float(old[i] & 0xffff0000u) + __uint_as_float(w[i] & 0xffff0000u)) << 16;
        *reinterpret_cast<u32x4_t*>(residual + at) = w;
      } else {
        *reinterpret_cast<u32x4_t*>(y + at) = w;
      }
    }
  }
}

int launch_gemm_tall_lora(const uint16_t* x, const uint16_t* W, const uint16_t* b, int M, int N, int K, float* out, uint16_t* y,
                          uint16_t* residual, const LoraArgs& a, hipStream_t s) {
  const int tiles = ceil_div(N, kTallN) * ceil_div(M, kTallM);
  const auto kernel = out ? gemm_tall_lora_kernel<true> : gemm_tall_lora_kernel<false>;
  hipLaunchKernelGGL(kernel, dim3(8 * ceil_div(tiles, 8)), dim3(512), 0, s, x, W, b, M, N, K, out, y, residual, a);
  return check_launch("gemm_tall_lora");
}

// Rounds over the CUs, one workgroup each: a round takes 35 to 40 us (K = 2,880), one of 128 x 128 tiles 28 to 34.  5,120 x 2,880,
// these tiles / those, a prompt with short sequences beside it: 800 rows of 20 adapters (1 round / 2) 50.0 / 49.3 us, 1,000 of 5
// (1 / 2) 40.6 / 50.0, 2,096 of 12 (2 / 3) 71 to 76 / 82 to 85, 3,000 of 9 (3 / 4) 107 / 128, 4,096 of 2 (4 / 5) 150 / 167; in
// sequences of three 800 of 20 50.8 / 64.8, 2,096 of 12 92.9 / 107.6; 2,880 x 4,096: 1,500 rows of 8 (1 / 2) 51.0 / 64.7, 2,000 of 24 in
// threes (1 / 2) 65.9 / 88.8.
bool gemm_tall_pays(int M, int N) {
  const int cus = device_cus(), n = ceil_div(N, kTallN);
  return ceil_div(ceil_div(M, kTallM) * n, cus) < ceil_div(ceil_div(M, 128) * n, cus);
}

}  // namespace flyai
