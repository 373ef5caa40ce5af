// Low-rank adapters of many requests at once, for the kernels that add them to a projection: the arguments, the down
// product h = scale (x A^T) of each row's adapter, and the up product d = h B^T.
#pragma once
#include <type_traits>

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
  // the workspace: h as two bf16 terms [M][n_seg][R32 high | R32 low], R32 = R rounded up to 32, and each row's adapter
  // and rank (0: none)
  uint16_t* h;
  int2* meta;
};

// lora.hip: h alone; the projection's planes with the up products in them (in the tiled kernel's plane, or as one more)
int launch_lora_down(const uint16_t* x, int M, int K, const LoraArgs& a, hipStream_t s);
int launch_gemm_lora_planes(const uint16_t* x, const uint16_t* W, int M, int N, int K, float* part, int* slices, const LoraArgs& a,
                            hipStream_t s);
size_t lora_h_bytes(int M, int R, int n_seg);
void lora_bind(LoraArgs* a, char* ws, int M);
int make_lora_args(LoraArgs* out, const uint16_t* A, const uint16_t* B, const float* scale, const int32_t* ranks, int n, int R,
                   const int32_t* segments, int n_seg, int N, const int32_t* adapter, const int32_t* row_seq, int n_seqs);

constexpr int kLoraCols = 32;  // rank columns of one product: an MFMA's K

__host__ __device__ inline int lora_cols(int R) { return (R + kLoraCols - 1) / kLoraCols * kLoraCols; }

// The segment of feature f (wave-uniform when f is).
__device__ __forceinline__ int lora_segment(const LoraArgs& a, int f) {
  int seg = 0;
#pragma unroll
  for (int i = 0; i < 3; ++i) seg += i + 1 < a.n_seg && f >= a.seg_end[i];
  return seg;
}

// ---- down ----------------------------------------------------------------------------------------------------------
// The batch's work is the pairs of a window of rows and an adapter among them, up to 64 of its rows at a time, times the
// groups of 32 rank columns in every segment.  Each workgroup lists the pairs for itself (adapters of up to 64 * TILES rows
// in LDS, and how many pairs each window has) and takes every wgs-th item: none is launched in vain, whatever the mix.
// A window is WINDOW x 64 rows: wide ones gather an adapter's scattered rows into fewer items, but their list, a wave's, takes
// longer.  Beside the split-K kernel all of its rows (100 rows of 24 adapters 20.9 us, with windows of 64 rows 25.7; 200 rows
// 29.1 / 37.9); alone 128: a prompt with short sequences beside it (64 / 128 / 256: 2,096 rows of 12 adapters 21.1 / 17.6 / 18.9,
// 800 of 20 17.5 / 18.0 / 18.6, 1,000 of 20 at K = 4,096 16.5 / 17.0 / 19.8, 2,096 of one 16.6 / 15.8 / 17.1) is what it is chosen for;
// batches of nothing but short sequences would rather have 256 (2,096 of 12 in threes 62.9 / 41.9 / 35.5, 800 of 20
// 43.3 / 32.4 / 23.6).
// An item multiplies the window's rows that have the adapter, gathered, 16 to an MFMA tile, or (split) a half or a quarter of
// them where the batch has few, with 32 rows of A.  K is cut into
// eight parts, summed in pairs and then in order through LDS, a wave one part or (with four waves) a pair of them; lane
// (r, g) of an MFMA holds row r in its second operand, so a row's products never meet another row's: a row's h depends
// neither on its tile nor on the launch.
// What bounds it is how fast rows of x and A come from L2.  A wave loads whole 128-byte runs (8 rows an instruction) and
// turns them round in LDS of its own (the tiled GEMM's swizzle); loaded as MFMA operands, 16 rows of 64 bytes an
// instruction, every quarter of an instruction touched 16 lines, and 2,096 rows of 192 rank columns took 51 us; now 17 to 19.
// h is kept as two bf16 terms, the value and what its rounding left out: 16 significant bits for the
// bytes of one fp32 value, and the up product takes them as they are.  Each h is off by 2^-17 of itself, d = sum h B by 2^-17 of
// sum |h| |B| at most, which where the sum cancels is more than 2^-17 of d.
constexpr int kDownParts = 8;   // parts of K
constexpr int kDownRows = 64;   // rows of an item
constexpr int kDownCols = kLoraCols;

template <int WAVES, int TILES, int WINDOW>
struct LoraDownLds {
  union {
    char stage[WAVES][(kDownRows + kDownCols) * 128];       // a wave's 64-K group: rows of x, rows of A
    float red[WAVES][kDownRows][kDownCols + 4];
  };
  int adapter[kDownRows * TILES];       // -1 where the row has none, or one of rank 0
  int first[TILES / WINDOW + 1];        // pairs before the window
  int of_seq[64 * WAVES], rank_of[64 * WAVES];
  int row[WAVES][kDownRows];            // the item's rows within its window, for each wave
};

// A window's rows by adapter, in a wave's lanes: take() finds the first adapter that is left, the rows that have it (of) and
// their count, and they leave.
template <int WINDOW>
struct DownRows {
  int key[WINDOW];
  uint64_t left[WINDOW], of[WINDOW];
  int ad, count;
  __device__ __forceinline__ void start(int s, int adapter) { key[s] = adapter, left[s] = __ballot(adapter >= 0); }
  __device__ __forceinline__ bool any() const {
    uint64_t some = 0;
#pragma unroll
    for (int s = 0; s < WINDOW; ++s) some |= left[s];
    return some;
  }
  __device__ __forceinline__ void take() {
    int k = key[WINDOW - 1];
    uint64_t from = left[WINDOW - 1];
#pragma unroll
    for (int s = WINDOW - 2; s >= 0; --s) k = left[s] ? key[s] : k, from = left[s] ? left[s] : from;
    ad = __builtin_amdgcn_readlane(k, __builtin_ctzll(from));
    count = 0;
#pragma unroll
    for (int s = 0; s < WINDOW; ++s) {
      of[s] = __ballot(key[s] == ad);
      left[s] &= ~of[s];
      count += __builtin_popcountll(of[s]);
    }
  }
};

inline int lora_down_groups(const LoraArgs& a) { return a.n_seg * (lora_cols(a.R) / kDownCols); }

// One wave's part of an item's product: up to 8 NX gathered rows (`row`, n of them) against 32 rows of A from ar, over the
// 64-K groups [k0, k1): the sum of the parts before `mid` and from it on, each from zero.  D groups are in flight in
// registers.
template <int NX, int D, bool PAIR>
__device__ __forceinline__ void lora_down_part(const uint16_t* __restrict__ x, const uint16_t* __restrict__ ar, int a_rows, int K,
                                               int m0, int n, int k0, int mid, int k1, char* st, const int* row, f32x4_t (&acc)[4][2]) {
  constexpr int NP = (NX + 1) / 2;           // 16-row tiles (NX == 1: the upper half of one holds what LDS held, for nobody)
  constexpr int NI = NX + kDownCols / 8;     // load instructions a group: 8 rows each
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const uint16_t* src[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int q = 8 * (i < NX ? i : i - NX) + (lane >> 3);
    src[i] = i < NX ? x + (size_t)(m0 + row[min(q, n - 1)]) * K : ar + (size_t)min(q, a_rows - 1) * K;
  }
  u32x4_t buf[D][NI];
  auto load = [&](u32x4_t (&b)[NI], int kg) __attribute__((always_inline)) {
    const int k = 64 * min(kg, k1 - 1);
    const int within = k + 64 <= K ? 7 : 3;  // the last group may have 32 K: the others are read again and not used
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = (lane & 7) ^ (4 * ((i < NX ? i : i - NX) & 1) + (lane >> 4));  // position lane % 8 holds chunk c: the row's swizzle
      b[i] = *reinterpret_cast<const u32x4_t*>(src[i] + k + 8 * (c & within));
    }
  };
#pragma unroll
  for (int d = 0; d < D; ++d) load(buf[d], k0 + d);
  const int frag = r * 128 + ((g ^ ((r >> 1) & 7)) << 4);
  f32x4_t head[PAIR ? NP : 1][2];
  if constexpr (PAIR) {
#pragma unroll
    for (int p = 0; p < NP; ++p) head[p][0] = head[p][1] = f32x4_t{-0.f, -0.f, -0.f, -0.f};  // -0 + x is x
  }
  for (int kb = k0; kb < k1; kb += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (kb + d >= k1) break;
      if constexpr (PAIR) {
        if (kb + d == mid) {
#pragma unroll
          for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int c = 0; c < 2; ++c) head[p][c] = acc[p][c], acc[p][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) *reinterpret_cast<u32x4_t*>(st + 1024 * (i < NX ? i : i - NX + 2 * NP) + 16 * lane) = buf[d][i];
      asm volatile("" ::: "memory");  // this wave's LDS operations complete in order
      load(buf[d], kb + d + D);
      const bool half = 64 * (kb + d) + 64 > K;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (j == 1 && half) break;
        bf16x8_t av[2], xv[NP];
#pragma unroll
        for (int c = 0; c < 2; ++c) av[c] = as_bf16x8(*reinterpret_cast<const uint4*>(st + 2048 * NP + 2048 * c + (frag ^ (j << 6))));
#pragma unroll
        for (int p = 0; p < NP; ++p) xv[p] = as_bf16x8(*reinterpret_cast<const uint4*>(st + 2048 * p + (frag ^ (j << 6))));
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
          for (int c = 0; c < 2; ++c) acc[p][c] = mfma16x16x32(av[c], xv[p], acc[p][c]);
      }
      asm volatile("" ::: "memory");
    }
  }
  if constexpr (PAIR) {
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int c = 0; c < 2; ++c) acc[p][c] = head[p][c] + acc[p][c];
  }
}

template <int WAVES, int TILES, int WINDOW>
__device__ __forceinline__ void lora_down(const uint16_t* __restrict__ x, int M, int K, const LoraArgs& a, int wg, int wgs,
                                          LoraDownLds<WAVES, TILES, WINDOW>& l) {
  constexpr int kThreads = 64 * WAVES, kPairs = kDownParts / WAVES;  // parts a wave
  static_assert(kPairs == 1 || kPairs == 2, "a wave takes a part or a pair");
  constexpr int kSpan = kDownRows * WINDOW;
  constexpr int kWindows = TILES / WINDOW, kMine = (kWindows + WAVES - 1) / WAVES;  // windows a wave lists
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4;
  const int cols = lora_cols(a.R), per_seg = cols / kDownCols, groups = a.n_seg * per_seg;
  const int KG = (K + 63) / 64;
  const int32_t* row_of = a.row_seq ? a.row_seq : a.adapter;
  // Rows, sequences and ranks are fetched side by side where the tables fit a workgroup: one round trip, not three.
  const bool small = a.n <= kThreads && (!a.row_seq || a.n_seqs <= kThreads);
  // A decode batch, one tile: every wave has the tables in its lanes, and no barrier is needed.
  const bool one = M <= kDownRows && a.n <= 64 && (!a.row_seq || a.n_seqs <= 64);
  int key1 = -1, rank1 = 0, pairs1 = 0;
  if (one) {
    const int sq = row_of[min(lane, M - 1)];
    const int of_seq = a.row_seq ? a.adapter[min(lane, a.n_seqs - 1)] : 0;
    const int rank_of = min(max(a.ranks[min(lane, a.n - 1)], 0), a.R);
    int ad = sq;
    if (a.row_seq) {
      ad = __builtin_amdgcn_ds_bpermute(4 * sq, of_seq);
      if ((unsigned)sq >= (unsigned)a.n_seqs) ad = -1;
    }
    rank1 = __builtin_amdgcn_ds_bpermute(4 * ad, rank_of);
    if ((unsigned)ad >= (unsigned)a.n || lane >= M) rank1 = 0;
    key1 = rank1 > 0 ? ad : -1;
    if (wg == 0 && tid < M) a.meta[tid] = make_int2(key1, rank1);
    for (uint64_t todo = __ballot(key1 >= 0); todo; ++pairs1)
      todo &= ~__ballot(key1 == __builtin_amdgcn_readlane(key1, __builtin_ctzll(todo)));
  }
  for (int t0 = 0; t0 < M; t0 += kDownRows * TILES) {
    const int rows = min(M - t0, kDownRows * TILES), windows = (rows + kSpan - 1) / kSpan;
    if (!one) {
      if (t0) __syncthreads();
      int fetched[kMine][WINDOW];
#pragma unroll
      for (int j = 0; j < kMine; ++j)
#pragma unroll
        for (int s = 0; s < WINDOW; ++s)
          fetched[j][s] = row_of[t0 + min(kSpan * (wave + WAVES * j) + kDownRows * s + lane, rows - 1)];
      if (t0 == 0 && small) {
        if (tid < a.n) l.rank_of[tid] = min(max(a.ranks[tid], 0), a.R);
        if (a.row_seq && tid < a.n_seqs) l.of_seq[tid] = a.adapter[tid];
      }
      if (tid == 0) l.first[0] = 0;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kMine; ++j) {
        const int w = wave + WAVES * j;
        if (w >= windows) break;
        DownRows<WINDOW> left;
#pragma unroll
        for (int s = 0; s < WINDOW; ++s) {
          const int i = kSpan * w + kDownRows * s + lane;
          int ad = fetched[j][s], rank = 0;
          if (a.row_seq) {
            const bool in = (unsigned)ad < (unsigned)a.n_seqs;
            const int sq = in ? ad : 0;
            ad = small ? l.of_seq[sq] : a.adapter[sq];
            if (!in) ad = -1;
          }
          if ((unsigned)ad < (unsigned)a.n) rank = small ? l.rank_of[ad] : min(max(a.ranks[ad], 0), a.R);
          if (i >= rows || rank == 0) ad = -1;
          l.adapter[i] = ad;
          if (wg == 0 && i < rows) a.meta[t0 + i] = make_int2(ad, ad < 0 ? 0 : rank);
          left.start(s, ad);
        }
        int n = 0;
        while (left.any()) {
          left.take();
          n += (left.count + kDownRows - 1) / kDownRows;
        }
        if (lane == 0) l.first[w + 1] = n;
      }
      __syncthreads();
      if (wave == 0) {  // running sums
        static_assert(kWindows <= 64, "a lane a window");
        int sum = lane < windows ? l.first[lane + 1] : 0;
#pragma unroll
        for (int off = 1; off < kWindows; off <<= 1) {
          const int o = __shfl_up(sum, off, 64);
          if (lane >= off) sum += o;
        }
        if (lane < windows) l.first[lane + 1] = sum;
      }
      __syncthreads();
    }
    const int pairs = one ? pairs1 : __builtin_amdgcn_readfirstlane(l.first[windows]);
    // few items of many rows are split as far as the workgroups last: 512 rows of one adapter of 192 rank columns are 48 items
    // of 64 rows, 14.1 us, or 192 of 16, 10.4
    const int split = rows < 32 * pairs ? 1 : 4 * pairs * groups <= wgs ? 4 : 2 * pairs * groups <= wgs ? 2 : 1;
    const int items = pairs * groups * split;
    const int before = one ? 0 : l.first[min(lane, windows)];
    // Long items first, and the second round's back from the last workgroup on, so that a short item is followed by another:
    // tiles of many adapters are often at one end of a batch, and the items of the other end are the longer (2,096 rows of 12
    // adapters 20.9 us -> 17.6, 800 rows of 20 22.0 -> 18.0; in sequences of three, items of one length, 800 of 20 30.0 -> 32.4).  Where rows share adapters, an adapter's groups of columns, which
    // read the same rows, go to one XCD, whose L2 then reads them once: 2,096 rows of one adapter 19.4 us -> 15.8, 4,096 of two
    // 33.9 -> 26.7; where they do not, it is 1,000 rows of 20 adapters at K = 4,096 17.7 so and 17.0 in turn.
    const bool back = !one && l.first[1] > pairs - l.first[windows - 1];
    const int me = rows >= 32 * pairs && wg < wgs / 8 * 8 ? wg % 8 * (wgs / 8) + wg / 8 : wg;
    for (int round = 0; round * wgs < items; ++round) {
      const int turn = round * wgs + (round & 1 ? wgs - 1 - me : me);
      if (turn >= items) continue;
      const int it = back ? items - 1 - turn : turn;
      int q0 = it % split * (kDownRows / split);  // the first of the item's rows among the adapter's
      const int ig = it / split;
      const int pair = ig / groups, seg = ig % groups / per_seg, c0 = ig % groups % per_seg * kDownCols;
      const uint64_t below = (1ull << lane) - 1;
      int m0 = t0, ad, n, rank;
      if (one) {
        uint64_t todo = __ballot(key1 >= 0);
        for (int i = 0; i < pair; ++i) todo &= ~__ballot(key1 == __builtin_amdgcn_readlane(key1, __builtin_ctzll(todo)));
        const int lead = __builtin_ctzll(todo);
        ad = __builtin_amdgcn_readlane(key1, lead), rank = __builtin_amdgcn_readlane(rank1, lead);
        const uint64_t rows_of = __ballot(key1 == ad);
        n = min(__builtin_popcountll(rows_of) - q0, kDownRows / split);
        const int at = __builtin_popcountll(rows_of & below) - q0;
        if (key1 == ad && at >= 0) l.row[wave][at] = lane;
      } else {
        const int w = __builtin_popcountll(__ballot(lane < windows && before <= pair)) - 1;  // the last that starts at or before it
        int nth = pair - __builtin_amdgcn_readlane(before, w);
        m0 += kSpan * w;
        DownRows<WINDOW> left;
#pragma unroll
        for (int s = 0; s < WINDOW; ++s) left.start(s, l.adapter[kSpan * w + kDownRows * s + lane]);
        for (;;) {
          left.take();
          const int parts = (left.count + kDownRows - 1) / kDownRows;
          if (nth < parts) break;
          nth -= parts;
        }
        ad = left.ad;
        q0 += kDownRows * nth;
        n = min(left.count - q0, kDownRows / split);
        rank = __builtin_amdgcn_readfirstlane(small ? l.rank_of[ad] : min(max(a.ranks[ad], 0), a.R));
        int past = -q0;
#pragma unroll
        for (int s = 0; s < WINDOW; ++s) {
          const int at = past + __builtin_popcountll(left.of[s] & below);
          if ((left.of[s] >> lane & 1) && at >= 0 && at < n) l.row[wave][at] = kDownRows * s + lane;
          past += __builtin_popcountll(left.of[s]);
        }
      }
      if (n <= 0 || c0 >= rank) continue;  // the same in every wave: columns past the rank's last 32 are never read
      const float scale = a.scale[ad];
      asm volatile("" ::: "memory");  // a wave's LDS operations complete in order
      f32x4_t acc[4][2];
#pragma unroll
      for (int p = 0; p < 4; ++p) acc[p][0] = acc[p][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      const uint16_t* ar = a.A + (((size_t)ad * a.n_seg + seg) * a.R + c0) * K;
      const int e = kPairs * wave, a_rows = min(rank - c0, kDownCols);
      const int k0 = KG * e / kDownParts, mid = kPairs == 2 ? KG * (e + 1) / kDownParts : -1, k1 = KG * (e + kPairs) / kDownParts;
      if (k0 == k1) {}  // fewer groups than waves
      // the fewer rows, the more groups in flight: with few rows there are few items, and latency is all there is
      else if (n <= 8) lora_down_part<1, kPairs == 2 ? 7 : 4, kPairs == 2>(x, ar, a_rows, K, m0, n, k0, mid, k1, l.stage[wave], l.row[wave], acc);
      else if (n <= 16) lora_down_part<2, 4, kPairs == 2>(x, ar, a_rows, K, m0, n, k0, mid, k1, l.stage[wave], l.row[wave], acc);
      else if (n <= 32) lora_down_part<4, 2, kPairs == 2>(x, ar, a_rows, K, m0, n, k0, mid, k1, l.stage[wave], l.row[wave], acc);
      else lora_down_part<8, 1, kPairs == 2>(x, ar, a_rows, K, m0, n, k0, mid, k1, l.stage[wave], l.row[wave], acc);
      __syncthreads();  // red lies over the stages
      // lane (r, g): rank columns 4g .. +3 of row r
#pragma unroll
      for (int p = 0; p < 4; ++p)
        if (16 * p < n) {
#pragma unroll
          for (int c = 0; c < 2; ++c) *reinterpret_cast<f32x4_t*>(&l.red[wave][16 * p + r][16 * c + 4 * g]) = acc[p][c];
        }
      __syncthreads();
      for (int i = tid; i < n * kDownCols; i += kThreads) {
        const int q = i / kDownCols, j = i % kDownCols;
        float v = 0.f;  // columns past the rank are zero, whatever A holds
        if (c0 + j < rank) {
#pragma unroll
          for (int e = 0; e < WAVES; e += WAVES / 4) {
            float pair = l.red[e][q][j];
            if (kPairs == 1) pair += l.red[e + 1][q][j];
            v = e ? v + pair : pair;
          }
          v *= scale;
        }
        uint16_t hi = f2bf(v);
        if ((hi & 0x7fff) == 0x7f80 && fabsf(v) <= 3.402823466e+38f) --hi;  // finite: bf16's largest, and the rest in the low term
        const float rest = v - bf2f(hi);
        uint16_t* o = a.h + ((size_t)(m0 + l.row[wave][q]) * a.n_seg + seg) * 2 * cols + c0 + j;
        o[0] = hi;
        o[cols] = rest == rest ? f2bf(rest) : 0;  // an infinity stays one: inf - inf would be NaN
      }
      __syncthreads();
    }
  }
}

// ---- up ------------------------------------------------------------------------------------------------------------
// d = h B^T in products of 32 rank columns, the high terms of h and then the low ones against the same columns of B: lane
// (r, g) of an operand takes columns 32c + 8g .. +7.  A sum starts from zero for each adapter and is kept by its own rows
// alone, so nothing of another row's adapter, an infinity or a NaN among it, reaches a row, and it does not depend on the
// tile.

// Columns past the rank as zero, whatever they hold; `left` of this lane's eight are within it.
__device__ __forceinline__ bf16x8_t lora_within(uint4 w, int left) {
  uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = 2 * i + 1 < left ? v[i] : 2 * i < left ? v[i] & 0xffffu : 0u;
  return as_bf16x8(make_uint4(v[0], v[1], v[2], v[3]));
}

// Where lane (r, g) reads its eight columns from 32c on in a row of B of R columns (clamped: those past R are masked).
__device__ __forceinline__ int lora_col(int R, int c, int g) { return min(kLoraCols * c + 8 * g, R - 8); }

// 64 columns from c0 of 8 rows of `pitch` elements each as one instruction reads them: lane L takes row L / 8 and the chunk
// that belongs at position L % 8 of row `at` + L / 8 of a tile in the GEMM's swizzle.  Columns past `end` are clamped.
__device__ __forceinline__ int lora_chunk(int at, int c0, int end) {
  const int lane = threadIdx.x & 63, q = at + (lane >> 3);
  return min(c0 + 8 * ((lane & 7) ^ ((q >> 1) & 7)), end - 8);
}

// The tile of workgroup b of a tiled GEMM, row-fastest (-1: none).  As in gemm_tiled_lds_kernel an XCD takes a band of whole
// feature columns, but within it the first and the last rows' tiles come first: a batch's short sequences, and with them
// tiles of many adapters, which take longer, are often at one of its ends, and a long tile must not start last.  2,096 rows of
// which 120 have 12 adapters, 5,120 x 2,880: 78.4 us in the other's order, 72.9 in this (4,096 rows of two 146.5 and 150.1).
__device__ __forceinline__ int lora_tile(int b, int gm, int gn) {
  const int per = (gm * gn + 7) / 8, start = b % 8 * per, end = min(start + per, gm * gn), i = b / 8;
  if (start + i >= end) return -1;
  if (gm <= 2) return start + i;
  const int first = (start + gm - 1) / gm, n_first = (end + gm - 1) / gm - first;  // columns whose first tile is in the band
  const int last = start / gm, n_last = end / gm - last;                           // ... whose last one is
  if (i < n_first) return (first + i) * gm;
  if (i < n_first + n_last) return (last + i - n_first) * gm + gm - 1;
  const int inner = last * (gm - 2) + max(start - last * gm - 1, 0) + i - n_first - n_last;  // inner tiles before it
  return inner / (gm - 2) * gm + 1 + inner % (gm - 2);
}

// h of a tiled GEMM's wave, 16 MT rows from m0 in the segment of feature f0, columns 0 .. 63: h[4 a + 2 t + i] is rows 16 a +
// 8 i .. +7, high (t = 0) or low terms, for 1 KiB of LDS each.
template <int MT>
__device__ __forceinline__ void lora_fetch_h(const LoraArgs& a, int M, int m0, int f0, u32x4_t (&h)[4 * MT]) {
  const int cols = lora_cols(a.R), seg = lora_segment(a, f0);
#pragma unroll
  for (int k = 0; k < 4 * MT; ++k) {
    const int row = m0 + 16 * (k >> 2) + 8 * (k & 1) + ((threadIdx.x & 63) >> 3);
    h[k] = *reinterpret_cast<const u32x4_t*>(a.h + ((size_t)min(row, M - 1) * a.n_seg + seg) * 2 * cols + (k & 2 ? cols : 0) +
                                             lora_chunk(8 * (k & 1), 0, cols));
  }
}

// The up products of 16 MT rows from m0 and 64 features from f0 (one segment; a wave's, uniform), added to a tiled GEMM's
// sums: lane (r, g) holds rows 16 t + 4g .. +3 of feature f0 + 16 b + r in sum[t][b], or (FEATURES) features f0 + 16 b + 4g ..
// +3 of row 16 t + r.  `who`: row m0 + lane's adapter and rank.  h(t, c, k): this lane's operand of row tile t, columns 32c ..
// +31, high (k = 0) or low terms; held_b: columns 0 .. 63 of adapter `held` (-1: of none), this wave's features, 16 to a
// tile; bl: room for an adapter's, which come in whole runs like the GEMM's operands (as MFMA operands from memory a tile of
// 128 rows of 45 adapters took 50,000 clocks, more than its projection).  Columns past the rank become zero on their way to
// LDS.  A CU runs this once a tile, so its time is the code's way from memory as much as anything: masking at the products,
// with twice the instructions, was 2 us slower at 2,096 rows, two adapters in flight (twice the code again) 10.
template <int MT, bool FEATURES, typename H>
__device__ __forceinline__ void lora_up_block(const LoraArgs& a, int M, int N, int m0, int f0, int2 who, const H& h, int held,
                                              const char* held_b, char* bl, f32x4_t (&sum)[MT][4]) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int key = lane < 16 * MT && m0 + lane < M && who.y > 0 ? who.x : -1;
  uint64_t todo = __ballot(key >= 0);
  if (!todo) return;
  int of_row[MT][FEATURES ? 1 : 4];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int v = 0; v < (FEATURES ? 1 : 4); ++v) of_row[t][v] = __builtin_amdgcn_ds_bpermute(4 * (16 * t + (FEATURES ? r : 4 * g + v)), key);
  uint32_t off[8];  // of the lane's chunks in an adapter's rows from f0 on
#pragma unroll
  for (int k = 0; k < 8; ++k) off[k] = min(8 * k + (lane >> 3), N - 1 - f0) * a.R + lora_chunk(8 * (k & 1), 0, a.R);
  u32x4_t nb[8];
  auto columns = [&](int ad) __attribute__((always_inline)) { return a.B + ((size_t)ad * N + f0) * a.R; };
  auto fetch = [&](int ad) __attribute__((always_inline)) {
    if (ad == held) return;
    const uint16_t* B = columns(ad);
#pragma unroll
    for (int k = 0; k < 8; ++k) nb[k] = *reinterpret_cast<const u32x4_t*>(B + off[k]);
  };
  const int frag = r * 128 + ((g ^ ((r >> 1) & 7)) << 4);
  int ad = __builtin_amdgcn_readlane(key, __builtin_ctzll(todo));
  fetch(ad);
  while (ad >= 0) {
    const int now = ad, rank = __builtin_amdgcn_readlane(who.y, __builtin_ctzll(todo));
    const uint64_t rows = __ballot(key == now);
    if (now == held) {
#pragma unroll
      for (int k = 0; k < 8; ++k) nb[k] = *reinterpret_cast<const u32x4_t*>(held_b + 1024 * k + 16 * lane);
    }
    if (rank < 2 * kLoraCols) {
      uint32_t keep[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int left = rank - 8 * ((lane & 7) ^ (4 * i + (lane >> 4)));  // of the chunk's eight columns
#pragma unroll
        for (int j = 0; j < 4; ++j) keep[i][j] = 2 * j + 1 < left ? 0xffffffffu : 2 * j < left ? 0xffffu : 0u;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) nb[k][j] &= keep[k & 1][j];
    }
    asm volatile("" ::: "memory");  // a wave's LDS operations complete in order
#pragma unroll
    for (int k = 0; k < 8; ++k) *reinterpret_cast<u32x4_t*>(bl + 1024 * k + 16 * lane) = nb[k];
    asm volatile("" ::: "memory");
    todo &= ~rows;
    ad = todo ? __builtin_amdgcn_readlane(key, __builtin_ctzll(todo)) : -1;
    if (ad >= 0) fetch(ad);  // on its way under this one's products
    auto product = [&](bf16x8_t w, bf16x8_t v, f32x4_t c) __attribute__((always_inline)) {
      return FEATURES ? mfma16x16x32(w, v, c) : mfma16x16x32(v, w, c);
    };
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      if (!(rows >> (16 * t) & 0xffff)) continue;
      f32x4_t up[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) up[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (kLoraCols * c >= rank) break;
        const bf16x8_t hi = h(t, c, 0), lo = h(t, c, 1);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const bf16x8_t w = as_bf16x8(*reinterpret_cast<const uint4*>(bl + 2048 * b + (frag ^ (c << 6))));
          up[b] = product(w, hi, up[b]);
          up[b] = product(w, lo, up[b]);
        }
      }
      for (int c = 2; kLoraCols * c < rank; ++c) {  // ranks past 64: straight from memory
        const int row = min(m0 + 16 * t + r, M - 1), left = rank - kLoraCols * c, cols = lora_cols(a.R);
        const uint16_t* hr = a.h + ((size_t)row * a.n_seg + lora_segment(a, f0)) * 2 * cols + kLoraCols * c + 8 * g;
        const bf16x8_t hi = as_bf16x8(*reinterpret_cast<const uint4*>(hr));
        const bf16x8_t lo = as_bf16x8(*reinterpret_cast<const uint4*>(hr + cols));
        const uint16_t* B = columns(now);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const bf16x8_t w = lora_within(*reinterpret_cast<const uint4*>(B + (uint32_t)(min(16 * b + r, N - 1 - f0) * a.R + lora_col(a.R, c, g))),
                                         left - 8 * g);
          up[b] = product(w, hi, up[b]);
          up[b] = product(w, lo, up[b]);
        }
      }
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int v = 0; v < 4; ++v) sum[t][b][v] += of_row[t][FEATURES ? 0 : v] == now ? up[b][v] : -0.f;
    }
  }
}

}  // namespace flyai
