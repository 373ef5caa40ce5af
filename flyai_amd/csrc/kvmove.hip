// The cache's slabs forked and compacted: every layer, K and V, every kv head in a launch (kForkDsts slabs; kMoveSlabs slabs and
// kMoveWords blocks of what they span).
#include <algorithm>

#include "common.h"

namespace flyai {

// Both kernels move bits only: what bounds them is the bytes, and for few positions the launch.  What the host knows of
// a call (slabs, positions) travels in the kernel's arguments, so a call makes no copy to the device and a captured
// one keeps its plan.

// ---- fork: positions [lo, hi) of one slab to the same positions of others --------------------------------------
// Equal positions have equal places within a head region's 64-position blocks, so the copy is of 16-byte chunks: eight
// dims of one position in K, eight consecutive positions of one dim in V (the edge chunks of V go element by element).
// A source chunk is read once and stored to every destination: 3,001 positions of 18 layers to four slabs, 553 MB, take 107 us,
// 5.2 TB/s; 77 positions of 12 layers 3.2 us, a launch and a round trip.
constexpr int kForkDsts = 64;
constexpr int kForkThreads = 256;
constexpr int kForkChunks = 2;  // 16-byte chunks a thread: a workgroup moves one 8 KiB block

struct ForkArgs {
  const uint16_t* src[2];  // K, V
  uint16_t* dst[2];
  int64_t src_layer, dst_layer;  // elements from a layer's pool to the next
  int64_t src_base;
  int src_cap, heads, lo, hi, n_dst;
  int64_t dst_base[kForkDsts];
  int dst_cap[kForkDsts];
};

__global__ __launch_bounds__(kForkThreads) void kv_fork_kernel(ForkArgs a) {
  const int kind = blockIdx.y & 1, head = blockIdx.y >> 1, layer = blockIdx.z;
  const int blk = (a.lo >> 6) + blockIdx.x;
  const uint16_t* src = a.src[kind] + layer * a.src_layer + a.src_base + (int64_t)head * a.src_cap * 64 + (int64_t)blk * 4096;
  uint16_t* dst = a.dst[kind] + layer * a.dst_layer + (int64_t)blk * 4096;
  u32x4_t v[kForkChunks];
#pragma unroll
  for (int j = 0; j < kForkChunks; ++j)
    v[j] = reinterpret_cast<const u32x4_t*>(src)[threadIdx.x + kForkThreads * j];
  int mask[kForkChunks];  // which of the chunk's elements are inside [lo, hi)
#pragma unroll
  for (int j = 0; j < kForkChunks; ++j) {
    const int c = threadIdx.x + kForkThreads * j, lane = c & 63;
    mask[j] = 0;
    if (kind == 0) {
      const int kt = c >> 7, n = lane & 15;
      const int pos = blk * 64 + 32 * (kt >> 1) + 8 * (n >> 2) + 4 * (kt & 1) + (n & 3);
      mask[j] = pos >= a.lo && pos < a.hi ? 255 : 0;
    } else {
      const int pos = blk * 64 + 32 * (c >> 8) + 8 * (lane >> 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) mask[j] |= (pos + i >= a.lo && pos + i < a.hi) << i;
    }
  }
  for (int d = 0; d < a.n_dst; ++d) {
    uint16_t* to = dst + a.dst_base[d] + (int64_t)head * a.dst_cap[d] * 64;
#pragma unroll
    for (int j = 0; j < kForkChunks; ++j) {
      const int c = threadIdx.x + kForkThreads * j;
      if (mask[j] == 255) {
        reinterpret_cast<u32x4_t*>(to)[c] = v[j];
      } else if (mask[j]) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (mask[j] >> i & 1) to[8 * c + i] = (uint16_t)(v[j][i >> 1] >> (16 * (i & 1)));
      }
    }
  }
}

// ---- compact: within a slab, the kept positions move up, in order ------------------------------------------------
// A kept position never moves down, so a part of the positions, read whole before it is written, overwrites nothing that
// a later part reads.  A slab's dims do not depend on each other: a workgroup owns 16 dims of one head of one layer's K or
// V and goes through the positions in parts of 256, through LDS, needing nothing from other workgroups.  What stays is a
// bitmap, a word per 64-position block.
// Four slabs of 2,041 moved rows in 8 layers, 267 MB: 198 us with the positions themselves in the arguments (704 a launch,
// 12 launches), 106 with parts of 1,024 in registers (whose unrolled code, 20 KB, cost a launch of 6 rows 18 us), now 62,
// 4.3 TB/s; parts of 128, 512 and 1,024 take 67, 68 and 71.  1,501 scattered rows of 6,000 (two slabs, 12 layers): 98 us, 82
// and 67, most of it for lines that few kept positions share.
// Each part costs a workgroup some 1.2 us whatever it keeps, so where few positions stay the parts are wider, as many blocks
// (16 to 64) as keep 256 positions at most, and V's elements are read one by one: 600 of 8,000 positions of one layer 38 us in
// parts of 256, 13.4 in wide ones, 100 of 4,000 (two slabs, three layers) 22 and 5.3.  Parts of eight blocks so were slower (a
// quarter of the positions kept: 76 us, 66 in parts of four).
constexpr int kMoveThreads = 256;
constexpr int kMoveBlocks = 4;    // 64-position blocks of a part
constexpr int kMoveWide = 64;     // ... of a part that keeps few
constexpr int kMoveKept = 64 * kMoveBlocks;  // positions that a part keeps at most
constexpr int kMoveRow = kMoveKept + 8;      // a dim's positions in LDS, + 16 B vs bank conflicts
constexpr int kMoveWords = 336;   // words of a launch: 21,504 positions
constexpr int kMoveSlabs = 16;

struct MoveSlab {
  int64_t base;
  int cap, dst;             // the first kept position goes to dst
  int block, first, words;  // words[first ..] are blocks block .. block + words - 1
  int part, kept;           // blocks of a part, positions kept in all
};

struct MoveArgs {
  uint16_t* pool[2];
  int64_t layer;
  MoveSlab slab[kMoveSlabs];
  uint64_t words[kMoveWords];
  uint16_t before[kMoveWords];  // positions that the slab's words before it keep
};
static_assert(sizeof(MoveArgs) <= 4096 && sizeof(ForkArgs) <= 4096, "kernel arguments are at most 4 KiB");

struct MoveLds {
  uint16_t kept[kMoveKept];  // of the part: offsets from its first position
  __align__(16) uint16_t data[16 * kMoveRow];
  uint64_t bits[kMoveWords];  // WIDE: the slab's words and `before`, read once
  int before[kMoveWords + 1];
};

// WIDE: parts of m.part blocks, kMoveBlocks otherwise.
template <bool WIDE>
__device__ __forceinline__ void compact_slab(const MoveArgs& a, const MoveSlab& m, MoveLds& l) {
  uint16_t *kept = l.kept, *data = l.data;
  uint64_t* bits = l.bits;
  int* before = l.before;
  const int kind = blockIdx.x & 1, dq = (blockIdx.x >> 1) & 3, head = blockIdx.x >> 3;
  uint16_t* region = a.pool[kind] + blockIdx.z * a.layer + m.base + (int64_t)head * m.cap * 64;
  const int tid = threadIdx.x;
  const int part = WIDE ? m.part : kMoveBlocks;
  if constexpr (WIDE) {
    for (int i = tid; i <= m.words; i += kMoveThreads) {
      if (i < m.words) bits[i] = a.words[m.first + i];
      before[i] = i < m.words ? a.before[m.first + i] : m.kept;
    }
    __syncthreads();
  }
  int dst = m.dst;
  for (int b0 = 0; b0 < m.words; b0 += part) {
    const int p0 = 64 * (m.block + b0);
    uint64_t words[kMoveBlocks];
    int n = 0;
    if constexpr (!WIDE) {
#pragma unroll
      for (int i = 0; i < kMoveBlocks; ++i) {
        words[i] = b0 + i < m.words ? a.words[min(m.first + b0 + i, kMoveWords - 1)] : 0;
        n += __builtin_popcountll(words[i]);
      }
      if (n == 0) continue;
      constexpr int kPer = 64 * kMoveBlocks / kMoveThreads;  // positions a thread
      const int blk = kPer * tid / 64, bit = kPer * tid % 64;
      uint64_t word = 0;
      int at = 0;
#pragma unroll
      for (int i = 0; i < kMoveBlocks; ++i) {
        if (i < blk) at += __builtin_popcountll(words[i]);
        if (i == blk) word = words[i];
      }
      at += __builtin_popcountll(word & ((1ull << bit) - 1));
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (word >> (bit + i) & 1) kept[at++] = (uint16_t)(64 * blk + bit + i);
    } else {
      n = __builtin_amdgcn_readfirstlane(before[min(b0 + part, m.words)] - before[b0]);
      if (n == 0) continue;
      const int per = 64 * part / kMoveThreads;  // positions a thread, of one word
      const int w = per * tid / 64, bit = per * tid % 64;
      if (b0 + w < m.words) {
        const uint64_t word = bits[b0 + w];
        int at = before[b0 + w] - before[b0] + __builtin_popcountll(word & ((1ull << bit) - 1));
        for (uint32_t some = word >> bit & ((1u << per) - 1); some; some &= some - 1)
          kept[at++] = (uint16_t)(64 * w + bit + __builtin_ctz(some));
      }
    }
    if (kind == 0) {
      // K: 16 dims of a row are two 16-byte chunks
      __syncthreads();
#pragma unroll 4
      for (int u = tid; u < 2 * n; u += kMoveThreads)
        reinterpret_cast<u32x4_t*>(data)[u] =
            *reinterpret_cast<const u32x4_t*>(region + kv_k_off(p0 + kept[u >> 1], 16 * dq + 8 * (u & 1)));
      __syncthreads();
      for (int u = tid; u < 2 * n; u += kMoveThreads)
        *reinterpret_cast<u32x4_t*>(region + kv_k_off(dst + (u >> 1), 16 * dq + 8 * (u & 1))) = reinterpret_cast<u32x4_t*>(data)[u];
    } else {
      // V: a chunk is one dim of eight positions; those with none kept are not read.  A destination chunk's elements come
      // from wherever each lies.  A wide part's are read one by one, in their order.
      if constexpr (WIDE) {
        __syncthreads();
#pragma unroll 4
        for (int u = tid; u < 16 * n; u += kMoveThreads)
          data[(u & 15) * kMoveRow + (u >> 4)] = region[kv_v_off(p0 + kept[u >> 4], 16 * dq + (u & 15))];
      } else {
        constexpr int kBlocks = kMoveThreads / 16 / 8;  // that an iteration reads
        static_assert(kMoveBlocks % kBlocks == 0 && kMoveThreads % 128 == 0, "whole iterations of whole blocks");
#pragma unroll
        for (int j = 0; j < 16 * 8 * kMoveBlocks / kMoveThreads; ++j) {
          const int u = tid + kMoveThreads * j, d = u & 15, g = u >> 4;  // chunk: dim, eighth positions
          uint64_t word = 0;
#pragma unroll
          for (int i = 0; i < kBlocks; ++i)
            if (g >> 3 == kBlocks * j + i) word = words[kBlocks * j + i];
          if (word >> (8 * (g & 7)) & 255)
            *reinterpret_cast<u32x4_t*>(data + d * kMoveRow + 8 * g) = *reinterpret_cast<const u32x4_t*>(region + kv_v_off(p0 + 8 * g, 16 * dq + d));
        }
      }
      __syncthreads();
      const int g0 = dst >> 3, units = 16 * (((dst + n - 1) >> 3) - g0 + 1);
      for (int u = tid; u < units; u += kMoveThreads) {
        const int d = u & 15, at = 8 * (g0 + (u >> 4)), i0 = at - dst;
        uint16_t e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int at_i = min(max(i0 + i, 0), n - 1);
          e[i] = data[d * kMoveRow + (WIDE ? at_i : kept[at_i])];
        }
        uint16_t* to = region + kv_v_off(at, 16 * dq + d);
        if (i0 >= 0 && i0 + 7 < n) {
          u32x4_t w;
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = e[2 * i] | (uint32_t)e[2 * i + 1] << 16;
          *reinterpret_cast<u32x4_t*>(to) = w;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i0 + i >= 0 && i0 + i < n) to[i] = e[i];
        }
      }
    }
    __syncthreads();  // the part's LDS is free again
    dst += n;
  }
}

__global__ __launch_bounds__(kMoveThreads) void kv_compact_kernel(MoveArgs a) {
  __shared__ MoveLds lds;
  const MoveSlab& m = a.slab[blockIdx.y];
  if (m.part > kMoveBlocks) compact_slab<true>(a, m, lds);
  else compact_slab<false>(a, m, lds);
}

static int check_slab(const char* what, int64_t base, int cap, int heads, int64_t pool_elems) {
  FLYAI_REQUIRE(cap > 0 && cap % 64 == 0 && base >= 0 && base % 8 == 0,
                "%s: a slab needs cap %% 64 == 0 and base %% 8 == 0", what);
  if (base > pool_elems - (int64_t)heads * cap * 64)  // no sum that could wrap
    return set_error(FLYAI_ERANGE, "%s: slab at %lld of %d positions ends past the pool (%lld elements)", what,
                     (long long)base, cap, (long long)pool_elems);
  return FLYAI_OK;
}

static int check_pools(const char* what, const void* k, const void* v, int64_t layer, int64_t elems, int n_layers,
                       int heads, int D) {
  FLYAI_REQUIRE(k && v, "%s: null pool", what);
  FLYAI_REQUIRE(((uintptr_t)k | (uintptr_t)v) % 16 == 0, "%s: pools must be 16-byte aligned", what);
  FLYAI_REQUIRE(n_layers >= 1 && n_layers <= 65535 && heads >= 1 && heads <= 4096 && D == 64,
                "%s: needs layers and kv heads, and head_dim 64", what);
  FLYAI_REQUIRE(n_layers == 1 || (layer % 8 == 0 && layer >= elems),
                "%s: the layer stride must be a multiple of 8 and no less than a layer's pool", what);
  return FLYAI_OK;
}

// Whether two pools of n_layers layers share no element: spans that lie apart, or layers at one distance that lie between
// each other's.
static bool pools_apart(const uint16_t* a, int64_t a_layer, int64_t a_elems, const uint16_t* b, int64_t b_layer, int64_t b_elems,
                        int n_layers) {
  const uintptr_t A = (uintptr_t)a, B = (uintptr_t)b;
  const uint64_t far_a = 2 * ((uint64_t)(n_layers - 1) * a_layer + a_elems), far_b = 2 * ((uint64_t)(n_layers - 1) * b_layer + b_elems);
  if (A <= B ? B - A >= far_a : A - B >= far_b) return true;
  if (n_layers == 1 || a_layer != b_layer) return false;
  const uint64_t step = 2 * (uint64_t)a_layer, off = A <= B ? (B - A) % step : (step - (A - B) % step) % step;  // b's layers behind a's
  return off >= 2 * (uint64_t)a_elems && step - off >= 2 * (uint64_t)b_elems;
}

}  // namespace flyai

using namespace flyai;

#define RUN(x)             \
  do {                     \
    const int rc__ = (x);  \
    if (rc__) return rc__; \
  } while (0)

extern "C" int flyai_kv_fork(const uint16_t* src_k, const uint16_t* src_v, int64_t src_layer, int64_t src_elems,
                             uint16_t* dst_k, uint16_t* dst_v, int64_t dst_layer, int64_t dst_elems, int32_t n_layers,
                             int32_t Hkv, int32_t D, const flyai_kv_slab* src_host, const flyai_kv_slab* dsts_host, int32_t n_dst,
                             int32_t lo, int32_t hi, flyai_stream_t stream) {
  RUN(check_pools("kv_fork", src_k, src_v, src_layer, src_elems, n_layers, Hkv, D));
  RUN(check_pools("kv_fork", dst_k, dst_v, dst_layer, dst_elems, n_layers, Hkv, D));
  const bool same = src_k == dst_k && src_v == dst_v && (n_layers == 1 || src_layer == dst_layer);
  FLYAI_REQUIRE(src_host && n_dst >= 0 && (n_dst == 0 || dsts_host), "kv_fork: null slab");
  const flyai_kv_slab src = *src_host;
  FLYAI_REQUIRE(0 <= lo && lo <= hi, "kv_fork: positions [%d, %d) are no range", lo, hi);
  RUN(check_slab("kv_fork", src.base, src.cap, Hkv, src_elems));
  if (hi > src.cap) return set_error(FLYAI_ERANGE, "kv_fork: position %d past the source's %d", hi, src.cap);
  for (int i = 0; i < n_dst; ++i) {
    const flyai_kv_slab& d = dsts_host[i];
    RUN(check_slab("kv_fork", d.base, d.cap, Hkv, dst_elems));
    if (hi > d.cap) return set_error(FLYAI_ERANGE, "kv_fork: position %d past destination %d's %d", hi, i, d.cap);
    // the destinations are written while the source is read, and side by side
    auto apart = [&](const flyai_kv_slab& o) {
      return o.base + (int64_t)Hkv * o.cap * 64 <= d.base || d.base + (int64_t)Hkv * d.cap * 64 <= o.base;
    };
    FLYAI_REQUIRE(!same || apart(src), "kv_fork: destination %d overlaps the source", i);
    for (int j = 0; j < i; ++j) FLYAI_REQUIRE(apart(dsts_host[j]), "kv_fork: destinations %d and %d overlap", j, i);
  }
  if (lo == hi || n_dst == 0) return FLYAI_OK;
  // K and V are written side by side, and the source is read meanwhile: its pools are the destinations' or share nothing
  FLYAI_REQUIRE(pools_apart(dst_k, dst_layer, dst_elems, dst_v, dst_layer, dst_elems, n_layers), "kv_fork: the K and V pools overlap");
  const uint16_t *srcs[2] = {src_k, src_v}, *dsts[2] = {dst_k, dst_v};
  for (int i = 0; i < 4 && !same; ++i)
    FLYAI_REQUIRE(pools_apart(srcs[i & 1], src_layer, src_elems, dsts[i >> 1], dst_layer, dst_elems, n_layers),
                  "kv_fork: the source's pools overlap the destinations' and are not the same");
  hipStream_t s = as_stream(stream);
  for (int i = 0; i < n_dst; i += kForkDsts) {
    ForkArgs a;
    a.src[0] = src_k, a.src[1] = src_v, a.dst[0] = dst_k, a.dst[1] = dst_v;
    a.src_layer = src_layer, a.dst_layer = dst_layer, a.src_base = src.base, a.src_cap = src.cap;
    a.heads = Hkv, a.lo = lo, a.hi = hi, a.n_dst = std::min(kForkDsts, n_dst - i);
    for (int j = 0; j < a.n_dst; ++j) a.dst_base[j] = dsts_host[i + j].base, a.dst_cap[j] = dsts_host[i + j].cap;
    hipLaunchKernelGGL(kv_fork_kernel, dim3(((hi - 1) >> 6) - (lo >> 6) + 1, 2 * Hkv, n_layers), dim3(kForkThreads), 0, s, a);
    RUN(check_launch("kv_fork"));
  }
  return FLYAI_OK;
}

extern "C" int flyai_kv_compact(uint16_t* k_pool, uint16_t* v_pool, int64_t layer, int64_t pool_elems, int32_t n_layers,
                                int32_t Hkv, int32_t D, const flyai_kv_move* moves_host, int32_t n_moves,
                                const int32_t* keep_host, flyai_stream_t stream) {
  RUN(check_pools("kv_compact", k_pool, v_pool, layer, pool_elems, n_layers, Hkv, D));
  FLYAI_REQUIRE(n_moves >= 0 && (n_moves == 0 || moves_host), "kv_compact: null moves");
  int64_t first = 0;
  for (int i = 0; i < n_moves; ++i) {
    const flyai_kv_move& m = moves_host[i];
    RUN(check_slab("kv_compact", m.base, m.cap, Hkv, pool_elems));
    FLYAI_REQUIRE(m.start >= 0 && m.n >= 0 && (m.n == 0 || keep_host), "kv_compact: move %d is no range", i);
    if ((int64_t)m.start + m.n > m.cap)
      return set_error(FLYAI_ERANGE, "kv_compact: move %d ends past its slab's %d positions", i, m.cap);
    const int32_t* keep = keep_host + first;
    for (int r = 0; r < m.n; ++r) {
      FLYAI_REQUIRE(keep[r] >= 0 && (r == 0 || keep[r] > keep[r - 1]),
                    "kv_compact: move %d must keep positions in strictly ascending order (entry %d)", i, r);
      if ((int64_t)m.start + keep[r] >= m.cap)
        return set_error(FLYAI_ERANGE, "kv_compact: move %d keeps position %d + %d of a slab of %d", i, m.start, keep[r], m.cap);
    }
    for (int j = 0; j < i; ++j) {
      const flyai_kv_move& o = moves_host[j];
      FLYAI_REQUIRE(o.base + (int64_t)Hkv * o.cap * 64 <= m.base || m.base + (int64_t)Hkv * m.cap * 64 <= o.base,
                    "kv_compact: moves %d and %d are of overlapping slabs", j, i);
    }
    first += m.n;
  }
  hipStream_t s = as_stream(stream);
  MoveArgs a;
  a.pool[0] = k_pool, a.pool[1] = v_pool, a.layer = layer;
  int slabs = 0, words = 0;
  auto flush = [&]() -> int {
    if (slabs == 0) return FLYAI_OK;
    FLYAI_REQUIRE(pools_apart(k_pool, layer, pool_elems, v_pool, layer, pool_elems, n_layers), "kv_compact: the K and V pools overlap");
    hipLaunchKernelGGL(kv_compact_kernel, dim3(8 * Hkv, slabs, n_layers), dim3(kMoveThreads), 0, s, a);
    slabs = words = 0;
    return check_launch("kv_compact");
  };
  first = 0;
  for (int i = 0; i < n_moves; ++i) {
    const flyai_kv_move& m = moves_host[i];
    const int32_t* keep = keep_host + first;
    first += m.n;
    int r = 0;
    while (r < m.n && keep[r] == r) ++r;  // positions that stay where they are
    while (r < m.n) {
      // a slab's kept positions go into one launch as far as its words last; the next launch takes up from there
      if (slabs == kMoveSlabs || words == kMoveWords) RUN(flush());
      MoveSlab& out = a.slab[slabs++];
      out = MoveSlab{m.base, m.cap, m.start + r, (m.start + keep[r]) >> 6, words, 0, kMoveWide, -r};
      for (; r < m.n; ++r) {
        const int pos = m.start + keep[r], w = (pos >> 6) - out.block;
        if (out.first + w >= kMoveWords) break;
        for (; out.words <= w; ++out.words) a.words[words++] = 0;
        a.words[out.first + w] |= 1ull << (pos & 63);
      }
      out.kept += r;
      // the widest parts none of which keeps too many, from 1,024 positions on
      for (int w = 0, n = 0; w < out.words; ++w) a.before[out.first + w] = (uint16_t)n, n += __builtin_popcountll(a.words[out.first + w]);
      auto fits = [&](int part) {
        for (int w = 0; w < out.words; w += part)
          if ((w + part < out.words ? a.before[out.first + w + part] : out.kept) - a.before[out.first + w] > kMoveKept) return false;
        return true;
      };
      while (out.part > kMoveBlocks && (out.part == 2 * kMoveBlocks || out.words <= out.part / 2 || !fits(out.part))) out.part /= 2;
      if (r < m.n) RUN(flush());  // the rest moves into positions that this piece reads
    }
  }
  return flush();
}
