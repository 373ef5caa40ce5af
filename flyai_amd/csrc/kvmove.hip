// The cache's slabs forked and compacted: every layer, K and V, every kv head in one launch.
#include <algorithm>
#include <vector>

#include "common.h"

namespace flyai {

// Both kernels move bits only: what bounds them is the bytes, and for few positions the launch.  What the host knows of
// a call (slabs, positions) travels in the kernel's arguments, so a call makes no copy to the device and a captured
// one keeps its plan.

// ---- fork: positions [lo, hi) of one slab to the same positions of others --------------------------------------
// Equal positions have equal places within a head region's 64-position blocks, so the copy is of 16-byte chunks: eight
// dims of one position in K, eight consecutive positions of one dim in V (the edge chunks of V go element by element).
// A source chunk is read once and stored to every destination.
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

// ---- compact: within a slab, position start + i takes position start + keep[i] --------------------------------
// A slab's dims are independent of each other: a workgroup owns 16 dims of one head of one layer's K or V, reads all
// of its rows into registers and only then writes, so it needs nothing from any other workgroup.  A launch takes up to
// kMoveRows rows; with keep ascending, a later launch's sources lie past every earlier one's destinations.
constexpr int kMoveRows = 704;
constexpr int kMoveSlabs = 24;
constexpr int kMoveThreads = 256;

struct MoveSlab {
  int64_t base;
  int cap, start, first, n;  // rows start .. start + n - 1 take start0 + keep[first ..]
  int from;                  // what keep counts from
};

struct MoveArgs {
  uint16_t* pool[2];
  int64_t layer;
  int heads, n_slabs;
  MoveSlab slab[kMoveSlabs];
  int keep[kMoveRows];
};
static_assert(sizeof(MoveArgs) <= 4096 && sizeof(ForkArgs) <= 4096, "kernel arguments are at most 4 KiB");

__global__ __launch_bounds__(kMoveThreads) void kv_compact_kernel(MoveArgs a) {
  const int kind = blockIdx.x & 1, dq = (blockIdx.x >> 1) & 3, head = blockIdx.x >> 3, layer = blockIdx.z;
  const MoveSlab& m = a.slab[blockIdx.y];
  uint16_t* region = a.pool[kind] + layer * a.layer + m.base + (int64_t)head * m.cap * 64;
  const int* keep = a.keep + m.first;
  const int n = m.n;
  if (kind == 0) {
    // K: 16 dims of a row are two 16-byte chunks
    constexpr int kPer = (2 * kMoveRows + kMoveThreads - 1) / kMoveThreads;
    u32x4_t v[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int u = threadIdx.x + kMoveThreads * j;
      if (u < 2 * n) v[j] = *reinterpret_cast<const u32x4_t*>(region + kv_k_off(m.from + keep[u >> 1], 16 * dq + 8 * (u & 1)));
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int u = threadIdx.x + kMoveThreads * j;
      if (u < 2 * n) *reinterpret_cast<u32x4_t*>(region + kv_k_off(m.start + (u >> 1), 16 * dq + 8 * (u & 1))) = v[j];
    }
  } else {
    // V: a destination chunk is one dim of eight positions; its elements come from eight places
    constexpr int kPer = (16 * (kMoveRows / 8 + 1) + kMoveThreads - 1) / kMoveThreads;
    const int g0 = m.start >> 3, units = 16 * (((m.start + n - 1) >> 3) - g0 + 1);
    uint16_t v[kPer][8];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int u = threadIdx.x + kMoveThreads * j;
      if (u < units) {
        const int d = 16 * dq + (u & 15), i0 = 8 * (g0 + (u >> 4)) - m.start;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] = region[kv_v_off(m.from + keep[min(max(i0 + i, 0), n - 1)], d)];
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int u = threadIdx.x + kMoveThreads * j;
      if (u < units) {
        const int d = 16 * dq + (u & 15), p0 = 8 * (g0 + (u >> 4)), i0 = p0 - m.start;
        uint16_t* to = region + kv_v_off(p0, d);
        if (i0 >= 0 && i0 + 8 <= n) {
          u32x4_t w;
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = v[j][2 * i] | (uint32_t)v[j][2 * i + 1] << 16;
          *reinterpret_cast<u32x4_t*>(to) = w;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i0 + i >= 0 && i0 + i < n) to[i] = v[j][i];
        }
      }
    }
  }
}

static int check_slab(const char* what, int64_t base, int cap, int heads, int64_t pool_elems) {
  FLYAI_REQUIRE(cap > 0 && cap % 64 == 0 && base >= 0 && base % 8 == 0,
                "%s: a slab needs cap %% 64 == 0 and base %% 8 == 0", what);
  if (base + (int64_t)heads * cap * 64 > pool_elems)
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
    FLYAI_REQUIRE(src_k != dst_k || apart(src), "kv_fork: destination %d overlaps the source", i);
    for (int j = 0; j < i; ++j) FLYAI_REQUIRE(apart(dsts_host[j]), "kv_fork: destinations %d and %d overlap", j, i);
  }
  if (lo == hi) return FLYAI_OK;
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
      FLYAI_REQUIRE(keep[r] >= 0, "kv_compact: move %d keeps position %d", i, keep[r]);
      if ((int64_t)m.start + keep[r] >= m.cap)
        return set_error(FLYAI_ERANGE, "kv_compact: move %d keeps position %d + %d of a slab of %d", i, m.start, keep[r], m.cap);
      FLYAI_REQUIRE(m.n <= kMoveRows || r == 0 || keep[r] > keep[r - 1],
                    "kv_compact: move %d of more than %d rows must keep them in ascending order", i, kMoveRows);
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
  a.pool[0] = k_pool, a.pool[1] = v_pool, a.layer = layer, a.heads = Hkv, a.n_slabs = 0;
  int rows = 0;
  auto flush = [&]() {
    if (a.n_slabs == 0) return FLYAI_OK;
    hipLaunchKernelGGL(kv_compact_kernel, dim3(8 * Hkv, a.n_slabs, n_layers), dim3(kMoveThreads), 0, s, a);
    a.n_slabs = rows = 0;
    return check_launch("kv_compact");
  };
  first = 0;
  for (int i = 0; i < n_moves; ++i) {
    const flyai_kv_move& m = moves_host[i];
    const int32_t* keep = keep_host + first;
    first += m.n;
    int r = 0;
    while (r < m.n && keep[r] == r) ++r;  // rows that stay where they are
    const bool whole = m.n - r <= kMoveRows;
    while (r < m.n) {
      // a move of up to kMoveRows rows in any order goes into one launch whole; a longer one in pieces
      if (a.n_slabs == kMoveSlabs || rows == kMoveRows || (whole && rows + (m.n - r) > kMoveRows)) RUN(flush());
      const int n = std::min(m.n - r, kMoveRows - rows);
      a.slab[a.n_slabs++] = MoveSlab{m.base, m.cap, m.start + r, rows, n, m.start};
      std::copy(keep + r, keep + r + n, a.keep + rows);
      rows += n;
      r += n;
      if (r < m.n) RUN(flush());  // the next piece reads what this one must not have passed yet
    }
  }
  return flush();
}
