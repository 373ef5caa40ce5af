// Attention of a batch whose sequences share prefixes.
//
// A prefix's K/V lies in one slab, what follows it in each sequence's own.  Row (t, h) at position p of a sequence behind a
// prefix of P positions sees the prefix's keys [lo, P) and its own slab's [max(lo - P, 0), p - P], lo = max(0, p - window + 1)
// or 0; the softmax runs over both and the head's sink.  The rows of all the prefix's sequences are taken together, so
// its keys are read once per tile of rows, not once per sequence.
//
// Every key range is cut into chunks whose borders go by the slab alone (from its position 0).  A chunk's
// (m, l, O[64]) starts afresh, and a range's total folds its chunks in ascending order (fold below):
//   M' = max(M, m);  O' = O_c 2^(m - M') + O 2^(M - M');  L likewise.
// A work item takes a run of a range's chunks and leaves a record of each (one, of a run from the range's first chunk on: folded), which
// attn_shared_merge_kernel folds; or it takes the whole range and folds in its registers, by the same operations in the same order.  So the work is split where there are few
// rows and not where there are many, and a row's bits depend on neither, nor on the rest of the batch.
//
// The work lists are made on the GPU (attn_shared_plan_kernel), once for a step's layers: the host needs
// no lengths, only bounds, and the grids are sized by those.
//
// What bounds it: with many rows instruction issue.  A wave's block (32 rows, 64 keys) is 36 matrix instructions (576 clocks of the matrix
// unit) and 32 exponentials, 32 fused multiply-adds, 16 maxima of three and 16 conversions (some 500: 8.6, 2.6 to 4, 4 and 4 each).  A
// product keeps vector instructions from issue for about half of its 16 clocks: a loop of that mixture takes some 860 clocks a
// block, 1,720 for a SIMD's two waves, whose blocks take some 2,150.  256 streams of up to 4 tokens behind 32,749 positions (554 GFLOP) take 578
// to 616 us on different boxes, 0.96 to 0.90 PFLOP/s (a library's large product: 1.43); six questions of up to 300 tokens behind 4,099 (102
// GFLOP) 158 to 164.  With few rows the chain of a unit -- entry, token list, queries (3.5 us), then 1.1 us a block, of which two waves a
// SIMD take as long as one -- and the launches: 48 streams behind 8,000 positions 32 us, of which the plan's 7, the items' 22 and the merge's
// 5; 2 streams behind 513 21 to 23 (6, 7.5 and 3 to 4; the host's two calls are as long).  Three waves a SIMD (168 registers) and three buffers in
// turn were slower than two.
#include <type_traits>

#include "attn.h"

namespace flyai {

constexpr int kShRowTokens = 16;      // tokens of a prefix item's tile (4 waves x 2 tiles of 16 rows x 2 tokens)
constexpr int kShWaveTokens = 2;      // tokens of a wave item
// The most new tokens of a sequence whose own keys go to waves; more go to tiles (32 streams of up to 8 tokens: 80.3 us with 4, 81.9
// with 8, 79.7 with 1, which costs batches of two-token chunks a tile of 16 rows each).
constexpr int kShWaveSeq = 4;
constexpr int kShMaxSeqs = 4096, kShMaxPrefixes = 1024;
// A prefix's chunks: up to 16, or up to 24 where they would have more than 1,152 positions, of 384 positions at least (192 behind up
// to 1,536).  Finer ones give few rows more workgroups, coarser ones leave fewer records.  With 24 throughout, 32 streams' drafts behind
// 16,000 positions take 97 us in place of 90; with 16 throughout, 3 streams behind 32,000 take 41 in place of 33; with 768 at least, 8
// streams behind 4,000 take 24 in place of 20 (and 100 behind 6,000 51 in place of 54).
constexpr int kShChunks = 16, kShMoreChunks = 24, kShMoreFrom = 1152;
constexpr int kShMinChunk = 384, kShChunkStep = 192;
constexpr int kShOwnChunk = 384;  // (192: two to three percent slower with some hundred own positions a stream)
// What is split by chunks has room of its own: entries of workgroups and waves beyond one for each tile and group, and records beyond two
// for each token.  A prefix's tiles are split where they fill less than a round (kShRecCost), so up to some 2 / 3 of kShGrid / Hkv tiles of
// 16 tokens in up to 24 chunks; a sequence's own keys where they make fewer than 8 kShGrid items of up to 4 tokens a wave.  (What does not fit stays whole.)
constexpr int kShSpareEntries = 8192, kShSpareWaves = 4096;
constexpr int kShSplitRecs = 131072, kShOwnRecs = 16384;  // of all kv heads: 277 and 35 MB
constexpr int kShRecCost = 700;       // what a chunk's records cost, in positions
constexpr int kShGrid = 512;           // workgroups on the chip at once: two a CU
// workgroups of a kv head: head g's are those with blockIdx % Hkv == g, with 8 heads an XCD each, so that its L2 holds one head's keys
__host__ __device__ constexpr int sh_per_head(int Hkv) { return kShGrid / Hkv > 0 ? kShGrid / Hkv : 1; }

// A unit of work: `ntok` rows' tokens -- from `first` on in the list of a prefix's tokens (list), or token first + i at the slab's
// position pos0 + i -- and their keys from key_lo on.  stride 0: all the keys up to `end`, folded; otherwise those of key_lo's chunk, and
// the next `left` units are the same rows' next chunks.
struct ShEntry {
  int64_t base;   // of the slab
  int32_t cap;
  int32_t first;
  int32_t ntok;
  int32_t pos0;
  int32_t list;
  int32_t key_lo, end;  // slab positions
  int32_t chunk;        // positions of a chunk
  int32_t rec;          // record of the first token; token i's is rec + i, the next chunk's `stride` behind
  int32_t stride;
  int32_t left;
  int32_t is_first;     // of a split tile's units: its first chunk's.  The chunks that a workgroup takes from there on are folded into one record.
};

struct ShToken {  // where a token's records lie: n of them, stride apart
  int32_t p_rec, p_n, p_stride;
  int32_t p_folded;  // chunks that the prefix's first record holds: the next one is that of chunk p_folded
  int32_t o_rec, o_n, o_stride;
  int32_t pad;
};

// The split units are dealt out in shares of consecutive ones, the first n % per_head of them one larger: the end of the share that holds
// unit u.
__device__ __forceinline__ int sh_share_end(int n, int per_head, int u) {
  const int share = n / per_head, more = n % per_head;
  const int w = u < more * (share + 1) ? u / (share + 1) : more + (u - more * (share + 1)) / max(share, 1);
  return (w + 1) * share + min(w + 1, more);
}

// The units of workgroups: whole prefix tiles, then chunks of prefix tiles, then the sequences' own tiles; and those of waves.
struct ShHeader {
  int32_t n_whole, n_split, n_own, status;
  int32_t n_waves, n_tokens, window;
  int32_t T, S, n_prefix, Hkv;  // what the plan was made for
  int32_t pad[5];
};

// Byte layout of a plan, and how much each list holds at most.
struct ShLayout {
  int32_t T, S, n_prefix, max_entries, max_waves, max_recs;
  size_t o_entries, o_waves, o_list, o_tokens, bytes;
};

__host__ __device__ inline ShLayout sh_layout(int T, int S, int n_prefix, int Hkv) {
  auto least = [](int a, int b) { return a < b ? a : b; };
  ShLayout l;
  l.T = T;
  l.S = S;
  l.n_prefix = n_prefix;
  // the prefixes' tiles, those of the sequences with more than kShWaveSeq tokens
  l.max_entries = 2 * (T / kShRowTokens) + (n_prefix < T ? n_prefix : T) + T / (kShWaveSeq + 1) + least(1024 + 2 * T, kShSpareEntries);
  // the other sequences' groups, and the prefixes whose few tokens go to waves
  l.max_waves = T / kShWaveTokens + (S < T ? S : T) + (n_prefix < T ? n_prefix : T) + kShSpareWaves;
  l.max_recs = 2 * T + least(kShMoreChunks * T, kShSplitRecs / Hkv) + least(256 * T, kShOwnRecs / Hkv);
  size_t o = sizeof(ShHeader);
  l.o_entries = o;
  o += (size_t)l.max_entries * sizeof(ShEntry);
  l.o_waves = o;
  o += (size_t)l.max_waves * sizeof(ShEntry);
  l.o_list = o;
  o += (size_t)T * 8;
  l.o_tokens = o;
  o += (size_t)T * sizeof(ShToken);
  l.bytes = (o + 255) & ~(size_t)255;
  return l;
}

// a plan of another shape has its lists elsewhere: nothing is done with it
__device__ __forceinline__ bool sh_plan_fits(const ShHeader* h, const ShLayout& L, int Hkv) {
  return h->T == L.T && h->S == L.S && h->n_prefix == L.n_prefix && h->Hkv == Hkv;
}

// ---- the plan -------------------------------------------------------------------------------------


// inclusive sum over the wave's lanes, by DPP (no LDS round trips): within rows of 16, then across them
__device__ __forceinline__ int sh_wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, true);  // row_bcast:15 to rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, true);  // row_bcast:31 to rows 2 and 3
  return v;
}

// N exclusive sums over the workgroup at once; total gets the sums
template <int NT, int N>
__device__ __forceinline__ void sh_excl_scan(int (&v)[N], int (&total)[N], int (&red)[6][NT / 64]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int incl[N];
#pragma unroll
  for (int i = 0; i < N; ++i) incl[i] = sh_wave_scan(v[i]);
  __syncthreads();  // the last use of red is over
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (lane == 63) red[i][wave] = incl[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int sums = sh_wave_scan(lane < NT / 64 ? red[i][lane] : 0);
    total[i] = __builtin_amdgcn_readlane(sums, NT / 64 - 1);
    v[i] = incl[i] - v[i] + (wave ? __builtin_amdgcn_readlane(sums, max(wave, 1) - 1) : 0);
  }
}

__device__ __forceinline__ int sh_prefix_chunk(int P) {
  auto part = [&](int n) { return ((P + n - 1) / n + kShChunkStep - 1) / kShChunkStep * kShChunkStep; };
  const int few = part(kShChunks), more = part(kShMoreChunks), c = max(min(few, kShMoreFrom), more);
  const int least = P <= 8 * kShChunkStep ? kShChunkStep : kShMinChunk;
  return c > least ? c : least;
}

struct ShBatch {
  const int32_t *q_lens, *starts;
  const int64_t* kv_base;
  const int32_t *kv_cap, *prefix_of, *prefix_len;
  const int64_t* prefix_base;
  const int32_t* prefix_cap;
  int S, n_prefix, Hkv, window, T;
  int64_t pool_elems;
};

// Bits of the status word
enum { kShPastSlab = 1, kShPastTokens = 2, kShBeforePrefix = 4, kShBadPrefix = 8, kShBadSequence = 16 };

__device__ __forceinline__ bool sh_slab_ok(int64_t base, int cap, int Hkv, int64_t pool) {
  return cap > 0 && cap <= kShMaxCap && cap % 64 == 0 && base >= 0 && base % 8 == 0 && base <= pool - (int64_t)Hkv * cap * 64;
}

// What the plan keeps of a sequence and of a prefix, in LDS.
template <int MAX>
struct ShSeqs {
  int32_t cu[MAX + 1];  // its first token
  int32_t own0[MAX];    // the slab position of its first token; -1: the sequence has no tokens, or is refused
  int32_t prefix[MAX];  // -1: none
  int32_t place[MAX];   // its first listed token's place among its prefix's
  int32_t entry0[MAX], rec0[MAX];  // its first entry (of its kind) and record
};
template <int MAX>
struct ShPrefixes {
  int32_t len[MAX];  // -1: refused
  int32_t cap[MAX];
  int64_t base[MAX];
  int32_t count[MAX];  // listed tokens
  int32_t lo[MAX];     // the first position that any of them sees
  int32_t list0[MAX];
  int32_t tile0[MAX];  // its first tile, of all prefixes' (wave entry, for a prefix of few tokens)
  int32_t unit0[MAX], rec0[MAX];  // of its tiles that are split: the first unit and record
};
constexpr int kShMaxOwnChunks = 4096;  // of a sequence, for the counts to stay in 32 bits: past it no sequence is split

// Made by one workgroup, so that nothing but LDS lies between the counts and the lists: one round trip for the lengths, three sums over the
// workgroup, the lists.  A prefix's tokens are listed in the order in which its sequences' counts arrive at an LDS counter: which rows
// share a tile may change from launch to launch, a row's result does not (no row's steps depend on its tile mates).
// Small batches have a workgroup of their own size, with fewer waves at each barrier and half the code to fetch: 5.8 us in place of 7.5
// with 2 sequences; 256 sequences of 1,000 tokens take the large one, 9.3.
template <int NT, int PER>
__global__ __launch_bounds__(NT) void attn_shared_plan_kernel(ShBatch b, char* __restrict__ plan) {
  const ShLayout L = sh_layout(b.T, b.S, b.n_prefix, b.Hkv);
  ShHeader* hdr = reinterpret_cast<ShHeader*>(plan);
  ShEntry* entries = reinterpret_cast<ShEntry*>(plan + L.o_entries);
  ShEntry* waves = reinterpret_cast<ShEntry*>(plan + L.o_waves);
  int2* list = reinterpret_cast<int2*>(plan + L.o_list);
  ShToken* tokens = reinterpret_cast<ShToken*>(plan + L.o_tokens);
  __shared__ ShSeqs<NT * PER> sq;
  __shared__ ShPrefixes<NT> px;
  __shared__ int red[6][NT / 64];
  __shared__ int status_s;
  const int tid = threadIdx.x;
  const int per = (b.S + NT - 1) / NT;
  const int s0 = tid * per;
  int32_t status = 0;
  // everything that the batch is described by, in one round trip
  int q[PER], start[PER], prefix[PER], cap[PER];
  int64_t base[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const bool there = i < per && s0 + i < b.S;
    const int s = there ? s0 + i : 0;
    q[i] = start[i] = cap[i] = 0;
    prefix[i] = -1;
    base[i] = 0;
    if (there) {
      q[i] = b.q_lens[s];
      start[i] = b.starts[s];
      prefix[i] = b.prefix_of[s];
      cap[i] = b.kv_cap[s];
      base[i] = b.kv_base[s];
    }
  }
  if (tid < b.n_prefix) {  // (at most one a thread)
    const int len = b.prefix_len[tid], c = b.prefix_cap[tid];
    const int64_t pb = b.prefix_base[tid];
    px.len[tid] = len >= 0 && len <= c && sh_slab_ok(pb, c, b.Hkv, b.pool_elems) ? len : -1;
    px.cap[tid] = c;
    px.base[tid] = pb;
    px.count[tid] = 0;
    px.lo[tid] = INT32_MAX;
  }
  if (tid == 0) status_s = 0;
  int sum[1] = {0}, total[1];
#pragma unroll
  for (int i = 0; i < PER; ++i) sum[0] += min(max(q[i], 0), b.T + 1);  // (what is past T is refused: no sum passes 2^31)
  sh_excl_scan<NT, 1>(sum, total, red);
  const int n_tokens = min(total[0], b.T);
  if (total[0] > b.T) status |= kShPastTokens;

  // the tokens of a sequence that see its prefix: the first of them, those below P + window - 1
  auto listed = [&](int n, int own0, int p) __attribute__((always_inline)) {
    if (p < 0 || px.len[p] == 0) return 0;
    return b.window > 0 ? (int)min((int64_t)n, max((int64_t)0, (int64_t)b.window - 1 - own0)) : n;
  };
  // the first chunk and the number of chunks of its own keys
  auto own_chunks = [&](int n, int own0, int* c0) __attribute__((always_inline)) {
    *c0 = b.window > 0 ? max(0, own0 - b.window + 1) / kShOwnChunk : 0;
    return (own0 + n - 1) / kShOwnChunk + 1 - *c0;
  };
  auto groups_of = [](int n) { return n <= kShWaveSeq ? (n + kShWaveTokens - 1) / kShWaveTokens : (n + kShRowTokens - 1) / kShRowTokens; };

  int own[PER];
  // the groups of tokens that go to waves and to tiles, their entries and the records if they are split by chunks; whether a sequence
  // is too long for that
  int seqs[6] = {0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    own[i] = -1;
    const int s = s0 + i;
    if (i >= per || s >= b.S) continue;
    const int first = sum[0];
    sum[0] += min(max(q[i], 0), b.T + 1);
    int st = 0, o = -1;
    if (q[i] < 0 || start[i] < 0) {
      st = kShBadSequence;
    } else if (q[i] > 0 && (int64_t)first + q[i] <= b.T) {
      const int p = prefix[i];
      const int P = p < 0 ? 0 : p < b.n_prefix ? px.len[p] : -1;
      if (P < 0) st = kShBadPrefix;
      else if (start[i] < P) st = kShBeforePrefix;
      else if (!sh_slab_ok(base[i], cap[i], b.Hkv, b.pool_elems)) st = kShBadSequence;
      else if ((int64_t)start[i] - P + q[i] > cap[i]) st = kShPastSlab;
      else o = start[i] - P;
    }
    status |= st;
    own[i] = o;
    sq.cu[s] = min(first, b.T);
    if (s == b.S - 1) sq.cu[b.S] = n_tokens;
    sq.own0[s] = o;
    sq.prefix[s] = prefix[i] < 0 ? -1 : prefix[i];
    if (o < 0) continue;
    const int n = listed(q[i], o, prefix[i]);
    if (n > 0) {
      sq.place[s] = atomicAdd(&px.count[prefix[i]], n);
      atomicMin(&px.lo[prefix[i]], b.window > 0 ? max(0, start[i] - b.window + 1) : 0);
    }
    int c0;
    const int nch = own_chunks(q[i], o, &c0);
    const int kind = q[i] > kShWaveSeq;
    seqs[kind] += groups_of(q[i]);
    seqs[2 + kind] += groups_of(q[i]) * min(nch, kShMaxOwnChunks);
    seqs[4] += q[i] * min(nch, kShMaxOwnChunks);
    seqs[5] += nch > kShMaxOwnChunks;
  }
  if (status) atomicOr(&status_s, status);
  int n_seqs[6];
  sh_excl_scan<NT, 6>(seqs, n_seqs, red);  // (its barriers also end the counting)

  // the prefixes: a thread has one
  const int np = tid < b.n_prefix ? px.count[tid] : 0;
  const bool few = np <= kShWaveTokens;
  int P = 0, C = 64, chunk0 = 0, chunks = 0, tiles = 0;
  if (np > 0) {
    P = px.len[tid];
    C = sh_prefix_chunk(P);
    chunk0 = px.lo[tid] / C;
    chunks = (P - 1) / C + 1 - chunk0;
    tiles = few ? 1 : (np + kShRowTokens - 1) / kShRowTokens;
  }
  // listed tokens; tiles of workgroups; entries of waves whole and by chunks, their records by chunks
  int ps[6] = {np, few ? 0 : tiles, few ? tiles : 0, few ? tiles * chunks : 0, few ? np * chunks : 0, few ? 0 : tiles * min(C, 4096)}, n_ps[6];
  sh_excl_scan<NT, 6>(ps, n_ps, red);
  // As many whole tiles as give every workgroup the same number; the rest by chunks, if the lists and the records hold them.  A chunk of C
  // positions costs what C + kShRecCost would without its records; of a rest that is the part r of a round some 0.7 r of the chunks are
  // in their tile's first record.  So the rest stays whole where its chunks would take longer than a round that not all workgroups
  // have a tile in.  With 43 and 93 tiles of 4,099 positions (64 workgroups) whole and by chunks 106 and 116, 164 and 172 us; with 23 and 84
  // 77 and 70, 165 and 156; with 35 of 9,000 175 and 143.
  const int per_head = sh_per_head(b.Hkv);
  int whole = n_ps[1] / per_head * per_head;
  const int64_t rest = n_ps[1] - whole, part = 10 * per_head - 7 * rest;  // 10 per_head (1 - 0.7 r)
  if (rest * (10 * per_head * (int64_t)n_ps[5] + kShRecCost * part * n_ps[1]) > 10 * (int64_t)per_head * per_head * n_ps[5]) whole = n_ps[1];
  auto split_of = [&](int w) __attribute__((always_inline)) { return few ? 0 : max(0, ps[1] + tiles - max(ps[1], w)); };
  int split = split_of(whole), split_tokens = np > 0 ? min(np, np - (tiles - split) * kShRowTokens) : 0;
  if (!split) split_tokens = 0;
  int us[2] = {split * chunks, split_tokens * chunks}, n_us[2];
  sh_excl_scan<NT, 2>(us, n_us, red);
  const bool fsplit = n_ps[3] + n_seqs[0] <= L.max_waves && n_ps[0] + n_ps[4] + b.T <= L.max_recs;
  const int few_recs = fsplit ? n_ps[4] : 0, few_waves = fsplit ? n_ps[3] : n_ps[2];
  if (whole + n_us[0] + n_seqs[1] > L.max_entries || n_ps[0] + few_recs + n_us[1] + b.T > L.max_recs) {  // (uniform)
    whole = n_ps[1];
    split = split_tokens = us[0] = us[1] = n_us[0] = n_us[1] = 0;
  }
  // records: one for each listed token, then those of the chunks, then the sequences' own
  const int ptiles = whole + n_us[0], precs = n_ps[0] + few_recs + n_us[1];
  const bool osplit = n_seqs[5] == 0 && ((int64_t)n_seqs[2] + 4 * n_seqs[3]) * b.Hkv < 8 * kShGrid &&
                      few_waves + n_seqs[2] <= L.max_waves && ptiles + n_seqs[3] <= L.max_entries && precs + n_seqs[4] <= L.max_recs;
  if (np > 0) {
    px.list0[tid] = ps[0];
    px.tile0[tid] = few ? (fsplit ? ps[3] : ps[2]) : ps[1];
    px.unit0[tid] = us[0];
    px.rec0[tid] = n_ps[0] + (few ? ps[4] : few_recs + us[1]);
  }
  // the sequences' entries and records: as scanned if they are split, else by groups and tokens
  int at[3] = {seqs[2], seqs[3], seqs[4]};
  if (!osplit) {
    int all[3];
    at[0] = seqs[0];
    at[1] = seqs[1];
    at[2] = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (own[i] >= 0) at[2] += q[i];
    int tokens_at[1] = {at[2]};
    sh_excl_scan<NT, 1>(tokens_at, reinterpret_cast<int (&)[1]>(all), red);
    at[2] = tokens_at[0];
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (own[i] < 0) continue;
    int c0;
    const int nch = osplit ? own_chunks(q[i], own[i], &c0) : 1, kind = q[i] > kShWaveSeq;
    sq.entry0[s0 + i] = kind ? ptiles + at[1] : few_waves + at[0];
    sq.rec0[s0 + i] = precs + at[2];
    (kind ? at[1] : at[0]) += groups_of(q[i]) * nch;
    at[2] += q[i] * nch;
  }
  if (tid == 0) {
    hdr->n_whole = whole;
    hdr->n_split = n_us[0];
    hdr->n_own = osplit ? n_seqs[3] : n_seqs[1];
    hdr->n_waves = few_waves + (osplit ? n_seqs[2] : n_seqs[0]);
    hdr->n_tokens = n_tokens;
    hdr->window = b.window;
    hdr->T = b.T;
    hdr->S = b.S;
    hdr->n_prefix = b.n_prefix;
    hdr->Hkv = b.Hkv;
  }
  __syncthreads();
  if (tid == 0) hdr->status = status_s;
  // a prefix's units: tiles, or a tile's chunks behind one another
  auto first_split = [&](int p) __attribute__((always_inline)) { return max(0, whole - px.tile0[p]); };  // its first tile that is split
  for (int p = tid >> 6; p < b.n_prefix; p += NT / 64) {
    const int n = px.count[p];
    if (!n) continue;
    const int len = px.len[p], c = sh_prefix_chunk(len), lo = px.lo[p], c0 = lo / c, nch = (len - 1) / c + 1 - c0;
    const bool w = n <= kShWaveTokens;
    const int nt = w ? 1 : (n + kShRowTokens - 1) / kShRowTokens, ts = w ? (fsplit ? 0 : 1) : min(nt, first_split(p));
    for (int i = tid & 63; i < ts + (nt - ts) * nch; i += 64) {
      const bool one = i < ts;  // whole
      const int t = one ? i : ts + (i - ts) / nch, k = one ? 0 : (i - ts) % nch;
      ShEntry e;
      e.base = px.base[p];
      e.cap = px.cap[p];
      e.first = px.list0[p] + t * kShRowTokens;
      e.ntok = min(kShRowTokens, n - t * kShRowTokens);
      e.pos0 = 0;
      e.list = 1;
      e.key_lo = max(lo, (c0 + k) * c);
      e.end = len;
      e.chunk = c;
      e.stride = one ? 0 : n - ts * kShRowTokens;
      e.rec = one ? e.first : px.rec0[p] + k * e.stride + (t - ts) * kShRowTokens;
      e.left = one ? 0 : nch - 1 - k;
      e.is_first = !one && k == 0;
      ShEntry* out = w ? waves + px.tile0[p] : one ? entries + px.tile0[p] : entries + whole + px.unit0[p] - ts;
      out[i] = e;
    }
  }
  for (int t = tid; t < n_tokens; t += NT) {
    int lo = 0, hi = b.S - 1;  // last sequence with cu <= t
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (sq.cu[mid] <= t) lo = mid; else hi = mid - 1;
    }
    ShToken k = {};
    const int own0 = sq.own0[lo], i = t - sq.cu[lo];
    if (own0 >= 0) {
      const int n = sq.cu[lo + 1] - sq.cu[lo], p = sq.prefix[lo];
      int c0;
      const int all = own_chunks(n, own0, &c0), nch = osplit ? all : 1;
      k.o_rec = sq.rec0[lo] + i;
      k.o_n = nch;
      k.o_stride = n;
      if (i < listed(n, own0, p)) {
        const int len = px.len[p], c = sh_prefix_chunk(len), where = sq.place[lo] + i, count = px.count[p];
        const bool w = count <= kShWaveTokens;
        const int ts = w ? (fsplit ? 0 : 1) : first_split(p);
        list[px.list0[p] + where] = make_int2(t, len + own0 + i);
        k.p_n = k.p_folded = 1;
        k.p_rec = px.list0[p] + where;
        if (where >= ts * kShRowTokens) {
          k.p_n = (len - 1) / c + 1 - px.lo[p] / c;
          k.p_stride = count - ts * kShRowTokens;
          k.p_rec = px.rec0[p] + where - ts * kShRowTokens;
          if (!w) {
            const int u = px.unit0[p] + (where / kShRowTokens - ts) * k.p_n;
            k.p_folded = min(k.p_n, sh_share_end(n_us[0], per_head, u) - u);
          }
        }
      }
      const int size = n <= kShWaveSeq ? kShWaveTokens : kShRowTokens;
      if (i % size == 0) {  // its group's entries
        const int64_t kv = b.kv_base[lo];
        const int kc = b.kv_cap[lo];
        for (int c = 0; c < nch; ++c) {
          ShEntry e;
          e.base = kv;
          e.cap = kc;
          e.first = t;
          e.ntok = min(size, n - i);
          e.pos0 = own0 + i;
          e.list = 0;
          const int klo = b.window > 0 ? max(0, e.pos0 - b.window + 1) : 0;
          e.key_lo = osplit ? max(klo, (c0 + c) * kShOwnChunk) : klo;
          e.end = osplit ? min(e.pos0 + e.ntok, (c0 + c + 1) * kShOwnChunk) : e.pos0 + e.ntok;  // (a chunk before the window is empty)
          e.chunk = kShOwnChunk;
          e.rec = sq.rec0[lo] + c * n + i;
          e.stride = osplit ? n : 0;
          e.left = 0;
          e.is_first = 0;
          (n <= kShWaveSeq ? waves : entries)[sq.entry0[lo] + (i / size) * nch + c] = e;
        }
      }
    }
    tokens[t] = k;
  }
}

// ---- the items ------------------------------------------------------------------------------------

// QT tiles of 16 query rows of a wave (row rq = 16 qt + n is token rq / 8, head rq % 8 of the group): the Q^T operand, the slab
// positions that a row sees, the chunk's running softmax (S^T and O^T as in attn.hip) and the range's total.
template <int QT>
struct ShRows {
  bf16x8_t qf[QT][2];
  int lo[QT], hi[QT];
  bool val[QT];
  float m[QT], tm[QT], tL[QT];
  f32x4_t O[QT][4], L[QT], tO[QT][4];  // (every element of L is the row's sum)
};

template <int QT>
__device__ __forceinline__ void sh_nothing(ShRows<QT>& R) {
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    R.tm[qt] = -1e30f;
    R.tL[qt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) R.tO[qt][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
}

template <int QT>
__device__ __forceinline__ void sh_fresh(ShRows<QT>& R) {
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    R.m[qt] = -1e30f;
    R.L[qt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) R.O[qt][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
}

// The fold of (m, l, O) into the total (M, L, O): the same operations in the items and in the merge.
struct ShFold {
  float M, a, c;  // the new maximum, what the total and the chunk are multiplied with
};
__device__ __forceinline__ ShFold sh_fold(float M, float m) {
  const float x = M > m ? M : m;
  return {x, __builtin_amdgcn_exp2f(M - x), __builtin_amdgcn_exp2f(m - x)};
}

template <int QT>
__device__ __forceinline__ void sh_fold_chunk(ShRows<QT>& R) {
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const ShFold f = sh_fold(R.tm[qt], R.m[qt]);
    R.tm[qt] = f.M;
    R.tL[qt] = fmaf(R.L[qt][0], f.c, R.tL[qt] * f.a);
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int v = 0; v < 4; ++v) R.tO[qt][dt][v] = fmaf(R.O[qt][dt][v], f.c, R.tO[qt][dt][v] * f.a);
  }
}

// rows of the entry's tokens tok0 .. : in the prefix's list, or behind one another
template <int QT>
__device__ __forceinline__ void sh_rows_init(ShRows<QT>& R, const ShEntry& e, int tok0, const int2* __restrict__ list,
                                             const uint16_t* __restrict__ q, int kv_head, int Hq, int window) {
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int rq = 16 * qt + n, ti = tok0 + (rq >> 3);
    R.val[qt] = ti < e.ntok;
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
    R.lo[qt] = 0;
    R.hi[qt] = INT32_MAX;  // a row that is none sees all (its scores are 0, nothing of it is written)
    if (R.val[qt]) {
      int2 tp = make_int2(e.first + ti, e.pos0 + ti);
      if (e.list) tp = list[e.first + ti];
      R.hi[qt] = tp.y;
      R.lo[qt] = window > 0 ? max(0, tp.y - window + 1) : 0;
      const uint16_t* qp = q + ((size_t)tp.x * Hq + kv_head * 8 + (rq & 7)) * 64 + 8 * g;
      a = *reinterpret_cast<const uint4*>(qp);
      b = *reinterpret_cast<const uint4*>(qp + 32);
    }
    R.qf[qt][0] = as_bf16x8(a);
    R.qf[qt][1] = as_bf16x8(b);
  }
  sh_nothing(R);
  sh_fresh(R);
}

// the keys that every row of the wave sees: [*lo, *hi]
template <int QT>
__device__ __forceinline__ void sh_interior(const ShRows<QT>& R, int* lo, int* hi) {
  int a = 0, b = INT32_MAX;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    a = max(a, R.lo[qt]);
    b = min(b, R.hi[qt]);
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    a = max(a, __shfl_xor(a, o, 64));
    b = min(b, __shfl_xor(b, o, 64));
  }
  *lo = scalar(a);
  *hi = scalar(b);
}

// Where a block has keys that some row does not see, their values may be infinite or NaN, and P is 0 there: 0 x inf would be NaN.
// Such values are left out of v (all of a block's fragments), and rows that see one get it by what the products of P with the
// classes' indicators say.  (A loop over the classes: the code is rarely run, and long.)
template <int QT>
__device__ __forceinline__ void sh_wild_values(ShRows<QT>& R, uint4 (&v)[4][2], const bf16x8_t (&pt)[QT][2]) {
#pragma unroll 1
  for (uint32_t kind = 0; kind < 3; ++kind) {  // +inf, -inf, NaN
    const uint32_t lo = kind == 0 ? 0x7f80u : kind == 1 ? 0xff80u : 0x7f81u, span = kind == 2 ? 0x7eu : 0u, mask = kind == 2 ? 0x7fffu : 0xffffu;
    const float add = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : NAN;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) {
      bf16x8_t f[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t w[4] = {v[dt][h].x, v[dt][h].y, v[dt][h].z, v[dt][h].w};
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          o[i] = ((w[i] & mask) - lo <= span ? 0x3f80u : 0u) | (((w[i] >> 16) & mask) - lo <= span ? 0x3f800000u : 0u);
        f[h] = as_bf16x8(make_uint4(o[0], o[1], o[2], o[3]));
      }
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        f32x4_t c = mfma16x16x32(f[0], pt[qt][0], f32x4_t{0.f, 0.f, 0.f, 0.f});
        c = mfma16x16x32(f[1], pt[qt][1], c);
#pragma unroll
        for (int i = 0; i < 4; ++i) R.O[qt][dt][i] += c[i] > 0.f ? add : 0.f;
      }
    }
  }
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t w[4] = {v[dt][h].x, v[dt][h].y, v[dt][h].z, v[dt][h].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if ((w[i] & 0x7f80u) == 0x7f80u) w[i] &= 0xffff0000u;
        if ((w[i] & 0x7f800000u) == 0x7f800000u) w[i] &= 0xffffu;
      }
      v[dt][h] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// One 64-key block against the wave's rows.  k(kt, step) and v(dt, half) give its fragments, from registers.  As in attn.hip: scores
// S^T = K . Q^T, P = 2^(s scale - m) rounded to bf16 (2^-8 of each at most: the matrix units take 16 bits; the row sum takes the rounded
// values), O^T += V^T . P^T, L += 1 . P^T.  One row tile's scores are live at a time.
template <int QT, class KF, class VF, class AF>
__device__ __forceinline__ void sh_block(ShRows<QT>& R, KF&& k, VF&& v, AF&& after_scores, int kb, bool interior, int key_lo, int key_hi) {
  const int g = (threadIdx.x & 63) >> 4;
  const float scale = 0.125f * kLog2e;
  const bf16x8_t ones = as_bf16x8(make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u));
  bf16x8_t pt[QT][2];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    f32x4_t s[4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      s[kt] = mfma16x16x32(as_bf16x8(k(kt, 0)), R.qf[qt][0], f32x4_t{0.f, 0.f, 0.f, 0.f});
      s[kt] = mfma16x16x32(as_bf16x8(k(kt, 1)), R.qf[qt][1], s[kt]);
    }
    if (qt == QT - 1) after_scores();
    float bmax = -INFINITY;
    if (!interior) {
      // (tile_key(kt, 4 g + i) is 8 g + tile_key(kt, i); a row that sees nothing has a count of 0)
      const int lo = max(key_lo, R.lo[qt]), from = kb + 8 * g - lo;
      const uint32_t count = (uint32_t)max(min(key_hi - 1, R.hi[qt]) - lo + 1, 0);
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[kt][i] = (uint32_t)(from + tile_key(kt, i)) < count ? s[kt][i] : -INFINITY;
    }
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) bmax = fmaxf(bmax, s[kt][i]);
    // (a row's largest score lies in one of its four lanes: they are compared only where one of the wave's lanes is past its row's slack)
    if (__ballot(bmax * scale > R.m[qt] + kMaxSlack)) {
      const float m_blk = max_lane_groups(bmax) * scale;
      const bool move = m_blk > R.m[qt] + kMaxSlack;
      const float m_new = move ? m_blk : R.m[qt];
      const float alpha = __builtin_amdgcn_exp2f(R.m[qt] - m_new);
      R.m[qt] = m_new;
      R.L[qt] *= alpha;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) R.O[qt][dt] *= alpha;
    }
    const float neg_m = -R.m[qt];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) pt[qt][kt >> 1][(kt & 1) * 4 + i] = (__bf16)__builtin_amdgcn_exp2f(fmaf(s[kt][i], scale, neg_m));
    R.L[qt] = mfma16x16x32(ones, pt[qt][0], R.L[qt]);
    R.L[qt] = mfma16x16x32(ones, pt[qt][1], R.L[qt]);
  }
  if (!interior) {
    uint4 w[4][2];
    uint32_t wild = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // keys outside the item's range may never have been written
      const uint4 all = make_uint4(~0u, ~0u, ~0u, ~0u), there = mask_keys(all, kb + 32 * h + 8 * g, key_lo, key_hi);
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) {
        uint4 x = v(dt, h);
        x = make_uint4(x.x & there.x, x.y & there.y, x.z & there.z, x.w & there.w);
        w[dt][h] = x;
        // (the sum's top bit of a half is set where its exponent is all ones)
        wild |= ((x.x & 0x7fff7fffu) + 0x00800080u) | ((x.y & 0x7fff7fffu) + 0x00800080u) | ((x.z & 0x7fff7fffu) + 0x00800080u) |
                ((x.w & 0x7fff7fffu) + 0x00800080u);
      }
    }
    if (__ballot((wild & 0x80008000u) != 0)) sh_wild_values(R, w, pt);
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        R.O[qt][dt] = mfma16x16x32(as_bf16x8(w[dt][0]), pt[qt][0], R.O[qt][dt]);
        R.O[qt][dt] = mfma16x16x32(as_bf16x8(w[dt][1]), pt[qt][1], R.O[qt][dt]);
      }
    return;
  }
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) {
    const uint4 v0 = v(dt, 0), v1 = v(dt, 1);
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      R.O[qt][dt] = mfma16x16x32(as_bf16x8(v0), pt[qt][0], R.O[qt][dt]);
      R.O[qt][dt] = mfma16x16x32(as_bf16x8(v1), pt[qt][1], R.O[qt][dt]);
    }
  }
}

// The same for a block that every row sees whole and that moves no row's maximum: straight-line code, so that the accumulators stay
// where they are.  (A rescale's branch, or a branch around the block, costs 40 register copies a block: the two ways' accumulators
// meet in other registers.)  false: some row's maximum has to move, and nothing was done.
// FIRST: the rows' state is a fresh one, and the maximum is set (nothing is there that would have to be rescaled).
template <bool FIRST, class KF, class VF>
__device__ __forceinline__ bool sh_fast_block(ShRows<2>& R, KF&& k, VF&& v) {
  constexpr int QT = 2;
  const float scale = 0.125f * kLog2e;
  const bf16x8_t ones = as_bf16x8(make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u));
  // (K's fragments are read at once, V's first half before the maxima, its second before its products: read where they are used,
  // each is a wait for LDS)
  bf16x8_t kf[4][2], vf[4];
#pragma unroll
  for (int kt = 0; kt < 4; ++kt)
#pragma unroll
    for (int st = 0; st < 2; ++st) kf[kt][st] = as_bf16x8(k(kt, st));
  __builtin_amdgcn_sched_barrier(0);
  f32x4_t s[QT][4];
#pragma unroll
  for (int st = 0; st < 2; ++st)
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) s[qt][kt] = mfma16x16x32(kf[kt][st], R.qf[qt][st], st ? s[qt][kt] : f32x4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) vf[dt] = as_bf16x8(v(dt, 0));
  __builtin_amdgcn_sched_barrier(0);
  bool past = false;  // (sh_block's rule)
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    float bmax = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) bmax = fmaxf(bmax, s[qt][kt][i]);
    if (FIRST) {
      const float m_blk = max_lane_groups(bmax) * scale;
      R.m[qt] = m_blk > R.m[qt] + kMaxSlack ? m_blk : R.m[qt];
    } else {
      past |= bmax * scale > R.m[qt] + kMaxSlack;
    }
  }
  // (the wave with the exponentials goes first: the SIMD's other wave has its matrix products to fill with)
  __builtin_amdgcn_s_setprio(1);
  bf16x8_t pt[QT][2];
  auto weight = [&](int qt, int kt, int i) __attribute__((always_inline)) {
    pt[qt][kt >> 1][(kt & 1) * 4 + i] = (__bf16)__builtin_amdgcn_exp2f(fmaf(s[qt][kt][i], scale, -R.m[qt]));
  };
  // the weights of the first 32 keys; those of the others between their products, which a wave's own matrix units run beside them.
  // (The branch comes behind the first weights: they do not wait for the maxima.)
#pragma unroll
  for (int kt = 0; kt < 2; ++kt)
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int i = 0; i < 4; ++i) weight(qt, kt, i);
  if (!FIRST && __ballot(past)) {
    __builtin_amdgcn_s_setprio(0);
    return false;
  }
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) R.L[qt] = mfma16x16x32(ones, pt[qt][0], FIRST ? f32x4_t{0.f, 0.f, 0.f, 0.f} : R.L[qt]);
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      R.O[qt][dt] = mfma16x16x32(vf[dt], pt[qt][0], FIRST ? f32x4_t{0.f, 0.f, 0.f, 0.f} : R.O[qt][dt]);
#pragma unroll
      for (int i = 0; i < 2; ++i) weight(dt & 1, 2 + (dt >> 1), 2 * qt + i);
    }
  }
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) vf[dt] = as_bf16x8(v(dt, 1));
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_setprio(0);
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) R.L[qt] = mfma16x16x32(ones, pt[qt][1], R.L[qt]);
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) R.O[qt][dt] = mfma16x16x32(vf[dt], pt[qt][1], R.O[qt][dt]);
  return true;
}

// A record: O[64] of (record, kv head, head of the group), and apart from it (m, l).
__device__ __forceinline__ float* sh_rec_o(float* parts, int rec, int Hkv, int g, int h) {
  return parts + (((size_t)rec * Hkv + g) * 8 + h) * 64;
}
__device__ __forceinline__ float* sh_rec_ml(float* parts, int max_recs, int rec, int Hkv, int g, int h) {
  return parts + (size_t)max_recs * Hkv * 512 + (((size_t)rec * Hkv + g) * 8 + h) * 2;
}

// the end of the keys of `run` units from e on
__device__ __forceinline__ int sh_key_end(const ShEntry& e, int run) {
  return e.stride ? (int)min((int64_t)e.end, ((int64_t)(e.key_lo / e.chunk) + run) * e.chunk) : e.end;
}

// The last chunk folded in, and the total to the item's records.
template <int QT>
__device__ __forceinline__ void sh_put(ShRows<QT>& R, int rec0, int tok0, int kv_head, int Hkv, int max_recs, float* __restrict__ parts) {
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  sh_fold_chunk(R);
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    if (!R.val[qt]) continue;
    const int rq = 16 * qt + n, rec = rec0 + tok0 + (rq >> 3);
    float* o = sh_rec_o(parts, rec, Hkv, kv_head, rq & 7) + 4 * g;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) *reinterpret_cast<f32x4_t*>(o + 16 * dt) = R.tO[qt][dt];
    if (g == 0) *reinterpret_cast<float2*>(sh_rec_ml(parts, max_recs, rec, Hkv, kv_head, rq & 7)) = make_float2(R.tm[qt], R.tL[qt]);
  }
}

// An item of up to 2 tokens by one wave, K and V straight from the slab.
__device__ __forceinline__ void sh_wave_item(const ShEntry& e, int kv_head, const int2* __restrict__ list, const uint16_t* __restrict__ q,
                                             const uint16_t* __restrict__ k_pool, const uint16_t* __restrict__ v_pool, int Hq, int Hkv,
                                             int window, int max_recs, float* __restrict__ parts) {
  const int lane = threadIdx.x & 63;
  const int key_hi = sh_key_end(e, 1);
  const int64_t base = e.base + (int64_t)kv_head * e.cap * 64;
  const uint16_t *K = k_pool + base, *V = v_pool + base;
  ShRows<1> R;
  sh_rows_init(R, e, 0, list, q, kv_head, Hq, window);
  int int_lo, int_hi;
  sh_interior(R, &int_lo, &int_hi);
  int_lo = max(int_lo, e.key_lo);
  int_hi = min(int_hi, key_hi - 1);
  // K and V of the next block are loaded while this one computes, K into the same registers once the scores are made
  uint4 kc[4][2], vc[4][2], vn[4][2];
  int kb = e.key_lo & ~63;
  if (kb < key_hi) {
    load_k_tile(kc, K, kb, lane);
    load_v_tile(vn, V, kb, lane);
  }
  int next_fold = (kb / e.chunk + 1) * e.chunk;
  for (; kb < key_hi; kb += 64) {
    if (kb == next_fold) {
      sh_fold_chunk(R);
      sh_fresh(R);
      next_fold += e.chunk;
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      vc[t][0] = vn[t][0];
      vc[t][1] = vn[t][1];
    }
    auto next = [&]() __attribute__((always_inline)) {
      if (kb + 64 < key_hi) {
        load_k_tile(kc, K, kb + 64, lane);
        load_v_tile(vn, V, kb + 64, lane);
      }
    };
    sh_block(R, [&](int kt, int st) __attribute__((always_inline)) { return kc[kt][st]; },
             [&](int dt, int h) __attribute__((always_inline)) { return vc[dt][h]; }, next, kb,
             kb >= int_lo && kb + 63 <= int_hi, e.key_lo, key_hi);
  }
  sh_put(R, e.rec, 0, kv_head, Hkv, max_recs, parts);
}

// `run` units from e on, of up to 16 tokens, by a workgroup of 4 waves, 4 tokens each: a block's K and V go to LDS once for all of them (two
// buffers, the next block's loads in flight while this one computes).  The buffers are arrays of their own, picked at compile time, so
// that the compiler does not wait for one's loads before it reads the other.
__device__ __forceinline__ void sh_tile_item(const ShEntry& e, int run, int kv_head, const int2* __restrict__ list, const uint16_t* __restrict__ q,
                                             const uint16_t* __restrict__ k_pool, const uint16_t* __restrict__ v_pool, int Hq, int Hkv,
                                             int window, int max_recs, float* __restrict__ parts, uint4 (&buf0)[2][512],
                                             uint4 (&buf1)[2][512]) {
  typedef __attribute__((address_space(3))) void* lds_ptr;
  const int lane = threadIdx.x & 63, wave = scalar((int)threadIdx.x >> 6);
  const int key_lo = e.key_lo, key_hi = sh_key_end(e, run);
  const int64_t base = e.base + (int64_t)kv_head * e.cap * 64;
  const char *Kb = reinterpret_cast<const char*>(k_pool + base), *Vb = reinterpret_cast<const char*>(v_pool + base);
  auto issue = [&](uint4 (&dst)[2][512], int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int s0 = 256 * j + 64 * wave;
      const char* blk = (s0 < 512 ? Kb : Vb) + ((size_t)kb * 8 + (s0 & 511)) * 16;
      __builtin_amdgcn_global_load_lds((const void*)(blk + (uint32_t)lane * 16u), (lds_ptr)(&dst[0][0] + s0), 16, 0, 0);
    }
  };
  auto landed = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
    lds_barrier();
  };
  const int kb_first = e.key_lo & ~63;
  issue(buf0, kb_first);
  ShRows<2> R;
  sh_rows_init(R, e, 4 * wave, list, q, kv_head, Hq, window);
  int int_lo, int_hi;
  sh_interior(R, &int_lo, &int_hi);
  int_lo = max(int_lo, e.key_lo);
  int_hi = min(int_hi, key_hi - 1);
  landed();
  if (4 * wave >= e.ntok) {  // no rows: its part of the loads, and the barriers
    int odd = 0;
    for (int kb = kb_first; kb < key_hi; kb += 64, odd ^= 1) {
      if (kb + 64 < key_hi) {
        if (odd) issue(buf0, kb + 64);
        else issue(buf1, kb + 64);
      }
      landed();
    }
    return;
  }
  int rec = e.rec, next_fold = (kb_first / e.chunk + 1) * e.chunk;
  // a block by the straight-line code: false if it has to be done by the long one (its successor's loads are out by then)
  auto fast = [&](uint4 (&cur)[2][512], uint4 (&nxt)[2][512], int kb, auto first) __attribute__((always_inline)) {
    if (kb + 64 < key_hi) issue(nxt, kb + 64);
    if (!sh_fast_block<decltype(first)::value>(R, [&](int kt, int st) __attribute__((always_inline)) { return cur[0][kt * 128 + st * 64 + lane]; },
                                                  [&](int dt, int h) __attribute__((always_inline)) { return cur[1][h * 256 + dt * 64 + lane]; }))
      return false;
    landed();
    return true;
  };
  int odd = 0;
  bool fresh = true;
  for (int kb = kb_first; kb < key_hi;) {
    if (kb == next_fold) {
      if (e.stride && !e.is_first) {
        sh_put(R, rec, 4 * wave, kv_head, Hkv, max_recs, parts);
        sh_nothing(R);
        rec += e.stride;
      } else {
        sh_fold_chunk(R);
      }
      sh_fresh(R);
      next_fold += e.chunk;
      fresh = true;
    }
    // blocks up to the fold that every row sees whole
    const int fast_end = min(min(next_fold, key_hi), int_hi - 62);
    bool issued = false;
    if (kb >= int_lo && kb < fast_end) {
      if (fresh) {
        if (odd) fast(buf1, buf0, kb, std::true_type{});
        else fast(buf0, buf1, kb, std::true_type{});
        kb += 64;
        odd ^= 1;
        fresh = false;
      }
      while (kb < fast_end) {
        if (!odd) {
          issued = !fast(buf0, buf1, kb, std::false_type{});
          if (issued) break;
          kb += 64;
          odd = 1;
          if (kb >= fast_end) break;
        }
        issued = !fast(buf1, buf0, kb, std::false_type{});
        if (issued) break;
        kb += 64;
        odd = 0;
      }
      if (!issued) continue;
    }
    // any other block: its fragments are read before the next one's loads go out, with the buffer chosen at run time
    const uint4* cur = odd ? &buf1[0][0] : &buf0[0][0];
    uint4 kc[4][2], vc[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        kc[i][j] = cur[i * 128 + j * 64 + lane];
        vc[i][j] = cur[512 + j * 256 + i * 64 + lane];
      }
    if (!issued && kb + 64 < key_hi) {
      if (odd) issue(buf0, kb + 64);
      else issue(buf1, kb + 64);
    }
    sh_block(R, [&](int kt, int st) __attribute__((always_inline)) { return kc[kt][st]; },
             [&](int dt, int h) __attribute__((always_inline)) { return vc[dt][h]; }, [] {}, kb,
             kb >= int_lo && kb + 63 <= int_hi, key_lo, key_hi);
    landed();
    kb += 64;
    odd ^= 1;
    fresh = false;
  }
  sh_put(R, rec, 4 * wave, kv_head, Hkv, max_recs, parts);
}

__global__ __launch_bounds__(256, 2) void attn_shared_kernel(const uint16_t* __restrict__ q, const uint16_t* __restrict__ k_pool,
                                                             const uint16_t* __restrict__ v_pool, int Hq, int Hkv, ShLayout L,
                                                             const char* __restrict__ plan, float* __restrict__ parts) {
  __shared__ uint4 buf0[2][512], buf1[2][512];  // [K, V][a 64-key block]
  const ShHeader* hdr = reinterpret_cast<const ShHeader*>(plan);
  const ShEntry* entries = reinterpret_cast<const ShEntry*>(plan + L.o_entries);
  const ShEntry* waves = reinterpret_cast<const ShEntry*>(plan + L.o_waves);
  const int2* list = reinterpret_cast<const int2*>(plan + L.o_list);
  const int per_head = gridDim.x / Hkv, w = blockIdx.x / Hkv, g = blockIdx.x % Hkv;
  if (!sh_plan_fits(hdr, L, Hkv)) return;
  const int n_whole = hdr->n_whole, n_split = hdr->n_split, n_own = hdr->n_own, n_waves = hdr->n_waves, window = hdr->window;
  auto tile = [&](int i, int run) __attribute__((always_inline)) {
    const ShEntry e = entries[i];
    sh_tile_item(e, run, g, list, q, k_pool, v_pool, Hq, Hkv, window, L.max_recs, parts, buf0, buf1);
  };
  // the whole tiles dealt out, the split ones in equal shares of consecutive units, the sequences' own from the other end
  const int share = n_split / per_head, more = n_split % per_head;  // (sh_share_end's)
  const int s0 = n_whole + w * share + min(w, more), s1 = s0 + share + (w < more);
  int i = w < n_whole ? w : s0, own = per_head - 1 - w;
  for (;;) {
    int at, run = 1;
    if (i < n_whole) {
      at = i;
      i += per_head;
      if (i >= n_whole) i = s0;
    } else if (i < s1) {
      at = i;
      run = min(s1 - i, entries[i].left + 1);
      i += run;
    } else if (own < n_own) {
      at = n_whole + n_split + own;
      own += per_head;
    } else {
      break;
    }
    tile(at, run);
  }
  for (int i = (per_head - 1 - w) * 4 + scalar((int)threadIdx.x >> 6); i < n_waves; i += per_head * 4) {
    const ShEntry e = waves[i];
    sh_wave_item(e, g, list, q, k_pool, v_pool, Hq, Hkv, window, L.max_recs, parts);
  }
}

// The records of a token's 8 rows of a kv head, folded: the prefix's, the sequence's own, then both and the sink.  Thread (h = tid / 16,
// part = tid % 16) takes 4 dims, with kShMergeAhead records' loads out at once (one round trip to memory for most tokens): 4.9 us for 48
// tokens of 14 + 1 records a head, 13 us for 1,478 of two.  A token
// without any record (its sequence was refused) gets zeros.
constexpr int kShMergeAhead = 12;

__global__ __launch_bounds__(128) void attn_shared_merge_kernel(const float* __restrict__ parts_in, const char* __restrict__ plan, ShLayout L,
                                                                const float* __restrict__ sinks, int Hq, int Hkv, uint16_t* __restrict__ out) {
  const ShHeader* hdr = reinterpret_cast<const ShHeader*>(plan);
  const int t = blockIdx.x, g = blockIdx.y;
  if (t >= hdr->n_tokens || !sh_plan_fits(hdr, L, Hkv)) return;  // left as it was
  const ShToken k = reinterpret_cast<const ShToken*>(plan + L.o_tokens)[t];
  float* parts = const_cast<float*>(parts_in);
  const int h = threadIdx.x >> 4, part = threadIdx.x & 15;
  const float sink = sinks[g * 8 + h] * kLog2e;
  float Mt[2], Lt[2];
  f32x4_t Ot[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int rec0 = w ? k.o_rec : k.p_rec, stride = w ? k.o_stride : k.p_stride;
    const int skip = w ? 0 : max(k.p_folded - 1, 0), n = w ? k.o_n : k.p_n - skip;  // (what the first record holds besides)
    Mt[w] = -1e30f;
    Lt[w] = 0.f;
    Ot[w] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int c0 = 0; c0 < n; c0 += kShMergeAhead) {
      float2 ml[kShMergeAhead];
      f32x4_t o[kShMergeAhead];
#pragma unroll
      for (int j = 0; j < kShMergeAhead; ++j) {
        if (c0 + j >= n) break;  // uniform
        const int rec = rec0 + (c0 + j + (c0 + j ? skip : 0)) * stride;
        ml[j] = *reinterpret_cast<const float2*>(sh_rec_ml(parts, L.max_recs, rec, Hkv, g, h));
        o[j] = *reinterpret_cast<const f32x4_t*>(sh_rec_o(parts, rec, Hkv, g, h) + part * 4);
      }
#pragma unroll
      for (int j = 0; j < kShMergeAhead; ++j)
        if (c0 + j < n) {
          const ShFold f = sh_fold(Mt[w], ml[j].x);
          Mt[w] = f.M;
          Lt[w] = fmaf(ml[j].y, f.c, Lt[w] * f.a);
#pragma unroll
          for (int d = 0; d < 4; ++d) Ot[w][d] = fmaf(o[j][d], f.c, Ot[w][d] * f.a);
        }
    }
  }
  const float M = fmaxf(sink, fmaxf(Mt[0], Mt[1]));
  const float a = __builtin_amdgcn_exp2f(Mt[0] - M), c = __builtin_amdgcn_exp2f(Mt[1] - M);
  const float total = fmaf(Lt[1], c, Lt[0] * a) + __builtin_amdgcn_exp2f(sink - M);
  const float inv = k.o_n > 0 ? 1.0f / total : 0.f;
  uint32_t w2[2];
#pragma unroll
  for (int d = 0; d < 2; ++d) {
    const float x = fmaf(Ot[1][2 * d], c, Ot[0][2 * d] * a) * inv, y = fmaf(Ot[1][2 * d + 1], c, Ot[0][2 * d + 1] * a) * inv;
    w2[d] = (uint32_t)f2bf(x) | ((uint32_t)f2bf(y) << 16);
  }
  *reinterpret_cast<uint2*>(out + ((size_t)t * Hq + g * 8 + h) * 64 + part * 4) = make_uint2(w2[0], w2[1]);
}

static int check_shared_shape(const char* what, int T, int S, int n_prefix, int Hkv) {
  FLYAI_REQUIRE(T >= 0 && T <= 65536, "%s: n_tokens %d outside [0, 65536]", what, T);
  FLYAI_REQUIRE(S >= 0 && S <= kShMaxSeqs, "%s: n_seqs %d outside [0, %d]", what, S, kShMaxSeqs);
  FLYAI_REQUIRE(n_prefix >= 0 && n_prefix <= kShMaxPrefixes, "%s: n_prefixes %d outside [0, %d]", what, n_prefix, kShMaxPrefixes);
  FLYAI_REQUIRE(Hkv >= 1 && Hkv <= 64, "%s: n_kv_heads %d outside [1, 64]", what, Hkv);
  return FLYAI_OK;
}

}  // namespace flyai

using namespace flyai;

extern "C" size_t flyai_attn_shared_plan_bytes(int32_t T, int32_t S, int32_t n_prefix) {
  if (T < 0 || T > 65536 || S < 0 || S > kShMaxSeqs || n_prefix < 0 || n_prefix > kShMaxPrefixes) return 0;
  return sh_layout(T, S, n_prefix, 1).bytes;
}

extern "C" size_t flyai_attn_shared_workspace_bytes(int32_t T, int32_t Hkv) {
  if (T < 0 || T > 65536 || Hkv < 1 || Hkv > 64) return 0;
  return (size_t)sh_layout(T, 0, 0, Hkv).max_recs * Hkv * 8 * (64 + 2) * sizeof(float);
}

extern "C" int flyai_attn_shared_plan(const int32_t* q_lens, const int32_t* starts, const int64_t* kv_base, const int32_t* kv_cap,
                                      const int32_t* prefix_of, const int32_t* prefix_len, const int64_t* prefix_base,
                                      const int32_t* prefix_cap, int32_t S, int32_t n_prefix, int32_t Hkv, int32_t window, int32_t T,
                                      int64_t pool_elems, void* plan, flyai_stream_t stream) {
  const int rc = check_shared_shape("attn_shared_plan", T, S, n_prefix, Hkv);
  if (rc) return rc;
  FLYAI_REQUIRE(window >= 0 && pool_elems >= 0, "attn_shared_plan: window and pool_elems must be >= 0");
  FLYAI_REQUIRE((S == 0 || (q_lens && starts && kv_base && kv_cap && prefix_of)) &&
                    (n_prefix == 0 || (prefix_len && prefix_base && prefix_cap)) && plan && ((uintptr_t)plan & 15) == 0,
                "attn_shared_plan: null pointer, or a plan that is not 16-byte aligned");
  const ShBatch b = {q_lens, starts, kv_base, kv_cap, prefix_of, prefix_len, prefix_base, prefix_cap, S, n_prefix, Hkv, window, T, pool_elems};
  if (S <= 256 && n_prefix <= 256 && T <= 512)
    hipLaunchKernelGGL((attn_shared_plan_kernel<256, 1>), dim3(1), dim3(256), 0, as_stream(stream), b, static_cast<char*>(plan));
  else
    hipLaunchKernelGGL((attn_shared_plan_kernel<1024, kShMaxSeqs / 1024>), dim3(1), dim3(1024), 0, as_stream(stream), b, static_cast<char*>(plan));
  return check_launch("attn_shared_plan");
}

extern "C" int flyai_attn_shared(const uint16_t* q, const uint16_t* k_pool, const uint16_t* v_pool, const float* sinks, int32_t Hq,
                                 int32_t Hkv, int32_t D, int32_t T, int32_t S, int32_t n_prefix, const void* plan, void* workspace,
                                 uint16_t* out, flyai_stream_t stream) {
  const int rc = check_shared_shape("attn_shared", T, S, n_prefix, Hkv);
  if (rc) return rc;
  FLYAI_REQUIRE(D == 64 && Hq == 8 * Hkv, "attn_shared: needs head_dim 64 and 8 query heads per kv head");
  if (T == 0) return FLYAI_OK;
  FLYAI_REQUIRE(q && k_pool && v_pool && sinks && plan && workspace && out, "attn_shared: null pointer");
  FLYAI_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)k_pool & 15) == 0 && ((uintptr_t)v_pool & 15) == 0 &&
                    ((uintptr_t)out & 15) == 0 && ((uintptr_t)workspace & 15) == 0 && ((uintptr_t)plan & 15) == 0,
                "attn_shared: q, the pools, out, plan and workspace must be 16-byte aligned");
  const ShLayout L = sh_layout(T, S, n_prefix, Hkv);
  hipStream_t s = as_stream(stream);
  hipLaunchKernelGGL(attn_shared_kernel, dim3((unsigned)(sh_per_head(Hkv) * Hkv)), dim3(256), 0, s, q, k_pool, v_pool, Hq, Hkv, L,
                     static_cast<const char*>(plan), static_cast<float*>(workspace));
  const int rc2 = check_launch("attn_shared");
  if (rc2) return rc2;
  hipLaunchKernelGGL(attn_shared_merge_kernel, dim3(T, Hkv), dim3(128), 0, s, static_cast<const float*>(workspace),
                     static_cast<const char*>(plan), L, sinks, Hq, Hkv, out);
  return check_launch("attn_shared_merge");
}
