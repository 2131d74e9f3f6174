// What the attention kernels over the KV cache share (kv_attention.cu, kv_tile.cu): their
// arguments, the units their work is cut into, and who sees what.
#pragma once

#include "common.cuh"
#include "internal.h"

namespace q8lin {

constexpr int kKvD = 128;       // head width
constexpr int kKvMaxRows = 16;  // query rows of a unit: 8 or 16
constexpr int kKvChunk = 16;    // keys of a chunk: one warp's step
constexpr int kKvWarps = 8;     // warps of a CTA that shares its SM with no other
constexpr int kKvSlots = 3;     // half chunks (16 keys or 16 values) of a warp's ring
constexpr int kKvHalf = kKvChunk * kKvD * 4;
constexpr int kKvGrid = 148;    // CTAs that share the chunks of all units (one per SM)
constexpr int kKvTileRows = 128;  // query rows of a unit of the tcgen05 kernel
constexpr int kKvTileKeys = 64;   // keys of its tiles
// Chunks a CTA takes at least, and chunks that take as long as starting on a unit: about 5 us
// against 0.6 a chunk, and 9 us against 2.2 a tile.
constexpr int kKvLeast = kKvWarps, kKvPass = kKvWarps;
constexpr int kKvTileLeast = 2, kKvTilePass = 4;

enum KvMask : int { kMaskCausal = 0, kMaskTree = 1, kMaskBlocks = 2 };

struct KvArgs {
  const float* q;         // [batch][n][hq][128], rotated
  const float* k;         // [batch][hkv][max_t][128]
  const float* v;
  const int* pos;         // [batch]
  const uint32_t* anc;    // tree: [batch][n][words], bit j: node j is the row's node or above it
  const int* index;       // blocks: [batch][n][hkv][topk], ascending, -1 behind the last
  float* out;             // [batch][n][hq][128]
  float* acc;             // [slot][rows][128] unnormalised sums of a unit's part
  float* stat;            // [slot][2][rows] its maxima and sums
  float* scores;          // causal with weights, n * group <= 16: [batch][hkv][n * group][score_stride]
  int2* begun;            // split: where a unit's parts are, for the merge
  float2* norm;           // causal with weights, else: [batch][hkv][n * group] the row's maximum and 1 / sum
  float* qscale;          // and the power of two that its query went into the products under
  int batch, n, hq, hkv, group, max_t;
  int words, topk, block, score_stride;
  int rows;               // rows of a unit: 8, 16 or 128
  int chunk;              // keys of a chunk: 16, or 64 with units of 128 rows
  int least;              // chunks a CTA takes at least
  int each;               // CTAs for every unit (0: not one for each)
  int pass;               // chunks that take as long as starting on a unit
  int rgs;                // row groups of a kv head (tree, causal) or of a token (blocks)
  int units;
  int weight_reps;        // scores stored: groups of 128 keys a CTA of the merge adds the weights of
  int split;              // 1: kKvGrid CTAs share all chunks evenly; 0: whole units
  float c;                // log2(e) * f32(1/sqrt(128))
};

// One unit: its rows, its keys.
struct KvUnit {
  int b, hk, i0;    // i0: the first row's token
  int r0, nrows;    // first row of the kv head's numbering (blocks: of the token's heads), rows
  int p;            // pos[b]
  int keys;         // causal / tree: keys [0, keys); blocks: last key + 1 of the own block
  int chunks;
  int picked;       // blocks: chosen blocks before the own one
};

template <int MASK>
__device__ __forceinline__ KvUnit kv_unit(const KvArgs& a, int u) {
  KvUnit x;
  const int rg = u % a.rgs;
  const int w = u / a.rgs;
  x.r0 = rg * a.rows;
  x.picked = 0;
  if (MASK == kMaskBlocks) {
    x.hk = w % a.hkv;
    const int row = w / a.hkv;
    x.b = row / a.n;
    x.i0 = row - x.b * a.n;
    x.nrows = min(a.rows, a.group - x.r0);
    x.p = a.pos[x.b];
    const bool ok = x.p >= 0 && x.p < a.max_t - x.i0;
    const int at = x.p + x.i0;
    x.keys = ok ? at + 1 : 0;
    x.picked = ok ? min(a.topk, at / a.block) : 0;
    x.chunks = ok ? x.picked * (a.block / kKvChunk) + (at % a.block) / kKvChunk + 1 : 0;
  } else {
    x.hk = w % a.hkv;
    x.b = w / a.hkv;
    x.nrows = min(a.rows, a.n * a.group - x.r0);
    x.i0 = x.r0 / a.group;
    x.p = a.pos[x.b];
    const int last = (x.r0 + x.nrows - 1) / a.group;
    x.keys = (x.p < 0 || x.p >= a.max_t) ? 0 : min(x.p + last + 1, a.max_t);
    x.chunks = (x.keys + a.chunk - 1) / a.chunk;
  }
  return x;
}

// First key of chunk c of the unit; `list`: the unit's chosen blocks.
template <int MASK>
__device__ __forceinline__ int kv_chunk_key(const KvArgs& a, const KvUnit& x, const int* list, int c) {
  if (MASK != kMaskBlocks) return c * kKvChunk;
  const int per = a.block / kKvChunk;
  const int nb = c / per;
  if (nb < x.picked) return list[nb] * a.block + (c - nb * per) * kKvChunk;
  return (x.keys - 1) / a.block * a.block + (c - x.picked * per) * kKvChunk;
}

template <int MASK>
__device__ __forceinline__ int kv_token(const KvArgs& a, const KvUnit& x, int r) {
  return MASK == kMaskBlocks ? x.i0 : (x.r0 + r) / a.group;
}
// Offset of row r (0 <= r < nrows) of the unit in q and out.
template <int MASK>
__device__ __forceinline__ size_t kv_row_offset(const KvArgs& a, const KvUnit& x, int r) {
  const int i = kv_token<MASK>(a, x, r);
  const int h = x.hk * a.group + (MASK == kMaskBlocks ? x.r0 + r : (x.r0 + r) % a.group);
  return (((size_t)x.b * a.n + i) * a.hq + h) * kKvD;
}
// Is the row one at all: inside the cache and, in a tree, a node.
template <int MASK>
__device__ __forceinline__ bool kv_row_valid(const KvArgs& a, const KvUnit& x, int r) {
  if (r >= x.nrows || x.p < 0) return false;
  const int i = kv_token<MASK>(a, x, r);
  if (x.p >= a.max_t - i) return false;
  if (MASK == kMaskTree) return (a.anc[((size_t)x.b * a.n + i) * a.words + (i >> 5)] >> (i & 31)) & 1u;
  return true;
}
// Bit e: does row r see key j + e (e < 32).  Two independent loads at most: a loop over the words,
// or a look per key, is a chain of L2 latencies in front of the unit's last chunk.
template <int MASK>
__device__ __forceinline__ uint32_t kv_sees(const KvArgs& a, const KvUnit& x, int r, int j) {
  const int i = kv_token<MASK>(a, x, min(r, x.nrows - 1));
  if (MASK == kMaskTree) {
    const int e0 = j - x.p;  // node number of key j
    if (e0 <= -32) return ~0u;
    const uint32_t* anc = a.anc + ((size_t)x.b * a.n + i) * a.words;
    const int w = e0 >> 5;  // -1: keys before the tree, which all rows see
    const uint32_t lo = w < 0 ? ~0u : w < a.words ? anc[w] : 0u;
    const uint32_t hi = w + 1 < a.words ? anc[w + 1] : 0u;
    return __funnelshift_r(lo, hi, e0 & 31);
  }
  const int lim = min(x.p + i + 1, x.keys) - j;
  return lim >= 32 ? ~0u : lim <= 0 ? 0u : (1u << lim) - 1;
}
// Bit e: is there a cache row j + e (e < 32); a tree's row that no node was written to is none, and
// must not reach the sums.  By whole warps, a lane per row.
template <int MASK>
__device__ __forceinline__ uint32_t kv_rows_there(const KvArgs& a, const KvUnit& x, int j) {
  j += threadIdx.x & 31;
  bool there = j < x.keys;
  if (MASK == kMaskTree && there && j >= x.p) {
    const int e = j - x.p;
    there = e < a.n && ((a.anc[((size_t)x.b * a.n + e) * a.words + (e >> 5)] >> (e & 31)) & 1u);
  }
  return __ballot_sync(kFull, there);
}

struct KvFind {
  int sum[32], top[32], before[32];  // of the warps
  int unit, off, left, quota;
};

// The split of all units' chunks over the kKvGrid CTAs: fills what CTA `cta` starts with (unit =
// units: nothing) and the chunks of a CTA's share, and returns those that CTA `cta` takes.
// Evenly, a CTA takes quota chunks wherever they lie and so begins a second unit in most cases; or
// every unit gets CTAs of its own, which then take up to `quota` chunks of it.  Starting on a
// unit costs about a.pass chunks' time (query rows, first copies, joining the parts), so units
// get their own CTAs where that adds at most a.pass chunks to the share.  (Evenly and so: trees of 64
// nodes x 8 heads behind 200 rows 26.4 and 21.5 us, 5 ragged trees of 33 nodes 37.6 and 33.4, 16 heads
// of 16 K rows 71.4 and 63.8, one block-sparse token 21.6 and 17.9.  64 units of 122 tiles stay
// even, 53 tiles to a CTA and not 64: 157 us against 173.)
template <int MASK, int THREADS>
__device__ int kv_find(const KvArgs& a, KvFind& sm, int cta) {
  constexpr int kPer = (2 * kKvGrid + THREADS - 1) / THREADS;  // more units are not split
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int c[kPer], sum = 0, top = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    c[i] = tid * kPer + i < a.units ? kv_unit<MASK>(a, tid * kPer + i).chunks : 0;
    sum += c[i];
    top = max(top, c[i]);
  }
  sum = __reduce_add_sync(kFull, sum);
  top = __reduce_max_sync(kFull, top);
  if (lane == 0) {
    sm.sum[warp] = sum;
    sm.top[warp] = top;
  }
  if (tid == 0) {
    sm.unit = a.units;
    sm.off = 0;
    sm.left = 0;
  }
  __syncthreads();
  sum = top = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    sum += sm.sum[w];
    top = max(top, sm.top[w]);
  }
  int quota = max((sum + kKvGrid - 1) / kKvGrid, a.least);
  bool own = false;
  if (a.each > 0) {
    // a share for which the units' CTAs are no more than there are
    const int spare = kKvGrid - a.units;
    const int q = max(min((top + a.each - 1) / a.each, (sum + spare - 1) / spare), a.least);
    if (q <= quota + a.pass) {
      own = true;
      quota = q;
    }
  }
  // before a unit: the CTAs that the ones in front of it get, or their chunks
  int w[kPer], upto = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    w[i] = own ? (c[i] + quota - 1) / quota : c[i];
    upto += w[i];
  }
  int at = -upto;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(kFull, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) sm.before[warp] = upto;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < THREADS / 32; ++v)
    if (v < warp) upto += sm.before[v];
  at += upto;
  const int start = own ? cta : cta * quota;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (at <= start && start < at + w[i]) {
      const int off = own ? (start - at) * quota : start - at;
      sm.unit = tid * kPer + i;
      sm.off = off;
      sm.left = own ? min(quota, c[i] - off) : quota;
    }
    at += w[i];
  }
  if (tid == 0) sm.quota = quota;
  __syncthreads();
  return sm.left;
}

}  // namespace q8lin
