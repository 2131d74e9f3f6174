// Upkeep of the f32 KV cache around the attention kernels: which rows an eviction keeps,
// moving kept rows together in place, the mean key of every block, and the blocks a query
// row attends over.
//
// Selection: the k largest of n values, equal values by the lower index, without sorting:
// the value of rank k digit by digit (8 bits at a time from the top, a 256-bin count per
// digit), then one ordered pass that emits the indices.  Floats compare as unsigned
// integers after flipping the sign bit (negative: all bits); -0 equals +0; NaN is lowest.
#include <cmath>

#include "common.cuh"
#include "internal.h"

namespace q8lin {

namespace {

constexpr int kKvD = 128;

__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long order_key(double x) {
  if (x != x) return 0ull;
  const unsigned long long u = (unsigned long long)__double_as_longlong(x + 0.0);
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

// Counts are kept eightfold, by lane: exponents crowd into few bins, and lanes of a warp that meet
// in one take turns.
constexpr int kHistCopies = 8, kHistStride = 257;
struct SelectSmem {
  unsigned hist[kHistCopies * kHistStride];
  unsigned count[256];
  unsigned digit, above, bin;
  unsigned warp[32][2];
};

// Rank-k threshold of key(0..n): keys with (key & mask) > prefix are chosen, and the first
// `ties` of those with (key & mask) == prefix.  1 <= k <= n.  Every thread of the CTA calls it.
template <typename U, typename F>
__device__ void select_threshold(F key, int n, int k, SelectSmem& sm, U& prefix, U& mask, int& ties) {
  const int tid = threadIdx.x;
  prefix = 0;
  mask = 0;
  int need = k;
  for (int shift = (int)sizeof(U) * 8 - 8; shift >= 0; shift -= 8) {
    for (int i = tid; i < kHistCopies * kHistStride; i += blockDim.x) sm.hist[i] = 0;
    __syncthreads();
    unsigned* mine = sm.hist + (tid & (kHistCopies - 1)) * kHistStride;
    for (int i = tid; i < n; i += blockDim.x) {
      const U v = key(i);
      if ((v & mask) == prefix) atomicAdd(&mine[(unsigned)(v >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid < 256) {
      unsigned c = 0;
#pragma unroll
      for (int h = 0; h < kHistCopies; ++h) c += sm.hist[h * kHistStride + tid];
      sm.count[tid] = c;
    }
    __syncthreads();
    if (tid < 32) {  // lane l: digits 255 - 8l down to 248 - 8l
      unsigned c[8], sum = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        c[e] = sm.count[255 - 8 * tid - e];
        sum += c[e];
      }
      unsigned upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned v = __shfl_up_sync(kFull, upto, o);
        if (tid >= o) upto += v;
      }
      unsigned at = upto - sum;
      if (at < (unsigned)need && (unsigned)need <= upto) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (at < (unsigned)need && (unsigned)need <= at + c[e]) {
            sm.digit = 255 - 8 * tid - e;
            sm.above = at;
            sm.bin = c[e];
          }
          at += c[e];
        }
      }
    }
    __syncthreads();
    prefix |= (U)sm.digit << shift;
    mask |= (U)255 << shift;
    need -= (int)sm.above;
    const bool all = sm.bin == (unsigned)need;  // the whole digit is chosen: no need to go on
    __syncthreads();
    if (all) break;
  }
  ties = need;
}

// Calls emit(rank, i) for the chosen of key(0..n) in ascending i.  Every thread calls it.
template <typename U, typename F, typename E>
__device__ void select_emit(F key, int n, U prefix, U mask, int ties, SelectSmem& sm, E emit) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  const int per = (n + (int)blockDim.x - 1) / (int)blockDim.x;
  const int i0 = min(n, tid * per), i1 = min(n, i0 + per);
  unsigned more = 0, same = 0;
  for (int i = i0; i < i1; ++i) {
    const U v = key(i) & mask;
    more += v > prefix;
    same += v == prefix;
  }
  unsigned um = more, us = same;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned a = __shfl_up_sync(kFull, um, o), b = __shfl_up_sync(kFull, us, o);
    if (lane >= o) {
      um += a;
      us += b;
    }
  }
  if (lane == 31) {
    sm.warp[warp][0] = um;
    sm.warp[warp][1] = us;
  }
  __syncthreads();
  unsigned bm = um - more, bs = us - same;  // chosen for certain, and equal ones, before i0
  for (int w = 0; w < warps; ++w)
    if (w < warp) {
      bm += sm.warp[w][0];
      bs += sm.warp[w][1];
    }
  for (int i = i0; i < i1; ++i) {
    const U v = key(i) & mask;
    const bool tie = v == prefix;
    if (v > prefix || (tie && bs < (unsigned)ties)) emit((int)(bm + min(bs, (unsigned)ties)), i);
    bm += v > prefix;
    bs += tie;
  }
  __syncthreads();
}

// One CTA per (sequence, kv head): the rows an eviction keeps, ascending, and the weights
// of the kept rows.  Keys come from shared memory where the row of weights fits.  Bound by its
// chain of four counting passes and an ordered one: 19 us for 4096 of 8001 rows (64 heads).
constexpr int kEvictThreads = 1024;
constexpr int kEvictSmemRows = 49152;
__global__ void __launch_bounds__(kEvictThreads)
kv_evict_kernel(const float* weight, const int* __restrict__ length, int hkv, int max_t, int keep, int sink,
                int recent, int staged, int* __restrict__ index, float* weight_out) {
  extern __shared__ uint32_t ev_keys[];
  __shared__ SelectSmem sm;
  const int tid = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  const size_t bh = blockIdx.x;
  const int len = min(max(length[bh / hkv], 0), max_t);
  const float* w = weight + bh * (size_t)max_t;
  int* idx = index + bh * (size_t)keep;
  const int kept = min(len, keep);
  if (len <= keep) {
    for (int i = tid; i < keep; i += kEvictThreads) idx[i] = i < len ? i : -1;
  } else {
    const int n = len - sink - recent, k = keep - sink - recent;
    for (int i = tid; i < sink; i += kEvictThreads) idx[i] = i;
    for (int i = tid; i < recent; i += kEvictThreads) idx[keep - recent + i] = len - recent + i;
    if (k > 0) {
      if (staged)
        for (int i = tid; i < n; i += kEvictThreads) ev_keys[i] = order_key(w[sink + i]);
      __syncthreads();
      auto key = [&](int i) { return staged ? ev_keys[i] : order_key(w[sink + i]); };
      uint32_t prefix, mask;
      int ties;
      select_threshold<uint32_t>(key, n, k, sm, prefix, mask, ties);
      select_emit<uint32_t>(key, n, prefix, mask, ties, sm, [&](int rank, int i) { idx[sink + rank] = sink + i; });
    }
  }
  if (!weight_out) return;
  __syncthreads();  // the indices of the CTA are written
  // weight_out may be weight: a row moves to a lower or the same place, so a group of rows is
  // read before any of it is written, and nothing behind it is
  float* wo = weight_out + bh * (size_t)max_t;
  for (int c = 0; c < kept; c += kEvictThreads) {
    const int i = c + tid;
    const float v = i < kept ? w[idx[i]] : 0.0f;
    __syncthreads();
    if (i < kept) wo[i] = v;
  }
  __syncthreads();
  for (int i = kept + tid; i < max_t; i += kEvictThreads) wo[i] = 0.0f;
}

// Row base + i of a cache head <- row base + index[i] for ascending indices, index[i] >= i,
// in place.  A row moves down, so rows are taken in ascending groups: a group is read whole
// before any of it is written, and later groups read only rows behind it.  A CTA owns a slice of
// `lanes` 16-byte pieces of the rows of one head of one cache, so no two CTAs meet.  Bound by HBM:
// 4096 of 8001 rows of 64 heads in 95 us, 5.6 TB/s read and written.
constexpr int kMoveThreads = 256;
constexpr int kMoveDepth = 8;
__global__ void __launch_bounds__(kMoveThreads, 4)
kv_move_kernel(float* __restrict__ kc, float* __restrict__ vc, const int* __restrict__ index,
               const int* __restrict__ base_dev, int hkv, int index_heads, int max_t, int count, int lanes) {
  pdl_launch_dependents();
  pdl_wait();
  const int bh = blockIdx.y, b = bh / hkv, h = bh - b * hkv;
  const int slices = 32 / lanes;
  const int slice = blockIdx.x % slices;
  const int base = base_dev ? base_dev[b] : 0;
  if (base < 0 || base >= max_t) return;
  float4* cache = reinterpret_cast<float4*>((blockIdx.x / slices ? vc : kc) + (size_t)bh * max_t * kKvD) +
                  (size_t)base * (kKvD / 4);
  const int limit = max_t - base;
  const int* idx = index + ((size_t)b * index_heads + (index_heads == 1 ? 0 : h)) * (size_t)count;
  const int piece = slice * lanes + threadIdx.x % lanes, r0 = threadIdx.x / lanes, step = kMoveThreads / lanes;
  for (int c = 0; c < count; c += step * kMoveDepth) {
    float4 v[kMoveDepth];
    bool move[kMoveDepth];
#pragma unroll
    for (int d = 0; d < kMoveDepth; ++d) {
      const int i = c + d * step + r0;
      const int from = i < count ? idx[i] : -1;
      move[d] = from > i && from < limit;
      if (move[d]) v[d] = cache[(size_t)from * (kKvD / 4) + piece];
    }
    __syncthreads();
#pragma unroll
    for (int d = 0; d < kMoveDepth; ++d)
      if (move[d]) cache[(size_t)(c + d * step + r0) * (kKvD / 4) + piece] = v[d];
  }
}

// Mean key of every block that rows [pos, pos + t) complete: f64 sum in row order, rounded
// once.  grid (blocks that t rows can complete, batch * hkv), one thread per dimension.
__global__ void __launch_bounds__(kKvD)
kv_block_keys_kernel(const float* __restrict__ kc, const int* __restrict__ pos_dev, int t, int hkv, int max_t, int block,
                     int blocks, float* __restrict__ keys) {
  pdl_launch_dependents();
  pdl_wait();
  const int bh = blockIdx.y, pos = pos_dev[bh / hkv];
  if (pos < 0 || pos >= max_t) return;
  const int end = min((int64_t)pos + t, (int64_t)max_t);
  const int c = pos / block + blockIdx.x;
  if ((int64_t)(c + 1) * block > end || c >= blocks) return;
  const float* k = kc + ((size_t)bh * max_t + (size_t)c * block) * kKvD + threadIdx.x;
  double s = 0.0;
#pragma unroll 8
  for (int r = 0; r < block; ++r) s += (double)k[(size_t)r * kKvD];
  keys[((size_t)bh * blocks + c) * kKvD + threadIdx.x] = (float)(s / block);
}

// The blocks a query row attends over besides its own.  Score of block c: sum over the heads of
// the group and the dimensions of q times the block's mean key, in f64, so the choice does not
// hang on the order of the sums.
//
// A block of 8 lanes takes 16 dimensions each of a block's key for the ROWS tokens of the CTA at
// once (the keys are what is read most), two keys in flight.  ROWS = 1 splits a row's blocks over a
// cluster of CTAs where rows alone leave SMs idle: each writes its order keys into the first
// CTA's shared memory, which chooses.  512 tokens x 2 heads over 250 blocks 31 us: latency of the
// f64 sums and of the bitwise search at eight warps an SM.
constexpr int kPickThreads = 256;
constexpr int kPickRows = 8;
template <int ROWS>
__global__ void __launch_bounds__(kPickThreads)
kv_pick_kernel(const float* __restrict__ q, const float* __restrict__ keys, const int* __restrict__ pos_dev, int n, int hq,
               int hkv, int max_t, int block, int blocks, int topk, int* __restrict__ index) {
  extern __shared__ unsigned long long pk_keys[];  // [ROWS][blocks]
  __shared__ SelectSmem sm;
  __shared__ alignas(16) double qs[ROWS][kKvD];
  const int tid = threadIdx.x;
  pdl_launch_dependents();
  uint32_t rank = 0, ranks = 1;
  if (ROWS == 1) {
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    // every CTA of the cluster runs before another writes into its shared memory
    if (ranks > 1)
      asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  pdl_wait();
  // a list: ROWS tokens of one sequence and kv head
  const int groups = (n + ROWS - 1) / ROWS;
  const int list = blockIdx.x / ranks, hk = list % hkv, bg = list / hkv, b = bg / groups, i0 = (bg - b * groups) * ROWS;
  const int group = hq / hkv, p = pos_dev[b];
  auto row_past = [&](int i) { return i < n && p >= 0 && p < max_t - i ? min((p + i) / block, blocks) : 0; };
  auto row_index = [&](int i) { return index + (((size_t)b * n + i) * hkv + hk) * topk; };
  int past = 0;  // blocks some row of the list has before its own: the last row's
  for (int r = 0; r < ROWS; ++r) past = max(past, row_past(i0 + r));
  if (past > topk) {
    for (int e = tid; e < ROWS * kKvD; e += kPickThreads) {
      const int r = e / kKvD, d = e % kKvD;
      double s = 0.0;
      if (i0 + r < n) {
        const float* row = q + (((size_t)b * n + i0 + r) * hq + hk * group) * kKvD + d;
#pragma unroll 8
        for (int h = 0; h < group; ++h) s += (double)row[(size_t)h * kKvD];
      }
      qs[r][d] = s;
    }
    __syncthreads();
    const float4* kb = reinterpret_cast<const float4*>(keys + ((size_t)b * hkv + hk) * blocks * kKvD);
    const int l8 = tid & 7;
    uint32_t first = (uint32_t)__cvta_generic_to_shared(pk_keys);
    if (ROWS == 1 && ranks > 1) asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(first) : "r"(first));
    constexpr int kStep = kPickThreads / 8;
    for (int c0 = (int)rank * kStep + (tid >> 3); c0 - (tid >> 3) < past; c0 += 2 * kStep * (int)ranks) {
      float4 k4[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const int c = c0 + u * kStep * (int)ranks;
          k4[u][m] = c < past ? kb[(size_t)c * 32 + m * 8 + l8] : make_float4(0.f, 0.f, 0.f, 0.f);
        }
      double s[2][ROWS];
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        s[0][r] = s[1][r] = 0.0;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const double2* qd = reinterpret_cast<const double2*>(&qs[r][(m * 8 + l8) * 4]);
          const double2 qa = qd[0], qb = qd[1];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            s[u][r] = fma(qa.x, (double)k4[u][m].x, s[u][r]);
            s[u][r] = fma(qa.y, (double)k4[u][m].y, s[u][r]);
            s[u][r] = fma(qb.x, (double)k4[u][m].z, s[u][r]);
            s[u][r] = fma(qb.y, (double)k4[u][m].w, s[u][r]);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int c = c0 + u * kStep * (int)ranks;
        if (ROWS == 1) {
          double v = s[u][0];
          v += __shfl_xor_sync(kFull, v, 1);
          v += __shfl_xor_sync(kFull, v, 2);
          v += __shfl_xor_sync(kFull, v, 4);
          if (c < past && l8 == 0)
            asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(first + 8u * (uint32_t)c), "l"(order_key(v)) : "memory");
        } else {
          // eight sums over eight lanes, each lane left with one row's: 7 shuffles for 24
          double v[ROWS];
#pragma unroll
          for (int r = 0; r < ROWS; ++r) v[r] = s[u][r];
#pragma unroll
          for (int o = ROWS / 2; o > 0; o >>= 1) {
            const bool up = (l8 & o) != 0;
#pragma unroll
            for (int r = 0; r < o; ++r) {
              const double send = up ? v[r] : v[r + o], keep = up ? v[r + o] : v[r];
              v[r] = keep + __shfl_xor_sync(kFull, send, o);
            }
          }
          if (c < past) pk_keys[l8 * blocks + c] = order_key(v[0]);
        }
      }
    }
  }
  if (ROWS == 1 && ranks > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank > 0) return;
  } else {
    __syncthreads();
  }
  if (ROWS == 1) {
    if (i0 >= n) return;
    int* idx = row_index(i0);
    if (past <= topk) {
      for (int e = tid; e < topk; e += kPickThreads) idx[e] = e < past ? e : -1;
      return;
    }
    auto key = [&](int c) { return pk_keys[c]; };
    unsigned long long prefix, mask;
    int ties;
    select_threshold<unsigned long long>(key, past, topk, sm, prefix, mask, ties);
    select_emit<unsigned long long>(key, past, prefix, mask, ties, sm, [&](int rk, int c) { idx[rk] = c; });
    return;
  }
  // a warp per row: the topk-th largest order key bit by bit from the top, then one ordered pass
  static_assert(ROWS == 1 || ROWS == kPickThreads / 32, "a warp per row");
  const int r = tid >> 5, lane = tid & 31, i = i0 + r;
  if (i >= n) return;
  int* idx = row_index(i);
  const int mine = row_past(i);
  if (mine <= topk) {
    for (int e = lane; e < topk; e += 32) idx[e] = e < mine ? e : -1;
    return;
  }
  const unsigned long long* kr = pk_keys + (size_t)r * blocks;
  // The threshold is the largest T with at least topk keys >= T; the search ends early when exactly
  // topk are.
  unsigned long long T = 0;
  for (int bit = 63; bit >= 0; --bit) {
    const unsigned long long t = T | (1ull << bit);
    int cnt = 0;
    for (int c = lane; c < mine; c += 32) cnt += kr[c] >= t;
    cnt = __reduce_add_sync(kFull, cnt);
    if (cnt >= topk) T = t;
    if (cnt == topk) break;
  }
  int above = 0;
  for (int c = lane; c < mine; c += 32) above += kr[c] > T;
  int ties = topk - __reduce_add_sync(kFull, above), out = 0;
  for (int c0 = 0; c0 < mine; c0 += 32) {
    const int c = c0 + lane;
    const unsigned long long k = c < mine ? kr[c] : 0ull;
    const unsigned tie = __ballot_sync(kFull, c < mine && k == T);
    const bool take = c < mine && (k > T || (k == T && __popc(tie & ((1u << lane) - 1)) < ties));
    const unsigned chosen = __ballot_sync(kFull, take);
    if (take) idx[out + __popc(chosen & ((1u << lane) - 1))] = c;
    out += __popc(chosen);
    ties -= min(ties, __popc(tie));
  }
}

cudaLaunchConfig_t kc_cfg(dim3 grid, dim3 block, size_t smem, cudaStream_t s, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  return cfg;
}

}  // namespace

cudaError_t launch_kv_evict(const float* weight, const int* length, int batch, int hkv, int max_t, int keep, int sink,
                            int recent, int* index, float* weight_out, int device, cudaStream_t s) {
  const bool staged = max_t <= kEvictSmemRows;
  const size_t smem = staged ? (size_t)max_t * 4 : 0;
  static int configured[128] = {0};
  cudaError_t e =
      ensure_smem((const void*)kv_evict_kernel, configured, device, (size_t)kEvictSmemRows * 4, false);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = kc_cfg(dim3((unsigned)(batch * hkv)), dim3(kEvictThreads), smem, s, attr);
  return cudaLaunchKernelEx(&cfg, kv_evict_kernel, weight, length, hkv, max_t, keep, sink, recent, staged ? 1 : 0, index,
                            weight_out);
}

cudaError_t launch_kv_move(float* kc, float* vc, const int* index, const int* base, int batch, int hkv, int index_heads,
                           int max_t, int count, cudaStream_t s) {
  // slices of 128 bytes, or of 32 (a DRAM sector) where the heads alone leave SMs idle (the whole
  // eviction of 64 heads, 8001 to 4096 rows: 114 us in slices of 128, 133 in slices of 32; of 2 heads,
  // 640 to 320, replayed from a graph: 10.3 and 9.1)
  const int lanes = batch * hkv * 2 * 4 >= 296 ? 8 : 2;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg =
      kc_cfg(dim3((unsigned)(2 * 32 / lanes), (unsigned)(batch * hkv)), dim3(kMoveThreads), 0, s, attr);
  return cudaLaunchKernelEx(&cfg, kv_move_kernel, kc, vc, index, base, hkv, index_heads, max_t, count, lanes);
}

cudaError_t launch_kv_block_keys(const float* kc, const int* pos, int batch, int t, int hkv, int max_t, int block,
                                 float* keys, cudaStream_t s) {
  const int blocks = (max_t + block - 1) / block;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg =
      kc_cfg(dim3((unsigned)(t / block + 1), (unsigned)(batch * hkv)), dim3(kKvD), 0, s, attr);
  return cudaLaunchKernelEx(&cfg, kv_block_keys_kernel, kc, pos, t, hkv, max_t, block, blocks, keys);
}

cudaError_t launch_kv_pick(const float* q, const float* keys, const int* pos, int batch, int n, int hq, int hkv,
                           int max_t, int block, int topk, int* index, int device, cudaStream_t s) {
  const int blocks = (max_t + block - 1) / block;
  const int64_t rows = (int64_t)batch * n * hkv;
  cudaLaunchAttribute attr[2];
  // eight tokens a CTA where that still fills the SMs and their order keys fit (512 tokens over 250
  // blocks, with their attention: 188.8 us, a token a CTA 190.5)
  if (n >= kPickRows && rows / kPickRows >= 74 && (size_t)blocks * 8 * kPickRows <= 128 * 1024) {
    static int configured[128] = {0};
    cudaError_t e = ensure_smem((const void*)kv_pick_kernel<kPickRows>, configured, device, 128 * 1024, false);
    if (e != cudaSuccess) return e;
    const int64_t lists = (int64_t)batch * hkv * ((n + kPickRows - 1) / kPickRows);
    cudaLaunchConfig_t cfg = kc_cfg(dim3((unsigned)lists), dim3(kPickThreads), (size_t)blocks * 8 * kPickRows, s, attr);
    return cudaLaunchKernelEx(&cfg, kv_pick_kernel<kPickRows>, q, keys, pos, n, hq, hkv, max_t, block, blocks, topk, index);
  }
  static int configured[128] = {0};
  cudaError_t e = ensure_smem((const void*)kv_pick_kernel<1>, configured, device, (size_t)kKvMaxBlocks * 8, false);
  if (e != cudaSuccess) return e;
  // a cluster of CTAs per row while there are SMs for it; at least 64 blocks a CTA (one token over 500
  // blocks, with its attention, replayed from a graph: 17.5 us, one CTA a row 24.9; 8 x 16 rows over 250: 47.8
  // and 50.7)
  unsigned ranks = 1;
  while (ranks < 8 && rows * ranks * 2 <= 296 && blocks >= 128 * (int)ranks) ranks *= 2;
  cudaLaunchConfig_t cfg = kc_cfg(dim3((unsigned)(rows * ranks)), dim3(kPickThreads), (size_t)blocks * 8, s, attr);
  attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
  attr[cfg.numAttrs].val.clusterDim.x = ranks;
  attr[cfg.numAttrs].val.clusterDim.y = 1;
  attr[cfg.numAttrs].val.clusterDim.z = 1;
  ++cfg.numAttrs;
  return cudaLaunchKernelEx(&cfg, kv_pick_kernel<1>, q, keys, pos, n, hq, hkv, max_t, block, blocks, topk, index);
}

}  // namespace q8lin
