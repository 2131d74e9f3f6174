// Attention of several query rows per kv head over the f32 KV cache: trees of drafted
// tokens, causal rows that also accumulate every key's softmax weight, and rows that
// attend over chosen blocks of keys.
//
//   out_r = sum_j p_rj v_j,  p_rj = 2^(s_rj - m_r) / l_r,  s_rj = q_r . k_j * log2(e)/sqrt(128)
//   over the keys j that row r sees; m_r the running maximum, l_r the running sum, both
//   f32, kept per warp and merged at the end (a row that sees nothing gives 0).
//
// Rows: sequence b has n new rows at positions pos[b] + i (pos in device memory).  The
// `group` query heads of one kv head read the same keys, so the rows of a kv head are
// numbered r = i * group + head-in-group and taken 16 at a time (a unit).
//
// Products: f32 operands as tf32 pairs on the tensor cores (mma.sync m16n8k8).  x = hi + lo
// with hi = x rounded to tf32's 11 significant bits and lo = x - hi (exact) rounded again, and
// a.b = hi.hi + lo.hi + hi.lo: what is dropped (lo.lo and lo's rounding) is below 3 * 2^-24 of
// each product, about f32's own rounding; f32's exponent range stays.
#include <cmath>

#include "common.cuh"
#include "internal.h"

namespace q8lin {

namespace {

constexpr int kKvD = 128;       // head width
constexpr int kKvRows = 16;     // query rows of a unit
constexpr int kKvChunk = 16;    // keys of a chunk: one warp's step
constexpr int kKvWarps = 4;
constexpr int kKvThreads = kKvWarps * 32;
constexpr int kKvStages = 2;    // chunks per warp in flight or in use
constexpr int kKvGrid = 148;    // CTAs that share the chunks of all units (one per SM)
constexpr int kKvSlotFloats = kKvRows * kKvD;

enum KvMask : int { kMaskCausal = 0, kMaskTree = 1, kMaskBlocks = 2 };

struct KvArgs {
  const float* q;         // [batch][n][hq][128], rotated
  const float* k;         // [batch][hkv][max_t][128]
  const float* v;
  const int* pos;         // [batch]
  const uint32_t* anc;    // tree: [batch][n][words], bit j: node j is the row's node or above it
  const int* index;       // blocks: [batch][n][hkv][topk], ascending, -1 behind the last
  float* out;             // [batch][n][hq][128]
  float* acc;             // [slot][16][128] unnormalised sums of a unit's part
  float* stat;            // [slot][2][16] its maxima and sums
  float* scores;          // causal with weights, n * group <= 16: [batch][hkv][n * group][score_stride]
  float* lse;             // causal with weights, else: [batch][hkv][n * group] log2 of the row's sum
  int batch, n, hq, hkv, group, max_t;
  int words, topk, block, score_stride;
  int rgs;                // row groups of a kv head (tree, causal) or of a row (blocks)
  int units;
  int split;              // 1: kKvGrid CTAs share all chunks evenly; 0: one CTA per unit
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
  x.r0 = rg * kKvRows;
  x.picked = 0;
  if (MASK == kMaskBlocks) {
    x.hk = w % a.hkv;
    const int row = w / a.hkv;
    x.b = row / a.n;
    x.i0 = row - x.b * a.n;
    x.nrows = min(kKvRows, a.group - x.r0);
    x.p = a.pos[x.b];
    const bool ok = x.p >= 0 && x.p < a.max_t - x.i0;
    const int at = x.p + x.i0;
    x.keys = ok ? at + 1 : 0;
    x.picked = ok ? min(a.topk, at / a.block) : 0;
    x.chunks = ok ? x.picked * (a.block / kKvChunk) + (at % a.block) / kKvChunk + 1 : 0;
  } else {
    x.hk = w % a.hkv;
    x.b = w / a.hkv;
    x.nrows = min(kKvRows, a.n * a.group - x.r0);
    x.i0 = x.r0 / a.group;
    x.p = a.pos[x.b];
    const int last = (x.r0 + x.nrows - 1) / a.group;
    x.keys = (x.p < 0 || x.p >= a.max_t) ? 0 : min(x.p + last + 1, a.max_t);
    x.chunks = (x.keys + kKvChunk - 1) / kKvChunk;
  }
  return x;
}

// First key of chunk c of the unit.
template <int MASK>
__device__ __forceinline__ int kv_chunk_key(const KvArgs& a, const KvUnit& x, int c) {
  if (MASK != kMaskBlocks) return c * kKvChunk;
  const int per = a.block / kKvChunk;
  const int nb = c / per;
  if (nb < x.picked) {
    const int blk = a.index[(((size_t)x.b * a.n + x.i0) * a.hkv + x.hk) * a.topk + nb];
    return blk * a.block + (c - nb * per) * kKvChunk;
  }
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
template <int MASK>
__device__ __forceinline__ bool kv_sees(const KvArgs& a, const KvUnit& x, int r, int j) {
  const int i = kv_token<MASK>(a, x, min(r, x.nrows - 1));
  if (MASK == kMaskTree) {
    const int e = j - x.p;
    if (e < 0) return true;
    if (e >= a.n) return false;
    return (a.anc[((size_t)x.b * a.n + i) * a.words + (e >> 5)] >> (e & 31)) & 1u;
  }
  return j <= x.p + i;
}

__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t a0, const uint32_t a1, const uint32_t a2,
                                         const uint32_t a3, const uint32_t b0, const uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = (__float_as_uint(__fsub_rn(x, __uint_as_float(hi))) + 0x1000u) & 0xffffe000u;
}
__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool there) {
  const uint32_t n = there ? 16u : 0u;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ float4 lds_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

struct KvSmem {
  // the unit's query rows as MMA fragments: [hi, lo][pair of k-steps][rows g, rows g + 8][lane]
  alignas(16) float4 q[2][8][2][32];
  alignas(16) float k[kKvWarps][kKvStages][kKvChunk][kKvD];
  alignas(16) float v[kKvWarps][kKvStages][kKvChunk][kKvD];
  alignas(16) float o[kKvWarps][kKvRows][kKvD + 4];
  float m[kKvWarps][kKvRows], l[kKvWarps][kKvRows];
  int ok[kKvRows];
  int seg[kKvWarps];
  int unit, off;
};

// Where CTA `cta` of the shared split starts: fills sm.unit / sm.off and returns the chunk
// count of one CTA (the whole work when it does not reach this CTA: unit = units).
template <int MASK>
__device__ int kv_find(const KvArgs& a, KvSmem& sm, int cta) {
  const int tid = threadIdx.x;
  const int per = (a.units + kKvThreads - 1) / kKvThreads;
  const int u0 = min(a.units, tid * per), u1 = min(a.units, u0 + per);
  int mine = 0;
  for (int u = u0; u < u1; ++u) mine += kv_unit<MASK>(a, u).chunks;
  int upto = mine;  // chunks of this thread's units and of those before them
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(kFull, upto, o);
    if ((tid & 31) >= o) upto += v;
  }
  if ((tid & 31) == 31) sm.seg[tid >> 5] = upto;
  if (tid == 0) {
    sm.unit = a.units;
    sm.off = 0;
  }
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < kKvWarps; ++w) {
    if (w < (tid >> 5)) upto += sm.seg[w];
    total += sm.seg[w];
  }
  const int quota = max((total + kKvGrid - 1) / kKvGrid, kKvWarps);
  const int start = cta * quota;
  if (upto - mine <= start && start < upto) {
    int at = upto - mine;
    for (int u = u0; u < u1; ++u) {
      const int c = kv_unit<MASK>(a, u).chunks;
      if (start < at + c) {
        sm.unit = u;
        sm.off = start - at;
        break;
      }
      at += c;
    }
  }
  __syncthreads();
  return quota;
}

template <int MASK, bool SCORES>
__global__ void __launch_bounds__(kKvThreads, 1) kv_attention_kernel(const KvArgs a) {
  extern __shared__ __align__(16) uint8_t kv_smem[];
  KvSmem& sm = *reinterpret_cast<KvSmem*>(kv_smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  pdl_wait();
  pdl_launch_dependents();  // the merge waits for this grid before it reads anything

  int u, off, left;
  if (a.split) {
    left = kv_find<MASK>(a, sm, blockIdx.x);
    u = sm.unit;
    off = sm.off;
  } else {
    u = a.units - 1 - (int)blockIdx.x;  // later rows see more keys: longest first
    off = 0;
    left = 0x7fffffff;
  }
  const uint32_t ks = (uint32_t)__cvta_generic_to_shared(&sm.k[warp][0][0][0]);
  const uint32_t vs = (uint32_t)__cvta_generic_to_shared(&sm.v[warp][0][0][0]);
  constexpr uint32_t kStage = kKvChunk * kKvD * 4;

  while (u < a.units && left > 0) {
    const KvUnit x = kv_unit<MASK>(a, u);
    const int c1 = min(x.chunks, off > x.chunks - left ? x.chunks : off + left);
    const float* kb = a.k + ((size_t)x.b * a.hkv + x.hk) * (size_t)a.max_t * kKvD;
    const float* vb = a.v + ((size_t)x.b * a.hkv + x.hk) * (size_t)a.max_t * kKvD;

    // this warp's chunks: off + warp, off + warp + 4, ...
    auto load = [&](int c, int stage) {
      const int j0 = kv_chunk_key<MASK>(a, x, c);
#pragma unroll
      for (int r = 0; r < kKvChunk; ++r) {
        const int j = j0 + r;
        bool there = j < x.keys;
        if (MASK == kMaskTree && j >= x.p) {
          const int e = j - x.p;  // a row no node was written to must not reach the sums
          there = there && e < a.n && ((a.anc[((size_t)x.b * a.n + e) * a.words + (e >> 5)] >> (e & 31)) & 1u);
        }
        const size_t o = (size_t)(there ? j : 0) * kKvD + lane * 4;
        const uint32_t row = stage * kStage + r * (kKvD * 4);
        cp_async16_zfill(ks + row + ((lane ^ ((r & 1) << 2)) << 4), kb + o, there);
        cp_async16_zfill(vs + row + ((lane ^ (((r >> 1) & 3) << 1)) << 4), vb + o, there);
      }
    };
    int c = off + warp;
#pragma unroll
    for (int s = 0; s < kKvStages; ++s) {
      if (c + s * kKvWarps < c1) load(c + s * kKvWarps, s);
      cp_async_commit();
    }
    // query rows -> fragments
    for (int e = tid; e < 8 * 2 * 32; e += kKvThreads) {
      const int ln = e & 31, half = (e >> 5) & 1, pair = e >> 6;
      const int r = (ln >> 2) + 8 * half;
      float4 qv = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < x.nrows)
        qv = *reinterpret_cast<const float4*>(a.q + kv_row_offset<MASK>(a, x, r) + pair * 16 + (ln & 3) * 4);
      uint4 h, w;
      split_tf32(qv.x, h.x, w.x);
      split_tf32(qv.y, h.y, w.y);
      split_tf32(qv.z, h.z, w.z);
      split_tf32(qv.w, h.w, w.w);
      *reinterpret_cast<uint4*>(&sm.q[0][pair][half][ln]) = h;
      *reinterpret_cast<uint4*>(&sm.q[1][pair][half][ln]) = w;
    }
    __syncthreads();

    // the first key some row of the unit does not see (chunks below it need no mask)
    const int open = MASK == kMaskTree ? x.p : MASK == kMaskCausal ? x.p + x.i0 + 1 : x.keys;
    float o[16][4];
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;

    for (int it = 0; c < c1; c += kKvWarps, ++it) {
      const int stage = it & (kKvStages - 1);
      cp_async_wait(kKvStages - 1);
      __syncwarp();
      const uint32_t kst = ks + stage * kStage, vst = vs + stage * kStage;
      const int j0 = kv_chunk_key<MASK>(a, x, c);
      // scores: a lane takes dimensions 16 pair + 4 t + e of key 8 nt + g.  The tensor cores
      // cut their f32 sums instead of rounding them, one cut per step: hi.hi runs in chains
      // of four steps, summed here with rounding; the cross terms are 2^-11 of it and run on.
      float s[2][4], cross[2][2][4];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][e] = cross[nt][0][e] = cross[nt][1][e] = 0.0f;
#pragma unroll
      for (int quad = 0; quad < 4; ++quad) {
        float h4[2][4];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) h4[nt][e] = 0.0f;
#pragma unroll
        for (int pair = 2 * quad; pair < 2 * quad + 2; ++pair) {
          const uint4 hg = *reinterpret_cast<const uint4*>(&sm.q[0][pair][0][lane]);
          const uint4 hh = *reinterpret_cast<const uint4*>(&sm.q[0][pair][1][lane]);
          const uint4 lg = *reinterpret_cast<const uint4*>(&sm.q[1][pair][0][lane]);
          const uint4 lh = *reinterpret_cast<const uint4*>(&sm.q[1][pair][1][lane]);
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            const int r = nt * 8 + g;
            const float4 kv = lds_f4(kst + r * (kKvD * 4) + (((pair * 4 + t) ^ ((r & 1) << 2)) << 4));
            uint32_t h0, h1, h2, h3, w0, w1, w2, w3;
            split_tf32(kv.x, h0, w0);
            split_tf32(kv.y, h1, w1);
            split_tf32(kv.z, h2, w2);
            split_tf32(kv.w, h3, w3);
            mma_tf32(h4[nt], hg.x, hh.x, hg.y, hh.y, h0, h1);
            mma_tf32(cross[nt][0], lg.x, lh.x, lg.y, lh.y, h0, h1);
            mma_tf32(cross[nt][1], hg.x, hh.x, hg.y, hh.y, w0, w1);
            mma_tf32(h4[nt], hg.z, hh.z, hg.w, hh.w, h2, h3);
            mma_tf32(cross[nt][0], lg.z, lh.z, lg.w, lh.w, h2, h3);
            mma_tf32(cross[nt][1], hg.z, hh.z, hg.w, hh.w, w2, w3);
          }
        }
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][e] += h4[nt][e];
      }
      float p[2][4];
      const bool masked = j0 + kKvChunk > open;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[nt][e] = __fmul_rn(__fadd_rn(s[nt][e], __fadd_rn(cross[nt][0][e], cross[nt][1][e])), a.c);
          if (masked) {
            const int j = j0 + nt * 8 + 2 * t + (e & 1);
            if (j >= x.keys || !kv_sees<MASK>(a, x, g + (e >> 1) * 8, j)) p[nt][e] = -INFINITY;
          }
        }
      if (SCORES) {
        float* sc = a.scores + ((size_t)x.b * a.hkv + x.hk) * x.nrows * (size_t)a.score_stride + j0 + 2 * t;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          if (g < x.nrows)
            *reinterpret_cast<float2*>(sc + (size_t)g * a.score_stride + nt * 8) = make_float2(p[nt][0], p[nt][1]);
          if (g + 8 < x.nrows)
            *reinterpret_cast<float2*>(sc + (size_t)(g + 8) * a.score_stride + nt * 8) =
                make_float2(p[nt][2], p[nt][3]);
        }
      }
      float x0 = fmaxf(fmaxf(p[0][0], p[0][1]), fmaxf(p[1][0], p[1][1]));
      float x1 = fmaxf(fmaxf(p[0][2], p[0][3]), fmaxf(p[1][2], p[1][3]));
      x0 = fmaxf(x0, __shfl_xor_sync(kFull, x0, 1));
      x1 = fmaxf(x1, __shfl_xor_sync(kFull, x1, 1));
      x0 = fmaxf(x0, __shfl_xor_sync(kFull, x0, 2));
      x1 = fmaxf(x1, __shfl_xor_sync(kFull, x1, 2));
      const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
      const float b0 = n0 == -INFINITY ? 0.0f : n0, b1 = n1 == -INFINITY ? 0.0f : n1;
      const float f0 = exp2f(m0 - b0), f1 = exp2f(m1 - b1);
      m0 = n0;
      m1 = n1;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        p[nt][0] = exp2f(p[nt][0] - b0);
        p[nt][1] = exp2f(p[nt][1] - b0);
        p[nt][2] = exp2f(p[nt][2] - b1);
        p[nt][3] = exp2f(p[nt][3] - b1);
      }
      l0 = l0 * f0 + ((p[0][0] + p[0][1]) + (p[1][0] + p[1][1]));
      l1 = l1 * f1 + ((p[0][2] + p[0][3]) + (p[1][2] + p[1][3]));
      // a value row that is not finite must not reach the rows that do not see it (0 * inf):
      // such a chunk, only where a mask is at work, takes the exact loop below
      bool odd = false;
      if (masked) {
        for (int r = 0; r < kKvChunk; ++r) {
          const float4 w = lds_f4(vst + r * (kKvD * 4) + lane * 16);
          odd |= !(fabsf(w.x) <= 3.402823466e38f && fabsf(w.y) <= 3.402823466e38f && fabsf(w.z) <= 3.402823466e38f &&
                   fabsf(w.w) <= 3.402823466e38f);
        }
        odd = __any_sync(kFull, odd);
      }
      if (!odd) {
        // output: a lane takes keys 8 nt + 2t, 2t + 1 and dimensions 32 w + 4 g + e; the chunk's
        // sum starts from 0 and joins the running one with rounding
        uint32_t ph[2][4], pl[2][4];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          split_tf32(p[nt][0], ph[nt][0], pl[nt][0]);
          split_tf32(p[nt][2], ph[nt][1], pl[nt][1]);
          split_tf32(p[nt][1], ph[nt][2], pl[nt][2]);
          split_tf32(p[nt][3], ph[nt][3], pl[nt][3]);
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          float d[4][4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int y = 0; y < 4; ++y) d[e][y] = 0.0f;
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            const int r0 = nt * 8 + 2 * t;  // r0 and r0 + 1 have the same swizzle
            const uint32_t at = vst + r0 * (kKvD * 4) + (((w * 8 + g) ^ (((r0 >> 1) & 3) << 1)) << 4);
            const float4 va = lds_f4(at), vb4 = lds_f4(at + kKvD * 4);
            const float av[4] = {va.x, va.y, va.z, va.w}, bv[4] = {vb4.x, vb4.y, vb4.z, vb4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t ah, al, bh, bl;
              split_tf32(av[e], ah, al);
              split_tf32(bv[e], bh, bl);
              mma_tf32(d[e], pl[nt][0], pl[nt][1], pl[nt][2], pl[nt][3], ah, bh);
              mma_tf32(d[e], ph[nt][0], ph[nt][1], ph[nt][2], ph[nt][3], al, bl);
              mma_tf32(d[e], ph[nt][0], ph[nt][1], ph[nt][2], ph[nt][3], ah, bh);
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            o[w * 4 + e][0] = fmaf(o[w * 4 + e][0], f0, d[e][0]);
            o[w * 4 + e][1] = fmaf(o[w * 4 + e][1], f0, d[e][1]);
            o[w * 4 + e][2] = fmaf(o[w * 4 + e][2], f1, d[e][2]);
            o[w * 4 + e][3] = fmaf(o[w * 4 + e][3], f1, d[e][3]);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          o[i][0] *= f0;
          o[i][1] *= f0;
          o[i][2] *= f1;
          o[i][3] *= f1;
        }
#pragma unroll
        for (int r = 0; r < kKvChunk; ++r) {
          const int src = (lane & ~3) | ((r & 7) >> 1);
          const float pa = __shfl_sync(kFull, p[r >> 3][r & 1], src);
          const float pb = __shfl_sync(kFull, p[r >> 3][2 + (r & 1)], src);
#pragma unroll
          for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int y = 0; y < 2; ++y) {  // accumulator columns 2t + y: dimensions 32 w + 4 (2t + y) + e
              const float4 q4 = lds_f4(vst + r * (kKvD * 4) + (((w * 8 + 2 * t + y) ^ (((r >> 1) & 3) << 1)) << 4));
              const float vv[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (pa != 0.0f) o[w * 4 + e][y] = fmaf(pa, vv[e], o[w * 4 + e][y]);
                if (pb != 0.0f) o[w * 4 + e][2 + y] = fmaf(pb, vv[e], o[w * 4 + e][2 + y]);
              }
            }
        }
      }
      __syncwarp();  // the stage is free
      if (c + kKvStages * kKvWarps < c1) load(c + kKvStages * kKvWarps, stage);
      cp_async_commit();
    }
    cp_async_wait(0);

    // the warps' parts, merged in warp order
    if (tid < x.nrows) sm.ok[tid] = kv_row_valid<MASK>(a, x, tid);
    l0 += __shfl_xor_sync(kFull, l0, 1);
    l1 += __shfl_xor_sync(kFull, l1, 1);
    l0 += __shfl_xor_sync(kFull, l0, 2);
    l1 += __shfl_xor_sync(kFull, l1, 2);
    if (t == 0) {
      sm.m[warp][g] = m0;
      sm.m[warp][g + 8] = m1;
      sm.l[warp][g] = l0;
      sm.l[warp][g + 8] = l1;
    }
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int d = 32 * w + 4 * (2 * t + y);
        *reinterpret_cast<float4*>(&sm.o[warp][g][d]) =
            make_float4(o[w * 4][y], o[w * 4 + 1][y], o[w * 4 + 2][y], o[w * 4 + 3][y]);
        *reinterpret_cast<float4*>(&sm.o[warp][g + 8][d]) =
            make_float4(o[w * 4][2 + y], o[w * 4 + 1][2 + y], o[w * 4 + 2][2 + y], o[w * 4 + 3][2 + y]);
      }
    __syncthreads();
    const bool whole = off == 0 && c1 == x.chunks;
    const size_t slot = a.split ? (size_t)blockIdx.x + u : (size_t)u;
    for (int r = 0; r < x.nrows; ++r) {
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kKvWarps; ++w) M = fmaxf(M, sm.m[w][r]);
      if (!sm.ok[r]) M = -INFINITY;
      float L = 0.0f, A = 0.0f;
      if (M != -INFINITY) {
#pragma unroll
        for (int w = 0; w < kKvWarps; ++w) {
          const float f = exp2f(sm.m[w][r] - M);
          if (f != 0.0f) {  // an empty part's sums are 0, and stay out
            L = fmaf(sm.l[w][r], f, L);
            A = fmaf(sm.o[w][r][tid], f, A);
          }
        }
      }
      if (whole)
        a.out[kv_row_offset<MASK>(a, x, r) + tid] = L > 0.0f ? __fdiv_rn(A, L) : (M == -INFINITY ? 0.0f : A / L);
      else
        a.acc[slot * kKvSlotFloats + r * kKvD + tid] = A;
      if (tid == 0 && a.stat) {
        a.stat[slot * 32 + r] = M;
        a.stat[slot * 32 + 16 + r] = L;
      }
      if (tid == 0 && a.lse && whole)
        a.lse[((size_t)x.b * a.hkv + x.hk) * a.n * a.group + x.r0 + r] = M == -INFINITY ? INFINITY : M + log2f(L);
    }
    left -= c1 - off;
    off = 0;
    ++u;
    if (!a.split) break;
    __syncthreads();  // sm.q, sm.o are free
  }
}

// Merge of the parts of every unit (one CTA per unit), and the weights of the keys where
// the scores were stored: weight[j] += sum over the rows of 2^(s_j - log2 sum).
// grid (units, key ranges): range 0 merges, every range adds its keys' weights.
constexpr int kKvWeightKeys = 1024;
template <int MASK, bool SCORES>
__global__ void __launch_bounds__(kKvThreads) kv_merge_kernel(const KvArgs a, float* __restrict__ weight) {
  __shared__ int red[kKvWarps][2];
  __shared__ float lse[kKvRows];
  const int tid = threadIdx.x, u = blockIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  const KvUnit x = kv_unit<MASK>(a, u);
  size_t slot0 = u;
  int parts = 1;
  if (a.split) {
    int before = 0, total = 0;
    for (int i = tid; i < a.units; i += kKvThreads) {
      const int c = kv_unit<MASK>(a, i).chunks;
      total += c;
      if (i < u) before += c;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      total += __shfl_xor_sync(kFull, total, o);
      before += __shfl_xor_sync(kFull, before, o);
    }
    if ((tid & 31) == 0) {
      red[tid >> 5][0] = total;
      red[tid >> 5][1] = before;
    }
    __syncthreads();
    total = before = 0;
    for (int w = 0; w < kKvWarps; ++w) {
      total += red[w][0];
      before += red[w][1];
    }
    const int quota = max((total + kKvGrid - 1) / kKvGrid, kKvWarps);
    const int c0 = before / quota, c1 = x.chunks > 0 ? (before + x.chunks - 1) / quota : c0 - 1;
    slot0 = (size_t)c0 + u;
    parts = c1 - c0 + 1;
  }
  if (x.chunks == 0) {  // no CTA came by
    if (blockIdx.y == 0)
      for (int r = 0; r < x.nrows; ++r) {
        a.out[kv_row_offset<MASK>(a, x, r) + tid] = 0.0f;
        if (a.lse && tid == 0) a.lse[((size_t)x.b * a.hkv + x.hk) * a.n * a.group + x.r0 + r] = INFINITY;
      }
    return;
  }
  if (!SCORES && parts == 1) return;
  const bool merge = blockIdx.y == 0 && parts > 1;
  for (int r = 0; r < x.nrows; ++r) {
    float M = -INFINITY;
    for (int s = 0; s < parts; ++s) M = fmaxf(M, a.stat[(slot0 + s) * 32 + r]);
    float L = 0.0f, A = 0.0f;
    if (M != -INFINITY)
      for (int s = 0; s < parts; ++s) {
        const float f = exp2f(a.stat[(slot0 + s) * 32 + r] - M);
        if (f != 0.0f) {
          L = fmaf(a.stat[(slot0 + s) * 32 + 16 + r], f, L);
          if (merge) A = fmaf(a.acc[(slot0 + s) * kKvSlotFloats + r * kKvD + tid], f, A);
        }
      }
    if (merge) a.out[kv_row_offset<MASK>(a, x, r) + tid] = M == -INFINITY ? 0.0f : __fdiv_rn(A, L);
    if (tid == 0) {
      const float z = M == -INFINITY ? INFINITY : M + log2f(L);
      lse[r] = z;
      if (a.lse && merge) a.lse[((size_t)x.b * a.hkv + x.hk) * a.n * a.group + x.r0 + r] = z;
    }
  }
  if (SCORES) {
    __syncthreads();
    const int j1 = min(x.keys, ((int)blockIdx.y + 1) * kKvWeightKeys);
    const size_t bh = (size_t)x.b * a.hkv + x.hk;
    for (int j = blockIdx.y * kKvWeightKeys + tid; j < j1; j += kKvThreads) {
      float w = 0.0f;
      for (int r = 0; r < x.nrows; ++r)
        if (lse[r] != INFINITY) w += exp2f(a.scores[(bh * x.nrows + r) * a.score_stride + j] - lse[r]);
      weight[bh * a.max_t + j] += w;
    }
  }
}

// Column sums of the softmax where the scores were not stored: every score once more, from
// the rows' log2 sums.  grid (64-key tiles, batch * hkv), a warp holds 16 keys' fragments
// and goes over the 16-row groups; sums per lane, then over the lanes of a key.
struct KvColSmem {
  alignas(16) float k[kKvWarps * kKvChunk][kKvD];
  alignas(16) float q[2][kKvRows][kKvD];
  float lse[2][kKvRows];
};
__global__ void __launch_bounds__(kKvThreads, 1) kv_column_kernel(const KvArgs a, float* __restrict__ weight) {
  extern __shared__ __align__(16) uint8_t kv_smem[];
  KvColSmem& sm = *reinterpret_cast<KvColSmem*>(kv_smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.y / a.hkv, hk = blockIdx.y - b * a.hkv;
  const int p = a.pos[b], rows = a.n * a.group;
  const int keys = (p < 0 || p >= a.max_t) ? 0 : min(p + a.n, a.max_t);
  const int j0 = blockIdx.x * (kKvWarps * kKvChunk);
  if (j0 >= keys) return;
  const size_t bh = (size_t)b * a.hkv + hk;
  const float* kb = a.k + bh * (size_t)a.max_t * kKvD;
  const uint32_t ks = (uint32_t)__cvta_generic_to_shared(&sm.k[0][0]);
  const uint32_t qs = (uint32_t)__cvta_generic_to_shared(&sm.q[0][0][0]);
  const int i_first = max(0, j0 - p);  // the first token that sees a key of the tile
  const int rg0 = (int)(((int64_t)i_first * a.group) / kKvRows);
  auto load_q = [&](int rg, int buf) {
    for (int e = tid; e < kKvRows * 32; e += kKvThreads) {
      const int r = e >> 5, ch = e & 31, row = rg * kKvRows + r;
      const bool there = row < rows;
      const int i = there ? row / a.group : 0, h = hk * a.group + (there ? row - i * a.group : 0);
      cp_async16_zfill(qs + buf * (kKvRows * kKvD * 4) + r * (kKvD * 4) + ((ch ^ ((r & 1) << 2)) << 4),
                       a.q + (((size_t)b * a.n + i) * a.hq + h) * kKvD + ch * 4, there);
    }
    if (tid < kKvRows) {
      const int row = rg * kKvRows + tid;
      sm.lse[buf][tid] = row < rows ? a.lse[bh * rows + row] : INFINITY;
    }
    cp_async_commit();
  };
  for (int e = tid; e < kKvWarps * kKvChunk * 32; e += kKvThreads) {
    const int r = e >> 5, ch = e & 31, j = j0 + r;
    cp_async16_zfill(ks + r * (kKvD * 4) + ((ch ^ ((r & 1) << 2)) << 4), kb + (size_t)(j < keys ? j : 0) * kKvD + ch * 4,
                     j < keys);
  }
  load_q(rg0, 0);
  cp_async_wait(0);
  __syncthreads();
  uint32_t kh[8][2][4], kl[8][2][4];
#pragma unroll
  for (int pair = 0; pair < 8; ++pair)
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      const int r = warp * kKvChunk + nt * 8 + g;
      const float4 kv = lds_f4(ks + r * (kKvD * 4) + (((pair * 4 + t) ^ ((r & 1) << 2)) << 4));
      split_tf32(kv.x, kh[pair][nt][0], kl[pair][nt][0]);
      split_tf32(kv.y, kh[pair][nt][1], kl[pair][nt][1]);
      split_tf32(kv.z, kh[pair][nt][2], kl[pair][nt][2]);
      split_tf32(kv.w, kh[pair][nt][3], kl[pair][nt][3]);
    }
  float sum[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
  const int rgs = (rows + kKvRows - 1) / kKvRows;
  for (int rg = rg0; rg < rgs; ++rg) {
    const int buf = (rg - rg0) & 1;
    if (rg + 1 < rgs) load_q(rg + 1, buf ^ 1);
    float s[2][3][4];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int z = 0; z < 3; ++z)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][z][e] = 0.0f;
#pragma unroll
    for (int pair = 0; pair < 8; ++pair) {
      const uint32_t at = qs + buf * (kKvRows * kKvD * 4) + g * (kKvD * 4) + (((pair * 4 + t) ^ ((g & 1) << 2)) << 4);
      const float4 qa = lds_f4(at), qb = lds_f4(at + 8 * kKvD * 4);
      uint32_t ah[4], al[4], bh4[4], bl4[4];
      split_tf32(qa.x, ah[0], al[0]);
      split_tf32(qa.y, ah[1], al[1]);
      split_tf32(qa.z, ah[2], al[2]);
      split_tf32(qa.w, ah[3], al[3]);
      split_tf32(qb.x, bh4[0], bl4[0]);
      split_tf32(qb.y, bh4[1], bl4[1]);
      split_tf32(qb.z, bh4[2], bl4[2]);
      split_tf32(qb.w, bh4[3], bl4[3]);
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int h = 0; h < 4; h += 2) {
          mma_tf32(s[nt][0], ah[h], bh4[h], ah[h + 1], bh4[h + 1], kh[pair][nt][h], kh[pair][nt][h + 1]);
          mma_tf32(s[nt][1], al[h], bl4[h], al[h + 1], bl4[h + 1], kh[pair][nt][h], kh[pair][nt][h + 1]);
          mma_tf32(s[nt][2], ah[h], bh4[h], ah[h + 1], bh4[h + 1], kl[pair][nt][h], kl[pair][nt][h + 1]);
        }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = g + 8 * half, row = rg * kKvRows + r;
      const float z = sm.lse[buf][r];
      const int last = p + row / a.group;  // rows past the cache have an infinite sum
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = j0 + warp * kKvChunk + nt * 8 + 2 * t + e;
          const float v = s[nt][0][half * 2 + e] + (s[nt][1][half * 2 + e] + s[nt][2][half * 2 + e]);
          if (j <= last && z != INFINITY) sum[nt][e] += exp2f(__fmul_rn(v, a.c) - z);
        }
    }
    cp_async_wait(0);
    __syncthreads();
  }
#pragma unroll
  for (int nt = 0; nt < 2; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float v = sum[nt][e];
      v += __shfl_xor_sync(kFull, v, 4);
      v += __shfl_xor_sync(kFull, v, 8);
      v += __shfl_xor_sync(kFull, v, 16);
      const int j = j0 + warp * kKvChunk + nt * 8 + 2 * t + e;
      if (g == 0 && j < keys) weight[bh * a.max_t + j] += v;
    }
}

// RoPE and append of a tree: one CTA per (sequence, node).  The node's path to the context is
// found by pointer doubling over the parents of its sequence (all nodes at once, log2(depth)
// rounds): jump[i] the ancestor 2^k above, path[i] the bits of the nodes from i up to it.
// jump ends at -1 (the context) or, where a parent is not below its node, at -2: such a node
// and everything under it is no row of the tree (nothing written, no bit set).
__global__ void __launch_bounds__(kKvMaxTree)
rope_tree_kernel(const float* __restrict__ qkv, const int* __restrict__ parents, const int* __restrict__ pos_dev,
                 const float* __restrict__ cos_t, const float* __restrict__ sin_t, float* __restrict__ kc,
                 float* __restrict__ vc, int n, int words, int hq, int hkv, int max_t, float* __restrict__ q_out,
                 uint32_t* __restrict__ anc) {
  __shared__ int jump[2][kKvMaxTree];
  __shared__ uint32_t path[2][kKvMaxTree][kKvMaxTree / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.y, i = blockIdx.x, tid = threadIdx.x;
  const int pos = pos_dev[b];
  const bool in = pos >= 0 && pos < max_t - i;
  const int m = i + 1;  // a path holds no node above its own number
  if (tid < m) {
    const int par = parents[(size_t)b * n + tid];
    jump[0][tid] = par >= -1 && par < tid ? par : -2;
    for (int w = 0; w < words; ++w) path[0][tid][w] = w == (tid >> 5) ? 1u << (tid & 31) : 0u;
  }
  int cur = 0;
  for (;;) {
    const int more = __syncthreads_or(tid < m && jump[cur][tid] >= 0);
    if (!more) break;
    if (tid < m) {
      const int to = jump[cur][tid];
      for (int w = 0; w < words; ++w)
        path[cur ^ 1][tid][w] = path[cur][tid][w] | (to >= 0 ? path[cur][to][w] : 0u);
      jump[cur ^ 1][tid] = to >= 0 ? jump[cur][to] : to;
    }
    cur ^= 1;
  }
  const bool node = in && jump[cur][i] == -1;
  int depth = -1;
  for (int w = 0; w < words; ++w) depth += __popc(path[cur][i][w]);
  if (tid < words) anc[((size_t)b * n + i) * words + tid] = node ? path[cur][i][tid] : 0u;
  const size_t row = (size_t)b * n + i;
  const int half = kKvD / 2, h4 = half / 4, d4 = kKvD / 4;
  float4* qo = reinterpret_cast<float4*>(q_out + row * hq * kKvD);
  if (!node) {
    for (int it = tid; it < hq * d4; it += blockDim.x) qo[it] = make_float4(0.f, 0.f, 0.f, 0.f);
    return;
  }
  const float4* xr = reinterpret_cast<const float4*>(qkv + row * (hq + 2 * hkv) * kKvD);
  const float4* c4 = reinterpret_cast<const float4*>(cos_t + (size_t)(pos + depth) * half);
  const float4* s4 = reinterpret_cast<const float4*>(sin_t + (size_t)(pos + depth) * half);
  for (int it = tid; it < (hq + hkv) * h4; it += blockDim.x) {
    const int head = it / h4, j = it - head * h4;
    const float4 x = xr[head * d4 + j], y = xr[head * d4 + h4 + j];
    const float4 c = __ldg(c4 + j), s = __ldg(s4 + j);
    const float4 lo = make_float4(__fadd_rn(__fmul_rn(x.x, c.x), __fmul_rn(y.x, -s.x)),
                                  __fadd_rn(__fmul_rn(x.y, c.y), __fmul_rn(y.y, -s.y)),
                                  __fadd_rn(__fmul_rn(x.z, c.z), __fmul_rn(y.z, -s.z)),
                                  __fadd_rn(__fmul_rn(x.w, c.w), __fmul_rn(y.w, -s.w)));
    const float4 hi = make_float4(__fadd_rn(__fmul_rn(y.x, c.x), __fmul_rn(x.x, s.x)),
                                  __fadd_rn(__fmul_rn(y.y, c.y), __fmul_rn(x.y, s.y)),
                                  __fadd_rn(__fmul_rn(y.z, c.z), __fmul_rn(x.z, s.z)),
                                  __fadd_rn(__fmul_rn(y.w, c.w), __fmul_rn(x.w, s.w)));
    float4* dst = head < hq
                      ? qo + head * d4
                      : reinterpret_cast<float4*>(kc + (((size_t)b * hkv + (head - hq)) * max_t + pos + i) * kKvD);
    dst[j] = lo;
    dst[h4 + j] = hi;
  }
  for (int it = tid; it < hkv * d4; it += blockDim.x) {
    const int hv = it / d4, j = it - hv * d4;
    reinterpret_cast<float4*>(vc + (((size_t)b * hkv + hv) * max_t + pos + i) * kKvD)[j] = xr[(hq + hkv + hv) * d4 + j];
  }
}

cudaLaunchConfig_t kv_cfg(dim3 grid, dim3 block, size_t smem, cudaStream_t s, cudaLaunchAttribute* attr) {
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

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

int tree_words(int n) { return (n + 31) / 32; }

// Rows of `rows` and units, and the parts of the workspace the core needs.
struct KvPlan {
  int rgs = 1;
  int64_t units = 0;
  bool split = false;
  size_t slots = 0;
};
KvPlan kv_plan(int64_t lists, int64_t rows_per_list) {
  KvPlan p;
  p.rgs = (int)((rows_per_list + kKvRows - 1) / kKvRows);
  p.units = lists * p.rgs;
  // with two units per SM and more the units themselves fill the GPU
  p.split = p.units < 2 * kKvGrid;
  p.slots = p.split ? (size_t)(kKvGrid + p.units) : (size_t)p.units;
  return p;
}
size_t core_bytes(const KvPlan& p, bool stat) {
  return (p.split ? up256(p.slots * kKvSlotFloats * 4) : 0) + (p.split || stat ? up256(p.slots * 32 * 4) : 0);
}
// Sets the core's part of the workspace; returns the bytes it takes.
size_t core_place(KvArgs& a, const KvPlan& p, bool stat, uint8_t* ws) {
  size_t o = 0;
  if (p.split) {
    a.acc = reinterpret_cast<float*>(ws);
    o += up256(p.slots * kKvSlotFloats * 4);
  }
  if (p.split || stat) {
    a.stat = reinterpret_cast<float*>(ws + o);
    o += up256(p.slots * 32 * 4);
  }
  a.rgs = p.rgs;
  a.units = (int)p.units;
  a.split = p.split ? 1 : 0;
  return o;
}

template <int MASK, bool SCORES>
cudaError_t launch_core(const KvArgs& a, float* weight, int device, cudaStream_t s) {
  static int configured[128] = {0};
  cudaError_t e =
      ensure_smem((const void*)kv_attention_kernel<MASK, SCORES>, configured, device, sizeof(KvSmem), false);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = kv_cfg(dim3((unsigned)(a.split ? kKvGrid : a.units)), dim3(kKvThreads), sizeof(KvSmem), s, attr);
  e = cudaLaunchKernelEx(&cfg, kv_attention_kernel<MASK, SCORES>, a);
  if (e != cudaSuccess || (!a.split && !SCORES)) return e;
  const unsigned ranges = SCORES ? (unsigned)((a.max_t + kKvWeightKeys - 1) / kKvWeightKeys) : 1u;
  cfg = kv_cfg(dim3((unsigned)a.units, ranges), dim3(kKvThreads), 0, s, attr);
  return cudaLaunchKernelEx(&cfg, kv_merge_kernel<MASK, SCORES>, a, weight);
}

KvArgs kv_args(const float* q, const float* kc, const float* vc, const int* pos, int batch, int n, int hq, int hkv,
               int max_t, float* out) {
  KvArgs a = {};
  a.q = q;
  a.k = kc;
  a.v = vc;
  a.pos = pos;
  a.out = out;
  a.batch = batch;
  a.n = n;
  a.hq = hq;
  a.hkv = hkv;
  a.group = hq / hkv;
  a.max_t = max_t;
  // scores / sqrt(128) as the other attention kernels: times the f32 rounding of 1/sqrt(128)
  a.c = (float)((double)(float)(1.0 / std::sqrt(128.0)) * 1.4426950408889634);
  return a;
}

bool weights_stored(int n, int group) { return (int64_t)n * group <= kKvRows; }
int score_stride(int max_t) { return (max_t + kKvChunk - 1) / kKvChunk * kKvChunk; }

}  // namespace

size_t attention_tree_workspace_bytes(int batch, int n, int hq, int hkv) {
  const KvPlan p = kv_plan((int64_t)batch * hkv, (int64_t)n * (hq / hkv));
  return up256((size_t)batch * n * hq * kKvD * 4) + up256((size_t)batch * n * tree_words(n) * 4) + core_bytes(p, false);
}

cudaError_t launch_rope_attention_tree(const float* qkv, const int* parents, const int* pos, const float* cos_t,
                                       const float* sin_t, float* kc, float* vc, int batch, int n, int hq, int hkv,
                                       int max_t, void* ws, float* out, int device, cudaStream_t s) {
  uint8_t* w = static_cast<uint8_t*>(ws);
  float* q = reinterpret_cast<float*>(w);
  w += up256((size_t)batch * n * hq * kKvD * 4);
  uint32_t* anc = reinterpret_cast<uint32_t*>(w);
  w += up256((size_t)batch * n * tree_words(n) * 4);
  KvArgs a = kv_args(q, kc, vc, pos, batch, n, hq, hkv, max_t, out);
  a.anc = anc;
  a.words = tree_words(n);
  core_place(a, kv_plan((int64_t)batch * hkv, (int64_t)n * a.group), false, w);
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = kv_cfg(dim3((unsigned)n, (unsigned)batch), dim3(kKvMaxTree), 0, s, attr);
  cudaError_t e = cudaLaunchKernelEx(&cfg, rope_tree_kernel, qkv, parents, pos, cos_t, sin_t, kc, vc, n, a.words, hq,
                                     hkv, max_t, q, anc);
  if (e != cudaSuccess) return e;
  return launch_core<kMaskTree, false>(a, nullptr, device, s);
}

size_t attention_weights_workspace_bytes(int batch, int n, int hq, int hkv, int max_t) {
  const int group = hq / hkv;
  const KvPlan p = kv_plan((int64_t)batch * hkv, (int64_t)n * group);
  const bool stored = weights_stored(n, group);
  return core_bytes(p, stored) + (stored ? up256((size_t)batch * hq * n * score_stride(max_t) * 4)
                                         : up256((size_t)batch * hq * n * 4));
}

cudaError_t launch_attention_weights(const float* q, const float* kc, const float* vc, const int* pos, int batch, int n,
                                     int hq, int hkv, int max_t, float* weight, void* ws, float* out, int device,
                                     cudaStream_t s) {
  KvArgs a = kv_args(q, kc, vc, pos, batch, n, hq, hkv, max_t, out);
  const bool stored = weights_stored(n, a.group);
  uint8_t* w = static_cast<uint8_t*>(ws);
  w += core_place(a, kv_plan((int64_t)batch * hkv, (int64_t)n * a.group), stored, w);
  if (stored) {
    a.scores = reinterpret_cast<float*>(w);
    a.score_stride = score_stride(max_t);
    return launch_core<kMaskCausal, true>(a, weight, device, s);
  }
  a.lse = reinterpret_cast<float*>(w);
  cudaError_t e = launch_core<kMaskCausal, false>(a, weight, device, s);
  if (e != cudaSuccess) return e;
  static int configured[128] = {0};
  e = ensure_smem((const void*)kv_column_kernel, configured, device, sizeof(KvColSmem), false);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  constexpr int tile = kKvWarps * kKvChunk;
  cudaLaunchConfig_t cfg = kv_cfg(dim3((unsigned)((max_t + tile - 1) / tile), (unsigned)(batch * hkv)),
                                  dim3(kKvThreads), sizeof(KvColSmem), s, attr);
  return cudaLaunchKernelEx(&cfg, kv_column_kernel, a, weight);
}

size_t attention_blocks_workspace_bytes(int batch, int n, int hq, int hkv) {
  return up256(core_bytes(kv_plan((int64_t)batch * n * hkv, hq / hkv), false) + 1);  // never 0: it may be allocated
}

cudaError_t launch_attention_blocks(const float* q, const float* kc, const float* vc, const int* pos, const int* index,
                                    int batch, int n, int hq, int hkv, int max_t, int block, int topk, void* ws,
                                    float* out, int device, cudaStream_t s) {
  KvArgs a = kv_args(q, kc, vc, pos, batch, n, hq, hkv, max_t, out);
  a.index = index;
  a.block = block;
  a.topk = topk;
  core_place(a, kv_plan((int64_t)batch * n * hkv, a.group), false, static_cast<uint8_t*>(ws));
  return launch_core<kMaskBlocks, false>(a, nullptr, device, s);
}

}  // namespace q8lin
