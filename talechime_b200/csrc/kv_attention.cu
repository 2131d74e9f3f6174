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
// numbered r = i * group + head-in-group and taken 8 or 16 at a time (a unit).
//
// Products: f32 operands as tf32 pairs on the tensor cores (mma.sync m16n8k8).  x = hi + lo
// with hi = x rounded to tf32's 11 significant bits and lo = x - hi (exact) cut to them, and
// a.b = hi.hi + lo.hi + hi.lo: what is dropped (lo.lo and lo's cut) is below 9 * 2^-24 of each
// product, on average f32's own rounding; f32's exponent range stays.
#include <cmath>

#include "common.cuh"
#include "internal.h"
#include "kv_core.cuh"

namespace q8lin {

namespace {

__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t a0, const uint32_t a1, const uint32_t a2,
                                         const uint32_t a3, const uint32_t b0, const uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The tensor cores read the upper 19 bits of a tf32 operand: lo goes in as it is and is cut there.
// (Integer rounding of hi, one operation each: cvt.rna.tf32 took the 16-row kernel from 70 to 79 us
// at 16 K rows x 16 heads, cutting lo here too cost 8 % of it.)
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(__fsub_rn(x, __uint_as_float(hi)));
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

constexpr int kKvList = 512;  // chosen blocks of a row held in shared memory; longer lists are read where they are
template <int NT, int W>
struct KvSmem {
  // each warp's ring of half chunks; after a unit's last chunk its output part [row][132]
  alignas(16) uint8_t ring[W][kKvSlots][kKvHalf];
  // the unit's query rows as MMA fragments: [hi, lo][16 dimensions][8 rows][lane]
  alignas(16) float4 q[2][8][NT][32];
  alignas(16) float p[W][NT][kKvChunk][8];  // a chunk's probabilities
  float m[W][8 * NT], l[W][8 * NT];
  float f[W][8 * NT];
  float M[8 * NT], L[8 * NT];
  KvFind find;
  int list[kKvList];
};

// The rows are the N side of the products and the keys, then the dimensions, the M side, so
// that 8 rows fill a tile: S^T = K Q^T and O^T = V^T P^T.  In an m16n8k8 fragment lane 4g + t
// holds rows g and g + 8 of A, column g of B, and columns 2t, 2t + 1 of the result.
//
// What bounds it: with up to 16 rows a kv head the cache's bytes, read once; the tf32 split of
// every key and value (4 operations each) and the products run beside the copies.
// (16 rows over 16 K keys x 16 heads 55 us, 4.8 TB/s with the tensor pipe 47 % busy; one token
// of 8 sequences over 8 K keys x 16 heads, weights' scores written, 164 us, 5.9 TB/s.  Rows over
// chosen blocks read them from the L2: 512 tokens x 17 blocks of 64 165 us, 6.9 TB/s of it.)
//
// W warps: 8 on an SM, or with 8 rows and whole units 4, twice on an SM, so that one CTA's start
// and end run beside the other's keys.  (8 against 4 warps: 512 units of 300 keys 59.6 and 44.5 us,
// of 1000 keys 110.5 and 98.0; 1024 units of 2000 keys 329 and 326; 512 tokens that attend over
// chosen blocks 203 and 186.  16 rows do not fit twice.)
template <int MASK, bool SCORES, int NT, int W>
__global__ void __launch_bounds__(W * 32, W == 4 ? 2 : 1) kv_attention_kernel(const KvArgs a) {
  constexpr int kThreads = W * 32;
  extern __shared__ __align__(16) uint8_t kv_smem[];
  KvSmem<NT, W>& sm = *reinterpret_cast<KvSmem<NT, W>*>(kv_smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  pdl_wait();
  pdl_launch_dependents();  // the merge waits for this grid before it reads anything

  int u, off, left;  // left: chunks to take
  if (a.split) {
    left = kv_find<MASK, kThreads>(a, sm.find, blockIdx.x);
    u = sm.find.unit;
    off = sm.find.off;
  } else {
    u = a.units - 1 - (int)blockIdx.x;  // later rows see more keys: longest first
    off = 0;
    left = 0x7fffffff;
  }
  const int quota = a.split ? sm.find.quota : left;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(&sm.ring[warp][0][0]);

  while (u < a.units && left > 0) {
    const KvUnit x = kv_unit<MASK>(a, u);
    const int c1 = min(x.chunks, off > x.chunks - left ? x.chunks : off + left);
    const float* kb = a.k + ((size_t)x.b * a.hkv + x.hk) * (size_t)a.max_t * kKvD;
    const float* vb = a.v + ((size_t)x.b * a.hkv + x.hk) * (size_t)a.max_t * kKvD;

    const int* list = nullptr;
    if (MASK == kMaskBlocks) {
      list = a.index + (((size_t)x.b * a.n + x.i0) * a.hkv + x.hk) * a.topk;
      if (x.picked <= kKvList) {
        for (int e = tid; e < x.picked; e += kThreads) sm.list[e] = list[e];
        __syncthreads();
        list = sm.list;
      }
    }
    // this warp's chunks: off + warp, off + warp + W, ...  Half h of its stream: the keys
    // (h even) or values of its chunk h / 2, copied into ring slot h % 3.
    const int c0 = off + warp;
    const int halves = c0 < c1 ? 2 * ((c1 - c0 + W - 1) / W) : 0;
    auto load = [&](int h, int slot) {
      if (h < halves) {
        const int j0 = kv_chunk_key<MASK>(a, x, list, c0 + (h >> 1) * W);
        const bool val = h & 1;
        const float* src = (val ? vb : kb) + (size_t)j0 * kKvD + lane * 4;
        const uint32_t dst = ring + slot * kKvHalf;
        const bool plain = j0 + kKvChunk <= (MASK == kMaskTree ? x.p : x.keys);
        if (plain) {
#pragma unroll
          for (int r = 0; r < kKvChunk; ++r)
            cp_async16(dst + r * (kKvD * 4) + ((lane ^ (val ? (r & 3) << 1 : (r & 1) << 2)) << 4), src + r * kKvD);
        } else {
          const uint32_t rows = kv_rows_there<MASK>(a, x, j0);
#pragma unroll 4
          for (int r = 0; r < kKvChunk; ++r) {
            const bool there = (rows >> r) & 1u;
            cp_async16_zfill(dst + r * (kKvD * 4) + ((lane ^ (val ? (r & 3) << 1 : (r & 1) << 2)) << 4),
                             there ? src + r * kKvD : kb, there);
          }
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int h = 0; h < kKvSlots; ++h) load(h, h);
    // query rows -> fragments
    for (int e = tid; e < 8 * NT * 32; e += kThreads) {
      const int ln = e & 31, nt = (e >> 5) % NT, pair = (e >> 5) / NT;
      const int r = (ln >> 2) + 8 * nt;
      float4 qv = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < x.nrows)
        qv = *reinterpret_cast<const float4*>(a.q + kv_row_offset<MASK>(a, x, r) + pair * 16 + (ln & 3) * 4);
      uint4 h, w;
      split_tf32(qv.x, h.x, w.x);
      split_tf32(qv.y, h.y, w.y);
      split_tf32(qv.z, h.z, w.z);
      split_tf32(qv.w, h.w, w.w);
      *reinterpret_cast<uint4*>(&sm.q[0][pair][nt][ln]) = h;
      *reinterpret_cast<uint4*>(&sm.q[1][pair][nt][ln]) = w;
    }
    __syncthreads();

    // the first key some row of the unit does not see (chunks below it need no mask)
    const int open = MASK == kMaskTree ? x.p : MASK == kMaskCausal ? x.p + x.i0 + 1 : x.keys;
    float o[NT][8][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.0f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.0f;
    }

    int slot = 0;
    for (int h = 0; h < halves; h += 2) {
      const int j0 = kv_chunk_key<MASK>(a, x, list, c0 + (h >> 1) * W);
      const bool masked = j0 + kKvChunk > open;
      uint32_t see[NT];  // tree: the keys that rows 2t (lower half) and 2t + 1 see, loaded beside the copies
      if (MASK == kMaskTree && masked) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          see[nt] = __byte_perm(kv_sees<MASK>(a, x, nt * 8 + 2 * t, j0), kv_sees<MASK>(a, x, nt * 8 + 2 * t + 1, j0),
                                0x5410) >> g;
      }
      cp_async_wait(2);
      __syncwarp();
      // Scores: a lane takes dimensions 16 pair + 4t + e of keys g and g + 8.  The tensor cores
      // cut their f32 sums instead of rounding them, one cut per step: hi.hi runs in chains of
      // four steps, summed here with rounding; the cross terms are 2^-11 of it.
      const uint32_t kst = ring + slot * kKvHalf;
      float hh[NT][4][4], cross[NT][4][4];
#pragma unroll
      for (int quad = 0; quad < 4; ++quad) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) hh[nt][quad][e] = cross[nt][quad][e] = 0.0f;
#pragma unroll
        for (int pair = 2 * quad; pair < 2 * quad + 2; ++pair) {
          const uint32_t at = kst + g * (kKvD * 4) + (((pair * 4 + t) ^ ((g & 1) << 2)) << 4);
          const float4 ka = lds_f4(at), kb4 = lds_f4(at + 8 * kKvD * 4);
          uint32_t ah[4], al[4], bh[4], bl[4];
          split_tf32(ka.x, ah[0], al[0]);
          split_tf32(ka.y, ah[1], al[1]);
          split_tf32(ka.z, ah[2], al[2]);
          split_tf32(ka.w, ah[3], al[3]);
          split_tf32(kb4.x, bh[0], bl[0]);
          split_tf32(kb4.y, bh[1], bl[1]);
          split_tf32(kb4.z, bh[2], bl[2]);
          split_tf32(kb4.w, bh[3], bl[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint4 qh = *reinterpret_cast<const uint4*>(&sm.q[0][pair][nt][lane]);
            const uint4 ql = *reinterpret_cast<const uint4*>(&sm.q[1][pair][nt][lane]);
            mma_tf32(hh[nt][quad], ah[0], bh[0], ah[1], bh[1], qh.x, qh.y);
            mma_tf32(cross[nt][quad], al[0], bl[0], al[1], bl[1], qh.x, qh.y);
            mma_tf32(hh[nt][quad], ah[2], bh[2], ah[3], bh[3], qh.z, qh.w);
            mma_tf32(cross[nt][quad], ah[0], bh[0], ah[1], bh[1], ql.x, ql.y);
            mma_tf32(cross[nt][quad], al[2], bl[2], al[3], bl[3], qh.z, qh.w);
            mma_tf32(cross[nt][quad], ah[2], bh[2], ah[3], bh[3], ql.z, ql.w);
          }
        }
      }
      __syncwarp();
      load(h + 3, slot);  // the keys are in registers: their slot is free
      slot = slot == kKvSlots - 1 ? 0 : slot + 1;

      float fac[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float p[4];  // [key g, g + 8][row 2t, 2t + 1] of the n-tile
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float big = __fadd_rn(__fadd_rn(hh[nt][0][e], hh[nt][1][e]), __fadd_rn(hh[nt][2][e], hh[nt][3][e]));
          const float low =
              __fadd_rn(__fadd_rn(cross[nt][0][e], cross[nt][1][e]), __fadd_rn(cross[nt][2][e], cross[nt][3][e]));
          p[e] = __fmul_rn(__fadd_rn(big, low), a.c);
          if (masked) {
            const int j = j0 + g + (e >> 1) * 8;
            if (MASK == kMaskTree ? !((see[nt] >> ((e & 1) * 16 + (e >> 1) * 8)) & 1u)
                                  : j >= x.keys || j > x.p + kv_token<MASK>(a, x, min(nt * 8 + 2 * t + (e & 1), x.nrows - 1)))
              p[e] = -INFINITY;
          }
        }
        if (SCORES) {
          float* sc = a.scores + ((size_t)x.b * a.hkv + x.hk) * x.nrows * (size_t)a.score_stride + j0 + g;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = nt * 8 + 2 * t + (e & 1);
            if (r < x.nrows) sc[(size_t)r * a.score_stride + (e >> 1) * 8] = p[e];
          }
        }
        float x0 = fmaxf(p[0], p[2]), x1 = fmaxf(p[1], p[3]);
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) {
          x0 = fmaxf(x0, __shfl_xor_sync(kFull, x0, s));
          x1 = fmaxf(x1, __shfl_xor_sync(kFull, x1, s));
        }
        const float n0 = fmaxf(m[nt][0], x0), n1 = fmaxf(m[nt][1], x1);
        const float b0 = n0 == -INFINITY ? 0.0f : n0, b1 = n1 == -INFINITY ? 0.0f : n1;
        fac[nt][0] = exp2f(m[nt][0] - b0);
        fac[nt][1] = exp2f(m[nt][1] - b1);
        m[nt][0] = n0;
        m[nt][1] = n1;
        p[0] = exp2f(p[0] - b0);
        p[1] = exp2f(p[1] - b1);
        p[2] = exp2f(p[2] - b0);
        p[3] = exp2f(p[3] - b1);
        l[nt][0] = fmaf(l[nt][0], fac[nt][0], p[0] + p[2]);
        l[nt][1] = fmaf(l[nt][1], fac[nt][1], p[1] + p[3]);
        *reinterpret_cast<float2*>(&sm.p[warp][nt][g][2 * t]) = make_float2(p[0], p[1]);
        *reinterpret_cast<float2*>(&sm.p[warp][nt][g + 8][2 * t]) = make_float2(p[2], p[3]);
      }
      cp_async_wait(2);
      __syncwarp();  // the values have landed, the probabilities are written
      const uint32_t vst = ring + slot * kKvHalf;
      // a value row that is not finite, or whose hi part is not (it rounds up), must not reach the
      // rows that do not see it (0 * inf): such a chunk, only where a mask is at work, takes the
      // exact loop below
      bool odd = false;
      constexpr float kHiFinite = 0x1.ffep127f;  // from here on hi is infinite
      if (masked) {
        for (int r = 0; r < kKvChunk; ++r) {
          const float4 w = lds_f4(vst + r * (kKvD * 4) + lane * 16);
          odd |= !(fabsf(w.x) < kHiFinite && fabsf(w.y) < kHiFinite && fabsf(w.z) < kHiFinite && fabsf(w.w) < kHiFinite);
        }
        odd = __any_sync(kFull, odd);
      }
      if (!odd) {
        // Output: a lane takes keys t, t + 4, t + 8, t + 12 and dimensions 32 w + 4g + e; the
        // chunk's sum starts from 0 and joins the running one with rounding.
        uint32_t ph[NT][2][2], pl[NT][2][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int y = 0; y < 2; ++y) split_tf32(sm.p[warp][nt][ks * 8 + y * 4 + t][g], ph[nt][ks][y], pl[nt][ks][y]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          float d[NT][2][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int z = 0; z < 2; ++z)
#pragma unroll
              for (int y = 0; y < 4; ++y) d[nt][z][y] = 0.0f;
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            const uint32_t at = vst + (ks * 8 + t) * (kKvD * 4) + (((w * 8 + g) ^ (t << 1)) << 4);
            const float4 va = lds_f4(at), vc = lds_f4(at + 4 * kKvD * 4);
            uint32_t ah[4], al[4], ch[4], cl[4];
            split_tf32(va.x, ah[0], al[0]);
            split_tf32(va.y, ah[1], al[1]);
            split_tf32(va.z, ah[2], al[2]);
            split_tf32(va.w, ah[3], al[3]);
            split_tf32(vc.x, ch[0], cl[0]);
            split_tf32(vc.y, ch[1], cl[1]);
            split_tf32(vc.z, ch[2], cl[2]);
            split_tf32(vc.w, ch[3], cl[3]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int z = 0; z < 2; ++z) {
                mma_tf32(d[nt][z], al[2 * z], al[2 * z + 1], cl[2 * z], cl[2 * z + 1], ph[nt][ks][0], ph[nt][ks][1]);
                mma_tf32(d[nt][z], ah[2 * z], ah[2 * z + 1], ch[2 * z], ch[2 * z + 1], pl[nt][ks][0], pl[nt][ks][1]);
                mma_tf32(d[nt][z], ah[2 * z], ah[2 * z + 1], ch[2 * z], ch[2 * z + 1], ph[nt][ks][0], ph[nt][ks][1]);
              }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int z = 0; z < 2; ++z)
#pragma unroll
              for (int y = 0; y < 4; ++y)
                o[nt][2 * w + z][y] = fmaf(o[nt][2 * w + z][y], fac[nt][y & 1], d[nt][z][y]);
        }
      } else {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int y = 0; y < 4; ++y) o[nt][i][y] *= fac[nt][y & 1];
          for (int r = 0; r < kKvChunk; ++r) {
            const float pa = sm.p[warp][nt][r][2 * t], pb = sm.p[warp][nt][r][2 * t + 1];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const float4 q4 = lds_f4(vst + r * (kKvD * 4) + (((w * 8 + g) ^ ((r & 3) << 1)) << 4));
              const float vv[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float* dst = o[nt][2 * w + (e >> 1)] + 2 * (e & 1);
                if (pa != 0.0f) dst[0] = fmaf(pa, vv[e], dst[0]);
                if (pb != 0.0f) dst[1] = fmaf(pb, vv[e], dst[1]);
              }
            }
          }
        }
      }
      __syncwarp();
      load(h + 4, slot);
      slot = slot == kKvSlots - 1 ? 0 : slot + 1;
    }
    cp_async_wait(0);
    __syncwarp();

    // the warps' parts, merged in warp order
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) l[nt][y] += __shfl_xor_sync(kFull, l[nt][y], s);
        if (g == 0) {
          const int r = nt * 8 + 2 * t + y;
          sm.m[warp][r] = kv_row_valid<MASK>(a, x, r) ? m[nt][y] : -INFINITY;
          sm.l[warp][r] = l[nt][y];
        }
        float* part = reinterpret_cast<float*>(&sm.ring[warp][0][0]) + (nt * 8 + 2 * t + y) * (kKvD + 4) + 4 * g;
#pragma unroll
        for (int w = 0; w < 4; ++w)
          *reinterpret_cast<float4*>(part + 32 * w) =
              make_float4(o[nt][2 * w][y], o[nt][2 * w][2 + y], o[nt][2 * w + 1][y], o[nt][2 * w + 1][2 + y]);
      }
    }
    __syncthreads();
    const size_t slot_id = a.split ? (size_t)blockIdx.x + u : (size_t)u;
    const bool whole = off == 0 && c1 == x.chunks;
    if (a.split && off == 0 && tid == 0)  // for the merge: the first CTA, and how many there are
      a.begun[u] = make_int2(blockIdx.x, 1 + (x.chunks - c1 + quota - 1) / quota);
    if (tid < x.nrows) {
      float M = -INFINITY, L = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) M = fmaxf(M, sm.m[w][tid]);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float f = M == -INFINITY ? 0.0f : exp2f(sm.m[w][tid] - M);
        sm.f[w][tid] = f;
        if (f != 0.0f) L = fmaf(sm.l[w][tid], f, L);  // an empty part's sums stay out
      }
      sm.M[tid] = M;
      sm.L[tid] = L;
      if (a.stat) {
        a.stat[slot_id * 2 * a.rows + tid] = M;
        a.stat[slot_id * 2 * a.rows + a.rows + tid] = L;
      }
    }
    __syncthreads();
    for (int e = tid; e < x.nrows * 32; e += kThreads) {
      const int r = e >> 5, d = (e & 31) * 4;
      float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float f = sm.f[w][r];
        const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(&sm.ring[w][0][0]) +
                                                          r * (kKvD + 4) + d);
        if (f != 0.0f) {
          A.x = fmaf(v.x, f, A.x);
          A.y = fmaf(v.y, f, A.y);
          A.z = fmaf(v.z, f, A.z);
          A.w = fmaf(v.w, f, A.w);
        }
      }
      if (whole) {
        if (sm.M[r] != -INFINITY) {
          const float L = sm.L[r];
          A = make_float4(__fdiv_rn(A.x, L), __fdiv_rn(A.y, L), __fdiv_rn(A.z, L), __fdiv_rn(A.w, L));
        }
        *reinterpret_cast<float4*>(a.out + kv_row_offset<MASK>(a, x, r) + d) = A;
      } else {
        *reinterpret_cast<float4*>(a.acc + (slot_id * a.rows + r) * kKvD + d) = A;
      }
    }
    left -= c1 - off;
    off = 0;
    ++u;
    if (!a.split) break;
    __syncthreads();  // the ring, sm.q and the statistics are free
  }
}

// Merge of the parts of every unit, and the weights of the keys where the scores were stored:
// weight[j] += sum over the rows of 2^(s_j - maximum) / sum.  (Not 2^(s_j - log2 of all): a maximum of
// 2^20 leaves the logarithm of the sum four bits.)  grid (units, rows + key ranges): CTA (u, r)
// merges row r, CTA (u, rows + k) adds the weights of range k.  Five CTAs on an SM: with four (8 registers
// more) the weights of 8 tokens x 16 heads over 8 K keys take 28 us, with five 22.
constexpr int kKvMergeThreads = 128;
constexpr int kKvWeightKeys = kKvMergeThreads;  // one key a thread at a time
template <int MASK, bool SCORES>
__global__ void __launch_bounds__(kKvMergeThreads, 5) kv_merge_kernel(const KvArgs a, float* __restrict__ weight) {
  __shared__ float fac[kKvGrid], rm[kKvMergeThreads / 32], rl[kKvMergeThreads / 32];
  __shared__ float2 norm[kKvMaxRows];  // the rows' maxima and 1 / sums
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, u = blockIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  const KvUnit x = kv_unit<MASK>(a, u);
  const bool merging = (int)blockIdx.y < a.rows;
  const int row = blockIdx.y;
  if (merging && (row >= x.nrows || !a.split)) return;
  if (x.chunks == 0) {  // no CTA came by
    if (merging) a.out[kv_row_offset<MASK>(a, x, row) + tid] = 0.0f;
    return;
  }
  const int key0 = ((int)blockIdx.y - a.rows) * kKvWeightKeys * a.weight_reps;
  if (!merging && key0 >= x.keys) return;
  size_t slot0 = u;
  int parts = 1;
  if (a.split) {
    const int2 d = a.begun[u];
    slot0 = (size_t)d.x + u;
    parts = d.y;
  }
  const float* stat = a.stat + slot0 * 2 * a.rows;
  if (merging) {
    if (parts == 1) return;
    float M = -INFINITY;
    for (int s = tid; s < parts; s += kKvMergeThreads) M = fmaxf(M, stat[s * 2 * a.rows + row]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(kFull, M, o));
    if (lane == 0) rm[warp] = M;
    __syncthreads();
    M = fmaxf(fmaxf(rm[0], rm[1]), fmaxf(rm[2], rm[3]));
    float L = 0.0f;
    for (int s = tid; s < parts; s += kKvMergeThreads) {
      const float f = M == -INFINITY ? 0.0f : exp2f(stat[s * 2 * a.rows + row] - M);
      fac[s] = f;
      if (f != 0.0f) L = fmaf(stat[(s * 2 + 1) * a.rows + row], f, L);
    }
    L = warp_sum(L);
    if (lane == 0) rl[warp] = L;
    __syncthreads();
    L = (rl[0] + rl[1]) + (rl[2] + rl[3]);
    const float* acc = a.acc + (slot0 * a.rows + row) * kKvD + tid;
    float A = 0.0f;
#pragma unroll 8
    for (int s = 0; s < parts; ++s) {
      const float f = fac[s], v = acc[(size_t)s * a.rows * kKvD];
      A = f != 0.0f ? fmaf(v, f, A) : A;
    }
    a.out[kv_row_offset<MASK>(a, x, row) + tid] = M == -INFINITY ? 0.0f : __fdiv_rn(A, L);
    return;
  }
  if (SCORES) {
    // the first keys' scores are on their way while the rows' sums are put together
    const size_t bh = (size_t)x.b * a.hkv + x.hk;
    float sc[kKvMaxRows], old = 0.0f;
    auto load = [&](int key) {
      if (key >= x.keys) return;
      old = weight[bh * a.max_t + key];
#pragma unroll
      for (int r = 0; r < kKvMaxRows; ++r)
        if (r < x.nrows) sc[r] = a.scores[(bh * x.nrows + r) * a.score_stride + key];
    };
    load(key0 + tid);
    for (int r = warp; r < x.nrows; r += kKvMergeThreads / 32) {  // a warp per row
      float M = -INFINITY, L = 0.0f;
      for (int s = lane; s < parts; s += 32) M = fmaxf(M, stat[s * 2 * a.rows + r]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(kFull, M, o));
      for (int s = lane; s < parts; s += 32) {
        const float f = M == -INFINITY ? 0.0f : exp2f(stat[s * 2 * a.rows + r] - M);
        if (f != 0.0f) L = fmaf(stat[(s * 2 + 1) * a.rows + r], f, L);
      }
      L = warp_sum(L);
      if (lane == 0) norm[r] = make_float2(M, M == -INFINITY ? 0.0f : __fdiv_rn(1.0f, L));
    }
    __syncthreads();
    for (int rep = 0; rep < a.weight_reps; ++rep) {
      const int key = key0 + rep * kKvWeightKeys + tid;
      if (key >= x.keys) return;
      if (rep > 0) load(key);
      float w = 0.0f;
#pragma unroll
      for (int r = 0; r < kKvMaxRows; ++r)
        if (r < x.nrows) {
          const float2 n = norm[r];
          if (n.y != 0.0f) w = fmaf(exp2f(sc[r] - n.x), n.y, w);
        }
      weight[bh * a.max_t + key] = old + w;
    }
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

// How the rows are cut into units and where the core's part of the workspace lies.
struct KvPlan {
  int rows = 8;
  int rgs = 1;
  int64_t units = 0;
  bool split = false;
  size_t slots = 0;
};
// Rows a kv head from which the tcgen05 kernel (128 rows a unit) takes over: from there on the core
// reads the keys more than once (16 rows a unit).  Its units start faster, so it keeps what can be no
// more than kKvCoreRows units x rows of the cache, about ten chunks a CTA.  (Trees, core and tcgen05
// kernel: 24 rows a kv head behind 100 rows 15.4 and 17.3 us, behind 8 K rows (16 K x 2) 29.1 and 30.4;
// 128 rows behind 500 (8 K) 19.4 and 20.6, behind 2 K (32 K) 23.9 and 22.8, behind 8 K 38.9 and 32.9;
// 512 rows behind 100 (6.4 K) 20.1 and 22.4, behind 500 (32 K) 25.9 and 22.5, behind 8 K 103.1 and
// 37.8; four sequences of 128 rows behind 500 (32 K) 24.2 and 21.8.)
constexpr int64_t kKvTileMinRows = 17;
constexpr int64_t kKvCoreRows = 10 * kKvGrid * kKvChunk;
KvPlan kv_plan(int64_t lists, int64_t rows_per_list, bool tile) {
  KvPlan p;
  p.rows = tile && rows_per_list >= kKvTileMinRows ? kKvTileRows : rows_per_list <= 8 ? 8 : kKvMaxRows;
  p.rgs = (int)((rows_per_list + p.rows - 1) / p.rows);
  p.units = lists * p.rgs;
  // with two units per SM and more the units themselves fill the GPU
  p.split = p.units < 2 * kKvGrid;
  p.slots = !p.split ? (size_t)p.units : p.rows == kKvTileRows ? (size_t)(2 * kKvGrid) : (size_t)(kKvGrid + p.units);
  return p;
}
KvPlan tree_plan(int batch, int n, int hq, int hkv, int max_t) {
  const int64_t lists = (int64_t)batch * hkv, rows = (int64_t)n * (hq / hkv);
  return kv_plan(lists, rows, lists * ((rows + kKvMaxRows - 1) / kKvMaxRows) * max_t > kKvCoreRows);
}
size_t begun_bytes(const KvPlan& p) { return (size_t)p.units * sizeof(int2); }
size_t core_bytes(const KvPlan& p, bool stat) {
  return (p.split ? up256(p.slots * p.rows * kKvD * 4) + up256(begun_bytes(p)) : 0) +
         (p.split || stat ? up256(p.slots * 2 * p.rows * 4) : 0);
}
// Sets the core's part of the workspace; returns the bytes it takes.
size_t core_place(KvArgs& a, const KvPlan& p, bool stat, uint8_t* ws) {
  size_t o = 0;
  if (p.split) {
    a.acc = reinterpret_cast<float*>(ws);
    o += up256(p.slots * p.rows * kKvD * 4);
    a.begun = reinterpret_cast<int2*>(ws + o);
    o += up256(begun_bytes(p));
  }
  if (p.split || stat) {
    a.stat = reinterpret_cast<float*>(ws + o);
    o += up256(p.slots * 2 * p.rows * 4);
  }
  a.rows = p.rows;
  a.chunk = p.rows == kKvTileRows ? kKvTileKeys : kKvChunk;
  a.each = p.units < kKvGrid ? (int)(kKvGrid / p.units) : 0;
  a.least = kKvLeast;
  a.pass = kKvPass;
  a.rgs = p.rgs;
  a.units = (int)p.units;
  a.split = p.split ? 1 : 0;
  return o;
}

template <int MASK, bool SCORES, int NT, int W>
cudaError_t launch_core_nt(const KvArgs& a, int device, cudaStream_t s) {
  static int configured[128] = {0};
  cudaError_t e = ensure_smem((const void*)kv_attention_kernel<MASK, SCORES, NT, W>, configured, device,
                              sizeof(KvSmem<NT, W>), W == 4);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg =
      kv_cfg(dim3((unsigned)(a.split ? kKvGrid : a.units)), dim3(W * 32), sizeof(KvSmem<NT, W>), s, attr);
  return cudaLaunchKernelEx(&cfg, kv_attention_kernel<MASK, SCORES, NT, W>, a);
}
// Units of 8 or 16 rows; causal rows come here with their scores stored.
template <int MASK>
cudaError_t launch_core(const KvArgs& a, float* weight, int device, cudaStream_t s) {
  constexpr bool SCORES = MASK == kMaskCausal;
  cudaError_t e = a.rows != 8 ? launch_core_nt<MASK, SCORES, 2, kKvWarps>(a, device, s)
                  : a.split   ? launch_core_nt<MASK, SCORES, 1, kKvWarps>(a, device, s)
                              : launch_core_nt<MASK, SCORES, 1, 4>(a, device, s);
  if (e != cudaSuccess || (!a.split && !SCORES)) return e;
  const unsigned ranges =
      SCORES ? (unsigned)((a.max_t + kKvWeightKeys * a.weight_reps - 1) / (kKvWeightKeys * a.weight_reps)) : 0u;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = kv_cfg(dim3((unsigned)a.units, (unsigned)a.rows + ranges), dim3(kKvMergeThreads), 0, s, attr);
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

bool weights_stored(int n, int group) { return (int64_t)n * group <= kKvMaxRows; }
int score_stride(int max_t) { return (max_t + kKvChunk - 1) / kKvChunk * kKvChunk; }

}  // namespace

size_t attention_tree_workspace_bytes(int batch, int n, int hq, int hkv) {
  // max_t decides on the kernel: room for either
  const int64_t lists = (int64_t)batch * hkv, rows = (int64_t)n * (hq / hkv);
  const size_t core = core_bytes(kv_plan(lists, rows, false), false), tile = core_bytes(kv_plan(lists, rows, true), false);
  return up256((size_t)batch * n * hq * kKvD * 4) + up256((size_t)batch * n * tree_words(n) * 4) +
         (core > tile ? core : tile);
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
  core_place(a, tree_plan(batch, n, hq, hkv, max_t), false, w);
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = kv_cfg(dim3((unsigned)n, (unsigned)batch), dim3(kKvMaxTree), 0, s, attr);
  cudaError_t e = cudaLaunchKernelEx(&cfg, rope_tree_kernel, qkv, parents, pos, cos_t, sin_t, kc, vc, n, a.words, hq,
                                     hkv, max_t, q, anc);
  if (e != cudaSuccess) return e;
  return a.rows == kKvTileRows ? launch_kv_tile(a, kMaskTree, device, s) : launch_core<kMaskTree>(a, nullptr, device, s);
}

size_t attention_weights_workspace_bytes(int batch, int n, int hq, int hkv, int max_t) {
  const int group = hq / hkv;
  const KvPlan p = kv_plan((int64_t)batch * hkv, (int64_t)n * group, true);
  const bool stored = weights_stored(n, group);
  return core_bytes(p, stored) + (stored ? up256((size_t)batch * hq * n * score_stride(max_t) * 4)
                                         : up256((size_t)batch * hq * n * 8) + up256((size_t)batch * hq * n * 4) +
                                               up256(kv_column_tile_bytes(batch, n, hq, hkv, max_t)));
}

cudaError_t launch_attention_weights(const float* q, const float* kc, const float* vc, const int* pos, int batch, int n,
                                     int hq, int hkv, int max_t, float* weight, void* ws, float* out, int device,
                                     cudaStream_t s) {
  KvArgs a = kv_args(q, kc, vc, pos, batch, n, hq, hkv, max_t, out);
  const bool stored = weights_stored(n, a.group);
  uint8_t* w = static_cast<uint8_t*>(ws);
  w += core_place(a, kv_plan((int64_t)batch * hkv, (int64_t)n * a.group, true), stored, w);
  if (stored) {
    a.scores = reinterpret_cast<float*>(w);
    a.score_stride = score_stride(max_t);
    // about eight CTAs an SM: each starts with a look at all units
    const int64_t groups = (int64_t)a.units * ((max_t + kKvWeightKeys - 1) / kKvWeightKeys);
    a.weight_reps = (int)(groups / 1184 < 1 ? 1 : groups / 1184 > 16 ? 16 : groups / 1184);
    return launch_core<kMaskCausal>(a, weight, device, s);
  }
  a.norm = reinterpret_cast<float2*>(w);
  w += up256((size_t)batch * hq * n * 8);
  a.qscale = reinterpret_cast<float*>(w);
  w += up256((size_t)batch * hq * n * 4);
  cudaError_t e = launch_kv_tile(a, kMaskCausal, device, s);
  if (e != cudaSuccess) return e;
  return launch_kv_column_tile(a, weight, reinterpret_cast<float*>(w), device, s);
}

size_t attention_blocks_workspace_bytes(int batch, int n, int hq, int hkv) {
  return up256(core_bytes(kv_plan((int64_t)batch * n * hkv, hq / hkv, false), false) + 1);  // never 0: it may be allocated
}

cudaError_t launch_attention_blocks(const float* q, const float* kc, const float* vc, const int* pos, const int* index,
                                    int batch, int n, int hq, int hkv, int max_t, int block, int topk, void* ws,
                                    float* out, int device, cudaStream_t s) {
  KvArgs a = kv_args(q, kc, vc, pos, batch, n, hq, hkv, max_t, out);
  a.index = index;
  a.block = block;
  a.topk = topk;
  core_place(a, kv_plan((int64_t)batch * n * hkv, a.group, false), false, static_cast<uint8_t*>(ws));
  return launch_core<kMaskBlocks>(a, nullptr, device, s);
}

}  // namespace q8lin
