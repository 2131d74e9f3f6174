// The attention core over the KV cache on tcgen05: units of 128 query rows against tiles of
// 64 keys, for kv heads with many rows (wide trees, prompt chunks).
//
// Products: f32 operands as pairs of f16 numbers under a power-of-two scale, three
// tcgen05.mma kind::f16 per product.  x s = hi + lo with a power of two s for each row (query, key or
// value), which brings the row's largest |x s| into [2^2, 2^14); hi = x s rounded to f16, lo = x s - hi
// (exact) rounded to f16; a.b = lo.hi + hi.lo + hi.hi.  An element is off by at most 2^-23 of itself or
// 2^-27 of its row's largest, and the dropped lo.lo is at most 2^-22 of a product.  A row's scale
// depends on other rows only where these are near it in size (row_scales), so a row that a
// query does not see may hold anything.
// The keys' scales leave with the scores.  The values' scales differ inside a sum: with 1 / s_j = w_j,
//   sum_j p_j v_j = 2^(d - 14) sum_j (2^(14 - d) p_j w_j) (v_j s_j),   d = ceil(log2 max_j p_j w_j)
// over the keys that the row sees, running as the maximum of the scores does.  So a probability is
// rounded (22 bits) against the largest share that a key the row sees has in its output, and neither
// unseen values nor heavy keys with small ones take bits from it.
//
// One CTA per SM, 16 warps of 128 registers:
//   * 7 convert, in turn, groups of 8 keys or values: cache rows to registers one group ahead, then
//     scaled hi / lo to swizzled shared memory, K as [64 keys][128 dims] in two stages, V transposed
//     as [128 dims][64 keys] in three.  K and V of a tile behind each other: the softmax needs
//     the scales of both (K two tiles ahead of V: 64 trees' units 191 us for 189);
//   * 1 issues the MMAs, S = Q K^T and O = P V (Q and P in TMEM, S and P double-buffered), so that
//     QK of a tile runs while the softmax of the one before is at work.  Issuing waits for the
//     tensor cores' queue, most of the tile's MMA time: a warp with other work cannot do it beside;
//   * 8 softmax: two threads a row, one for each half of the keys and then of the dimensions;
//     scores from TMEM, running maximum, share and sum, P' = 2^(14 - d) p w back to TMEM as hi / lo;
//     then the O tile of the tile before is added to registers.
// The tensor cores cut their f32 sums, so an O tile starts from 0 and joins the running sum with
// rounding.  TMEM (512 columns): Q 128, S 2 x 64, P 2 x 64, O 128.
//
// What bounds it: per 128 rows x 64 keys 24 MMAs of N = 64 and 12 of N = 128, 1632 cycles, a third
// of a tile's time (64 trees' units of 122 tiles, 53 tiles a CTA: 157 us with the launches around it
// where two inputs alternate in a graph, 180 where three do, by the clock that power leaves).  Issue
// slots are 57 % busy; the rest is the roles' chain through a tile (S, maximum, P, O) and instruction
// fetch: the unrolled loops of three roles are more than the instruction caches hold, so what
// shortens their code shortens the tile (one issue loop for the three products, one site each for the
// converters' loads and for adding O: 163 -> 154 us; the softmax's first pass 16 keys at a time: 196
// -> 193; two copies of the converter's loop in turn: 254).  A unit costs about 9 us beside its tiles.
#include <cmath>

#include "common.cuh"
#include "internal.h"
#include "kv_core.cuh"

namespace q8lin {

namespace {

constexpr int kKtThreads = 512;
constexpr int kKtConvertWarp = 8, kKtConverters = 7, kKtMmaWarp = 15;
constexpr uint32_t kKtTmemCols = 512;
constexpr uint32_t kTmQ = 0, kTmS = 128, kTmP = 256, kTmO = 384;
constexpr int kKtPScale = 14;     // P' = 2^(14 - d) p w
// A value row's 1 / s is at least this: p' = 2^(14 - d) p fits f32.  (It is reached by rows whose largest
// value is below 2^-102: they lose bits, under 2^-137 of size each.)
constexpr int kKtLeastShare = -112;

__device__ unsigned int g_kv_tile_fault;
__shared__ uint64_t s_kt_wait_ns;

// The units of this CTA and their tiles, in order.  With few units all CTAs share all tiles evenly
// (split); with many, CTA c takes whole units c, c + 148, ..., the ones with the latest rows, which
// see most, first.
struct KtCursor {
  int u, off, left;  // split: unit, its first tile here, tiles left of the CTA's share; else: u-th in the order
  int n;             // tiles of the unit here
  int t0 = 0;        // tiles of the CTA before it
  KvUnit x;
  // Unit k of the order without a split.
  __device__ static int in_order(const KvArgs& a, int k) {
    const int lists = a.units / a.rgs;
    return k % lists * a.rgs + a.rgs - 1 - k / lists;
  }
  // Moves to the first unit from u on with work; false when there is none.
  template <int MASK>
  __device__ bool seek(const KvArgs& a) {
    while (u < a.units && left > 0) {
      x = kv_unit<MASK>(a, a.split ? u : in_order(a, u));
      n = min(x.chunks - off, left);
      if (n > 0) return true;
      off = 0;
      u += a.split ? 1 : kKvGrid;
    }
    return false;
  }
  __device__ void pass(const KvArgs& a) {  // to the unit behind
    if (a.split) left -= n;
    t0 += n;
    off = 0;
    u += a.split ? 1 : kKvGrid;
  }
};

struct KtSmem {
  alignas(1024) uint8_t k[2][2][2][kKvTileKeys * 128];  // [stage][hi, lo][64 dims][key][128 B]
  alignas(1024) uint8_t v[3][2][kKvD * 128];            // [stage][hi, lo][dim][64 keys]
  alignas(16) float ksc[4][kKvTileKeys], vsc[4][kKvTileKeys];  // inverse scales of the rows of tiles t % 4
  alignas(16) float vlog[4][kKvTileKeys];               // log2 of vsc
  alignas(8) uint8_t vbad[4][8];                        // keys of the tile whose value row is not finite
  alignas(8) float2 top[2][2][kKvTileRows];             // the rows' maxima over either half of a tile
  alignas(8) uint64_t kfull[2], kfree[2], vfull[3], vfree[3];
  uint64_t vinfo[4];
  uint64_t sfull[2], pfull[2], qfull, ofull, ofree, done;
  KtCursor cursor[8];                  // the softmax warps' (registers are short there)
  alignas(16) float turn[2][4][32][36];  // rows of four warps: coalesced memory <-> a thread per row
  KvFind find;
  uint32_t tmem;
  int abort;
};

__device__ __forceinline__ uint32_t su32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t* b, uint32_t n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(b)), "r"(n) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(su32(b)) : "memory");
}
// Bounded wait; once one has run out (or another warp's has) every wait of the CTA fails.
__device__ __forceinline__ bool bar_wait_slow(uint32_t bar, uint32_t parity, volatile int* abort) {
  const uint64_t t0 = global_ns();
  while (!*abort) {
    if (global_ns() - t0 >= s_kt_wait_ns) {  // a limit of 0 allows no waiting at all
      atomicOr(&g_kv_tile_fault, 32u);
      *abort = 1;
    } else if (mb_try(bar, parity)) {
      return true;
    }
  }
  return false;
}
// By whole warps: the verdict is uniform.
__device__ __forceinline__ bool bar_wait(uint64_t* b, uint32_t parity, volatile int* abort) {
  const uint32_t bar = su32(b);
  return __all_sync(kFull, mb_try(bar, parity) || bar_wait_slow(bar, parity, abort));
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// K-major 128B-swizzled operand: 8-row atoms of 128 bytes, 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_sw128(const void* base) {
  uint64_t d = (su32(base) >> 4) & 0x3FFFull;
  d |= (uint64_t)1 << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// kind::f16, f16 operands, f32 sums, M = 128.
__host__ __device__ constexpr uint32_t kt_idesc(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24); }
// D (+)= A (TMEM) B^T (shared memory); by one lane.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// The lane that issues a warp's MMAs and commits.
__device__ __forceinline__ bool elected() {
  uint32_t e;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(e));
  return e != 0;
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(su32(bar)) : "memory");
}
// D = A B^T over 16 STEPS columns as lo.hi + hi.lo + hi.hi, SWAP: as hi.lo + lo.hi + hi.hi, which for A and
// B exchanged is the same sum in the same order.  HALF: bytes from B's first 64 columns to the next.
// The three run through one piece of code: the roles' loops fill the instruction caches.
template <int STEPS, int HALF, bool SWAP = false>
__device__ __forceinline__ void mma_pairs(uint32_t d, uint32_t ah, uint32_t al, const void* bh, const void* bl,
                                          uint32_t idesc) {
  const uint64_t dh = desc_sw128(bh), dl = desc_sw128(bl);
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const uint32_t a = pass == (SWAP ? 1 : 0) ? al : ah;
    const uint64_t b = pass == (SWAP ? 0 : 1) ? dl : dh;
#pragma unroll
    for (int kk = 0; kk < STEPS; ++kk)
      mma_ts(d, a + 8 * kk, b + 2 * (kk & 3) + (kk >> 2) * (HALF >> 4), idesc, pass + kk > 0);
  }
}

#define KT_R32(a) \
  a(0), a(1), a(2), a(3), a(4), a(5), a(6), a(7), a(8), a(9), a(10), a(11), a(12), a(13), a(14), a(15), a(16), a(17), \
      a(18), a(19), a(20), a(21), a(22), a(23), a(24), a(25), a(26), a(27), a(28), a(29), a(30), a(31)
// 32 columns of the thread's TMEM lane; valid after tm_wait_ld.
__device__ __forceinline__ void tm_ld32(uint32_t addr, uint32_t (&r)[32]) {
#define KT_OUT(i) "=r"(r[i])
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : KT_R32(KT_OUT)
      : "r"(addr)
      : "memory");
#undef KT_OUT
}
__device__ __forceinline__ void tm_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tm_ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tm_st8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t tm_ld1(uint32_t addr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(addr) : "memory");
  return r;
}
__device__ __forceinline__ void tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)),
        "l"(reinterpret_cast<const uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 times(float2 a, float b) { return mul2(a, make_float2(b, b)); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 lo2(const float4& v) { return make_float2(v.x, v.y); }
__device__ __forceinline__ float2 hi2(const float4& v) { return make_float2(v.z, v.w); }
__device__ __forceinline__ float2 unpack_f16(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// Two scaled values -> packed hi parts and packed lo parts.  (hi is read back from f16: cutting it
// with integer operations and then packing it loads the narrower integer pipe instead.)
__device__ __forceinline__ void split_f16(float2 x, uint32_t& hi, uint32_t& lo) {
  hi = pack_f16(x.x, x.y);
  const float2 l = fma2(unpack_f16(hi), make_float2(-1.0f, -1.0f), x);
  lo = pack_f16(l.x, l.y);
}
// Largest magnitude (bits of a float) -> the scale that brings it into [2^10, 2^14), at most 2^(most -
// 127), and its inverse.
__device__ __forceinline__ void scale_of(unsigned top, float& scale, float& inverse, int most = 251) {
  const int e = min(most, 267 - (int)(min(top, 0x7f7fffffu) >> 23 | 3u));
  scale = __uint_as_float((unsigned)e << 23);
  inverse = __uint_as_float((unsigned)(254 - e) << 23);
}
__device__ __forceinline__ float mag(float m, float x) { return fmaxf(m, fabsf(x)); }
__device__ __forceinline__ float mag4(float m, const float4& v) { return mag(mag(mag(mag(m, v.x), v.y), v.z), v.w); }
__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// 2^-8 of a largest magnitude (bits of a float); 0 where that is no normal number.
__device__ __forceinline__ unsigned near_of(unsigned top) { return top > (8u << 23) ? top - (8u << 23) : 0u; }
// The scale of 8 rows: that of the largest where each row has an element within 2^-8 of it; otherwise (an
// outlier, a row that is not there) every row is brought to its own scale here and `scale` is 1.  r:
// whole rows, 4 dimensions a lane (ROWS 8), or row 2 i + lane / 16 in r[2 i], r[2 i + 1] (ROWS 4);
// m: the lane's largest magnitudes of each.  Returns the inverse of row lane % 8's whole scale.
template <int ROWS>
__device__ __forceinline__ float row_scales(float4 (&r)[8], const float (&m)[ROWS], float& scale, int most = 251) {
  const int lane = threadIdx.x & 31, up = ROWS == 4 ? lane >> 4 : 0;
  float all = m[0], inverse;
#pragma unroll
  for (int i = 1; i < ROWS; ++i) all = fmaxf(all, m[i]);
  const unsigned top = __reduce_max_sync(kFull, __float_as_uint(all));
  const unsigned near = near_of(top);
  unsigned has = 0;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) has |= (__float_as_uint(m[i]) >= near ? 1u : 0u) << (ROWS == 4 ? 2 * i : i);
  has = __reduce_or_sync(kFull, has << up);
  scale_of(top, scale, inverse, most);
  if (__builtin_expect(has != 255u || top >= 0x7f800000u, 0)) {
    unsigned mine = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = ROWS == 8 ? m[e % ROWS] : (e & 1) == up ? m[e / 2 % ROWS] : 0.0f;
      const unsigned t = __reduce_max_sync(kFull, __float_as_uint(x));
      if ((lane & 7) == e) mine = t;
    }
    scale_of(mine, scale, inverse, most);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float s = __shfl_sync(kFull, scale, ROWS == 8 ? i : (i & ~1) + up);
      r[i] = make_float4(r[i].x * s, r[i].y * s, r[i].z * s, r[i].w * s);
    }
    scale = 1.0f;
  }
  return inverse;
}

// Cache rows pass the SM once: past L1, whose small rest beside 200 KB of shared memory holds
// the tree's masks and what registers cannot (a reload from L2 is 600 cycles of a warp's time).
__device__ __forceinline__ float4 ld_row(const float4* p) {
  const int4 v = ld_stream_v4(p);
  return make_float4(__int_as_float(v.x), __int_as_float(v.y), __int_as_float(v.z), __int_as_float(v.w));
}

// kv_find as a call of its own, on the fields it needs: inlined, its values stay in the roles' way
// (64-node trees 182 us instead of 165), and KvArgs by reference or value goes through memory.
template <int MASK>
__device__ __noinline__ int kt_find(KvFind& find, const int* pos, int n, int hkv, int group, int max_t, int rgs,
                                    int units, int each) {
  KvArgs a = {};
  a.pos = pos;
  a.n = n;
  a.hkv = hkv;
  a.group = group;
  a.max_t = max_t;
  a.rgs = rgs;
  a.units = units;
  a.each = each;
  a.rows = kKvTileRows;
  a.chunk = kKvTileKeys;
  a.least = kKvTileLeast;
  a.pass = kKvTilePass;
  return kv_find<MASK, kKtThreads>(a, find, blockIdx.x);
}

constexpr float kLeastFactor = 1.17549435e-38f;  // a factor of 0 would make NaN of -inf
// A row's maximum and the inverse of its sum; a row that sees nothing gives no key a weight.
__device__ __forceinline__ float2 row_norm(float m, float l) {
  return m == -INFINITY ? make_float2(INFINITY, 0.0f) : make_float2(m, __fdiv_rn(1.0f, l));
}
__device__ __forceinline__ size_t kv_row_number(const KvArgs& a, const KvUnit& x, int row) {
  return ((size_t)x.b * a.hkv + x.hk) * a.n * a.group + x.r0 + row;
}

template <int MASK>
__global__ void __launch_bounds__(kKtThreads, 1) kv_tile_kernel(const KvArgs a, uint64_t wait_ns) {
  extern __shared__ uint8_t kt_raw[];
  // aligned by an offset, not by a cast, so that the compiler keeps seeing shared memory
  KtSmem& sm = *reinterpret_cast<KtSmem*>(kt_raw + ((1024 - (su32(kt_raw) & 1023)) & 1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort = &sm.abort;
  if (tid == 0) {
    s_kt_wait_ns = wait_ns;
    for (int i = 0; i < 2; ++i) {
      bar_init(&sm.kfull[i], 8);
      bar_init(&sm.kfree[i], 1);
      bar_init(&sm.sfull[i], 2);
      bar_init(&sm.pfull[i], 8);
    }
    for (int i = 0; i < 3; ++i) {
      bar_init(&sm.vfull[i], 8);
      bar_init(&sm.vfree[i], 1);
    }
    for (int i = 0; i < 4; ++i) bar_init(&sm.vinfo[i], 8);
    bar_init(&sm.qfull, 8);
    bar_init(&sm.ofull, 1);
    bar_init(&sm.ofree, 8);
    bar_init(&sm.done, 1);
    sm.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kKtMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(&sm.tmem)),
                 "r"(kKtTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  pdl_launch_dependents();
  KtCursor start;
  if (a.split) {
    start.left = kt_find<MASK>(sm.find, a.pos, a.n, a.hkv, a.group, a.max_t, a.rgs, a.units, a.each);
    start.u = sm.find.unit;
    start.off = sm.find.off;
  } else {
    start.left = 0x7fffffff;
    start.u = blockIdx.x;
    start.off = 0;
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = sm.tmem;

  if (warp >= kKtConvertWarp && warp < kKtMmaWarp) {
    // ---------------- converters ----------------
    // The unit's groups in order: K and V of a tile in turn, 8 groups each; warp w takes groups w, w +
    // 7, ..., with no barrier between warps.
    const int h = lane & 15, ky = lane >> 4;
    KtCursor cur = start;
    bool dead = false;
    for (; cur.seek<MASK>(a); cur.pass(a)) {
      const KvUnit& x = cur.x;
      const size_t head = ((size_t)x.b * a.hkv + x.hk) * (size_t)a.max_t;
      // lane's pieces of a row: K dimensions 4 h .. and 64 + 4 h .. of row 2 i + lane / 16, V
      // dimensions 4 lane .. of row i
      const float4* kp = reinterpret_cast<const float4*>(a.k + (head + ky) * kKvD) + h;
      const float4* vp = reinterpret_cast<const float4*>(a.v + head * kKvD) + lane;
      const int c0 = cur.off, n = cur.n, items = 16 * n;
      // Rows below `plain` need no look.  Causal units read all the rows that were appended, also those behind
      // their own last: a key's scale depends on the group it is in, and all units have to agree on it.
      const int plain = MASK == kMaskTree ? x.p : min(x.p + a.n, a.max_t);
      auto rows_there = [&](int j0) {
        if (MASK == kMaskTree) return kv_rows_there<MASK>(a, x, j0);
        return __ballot_sync(kFull, j0 + lane < plain);
      };
      auto tile_of = [](int item) { return item >> 4; };
      auto is_v = [](int item) { return (item & 8) != 0; };
      float4 nx[8] = {};
      auto load = [&](int item) {
        const int j0 = (c0 + tile_of(item)) * kKvTileKeys + (item & 7) * 8;
        if (is_v(item)) {
          const float4* row = vp + (size_t)j0 * (kKvD / 4);
          if (j0 + 8 <= plain) {
#pragma unroll
            for (int i = 0; i < 8; ++i) nx[i] = ld_row(row + i * 32);
          } else {
            const uint32_t there = rows_there(j0);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              nx[i] = (there >> i) & 1u ? ld_row(row + i * 32) : make_float4(0.f, 0.f, 0.f, 0.f);
          }
        } else {
          const float4* row = kp + (size_t)j0 * (kKvD / 4);
          if (j0 + 8 <= plain) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              nx[2 * i] = ld_row(row + i * 64);
              nx[2 * i + 1] = ld_row(row + i * 64 + 16);
            }
          } else {
            const uint32_t rows = rows_there(j0) >> ky;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const bool there = (rows >> (2 * i)) & 1u;
              nx[2 * i] = there ? ld_row(row + i * 64) : make_float4(0.f, 0.f, 0.f, 0.f);
              nx[2 * i + 1] = there ? ld_row(row + i * 64 + 16) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
          }
        }
      };
      // the first round only loads
      for (int item = warp - kKtConvertWarp - kKtConverters; item < items; item += kKtConverters) {
        float4 r[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = nx[i];
        if (item + kKtConverters < items) load(item + kKtConverters);
        if (item < 0) continue;
        const int t = cur.t0 + tile_of(item), g = item & 7;
        if (!is_v(item)) {
          const int s = t & 1;
          float m[4], scale;
#pragma unroll
          for (int i = 0; i < 4; ++i) m[i] = mag4(mag4(0.0f, r[2 * i]), r[2 * i + 1]);
          const float inverse = row_scales<4>(r, m, scale);
          if (t >= 2 && !dead) dead = !bar_wait(&sm.kfree[s], ((t >> 1) - 1) & 1, abort);
          uint8_t* dst = &sm.k[s][0][h >> 3][(g * 8 + ky) * 128];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint4 hi, lo;
            split_f16(times(lo2(r[2 * i]), scale), hi.x, lo.x);
            split_f16(times(hi2(r[2 * i]), scale), hi.y, lo.y);
            split_f16(times(lo2(r[2 * i + 1]), scale), hi.z, lo.z);
            split_f16(times(hi2(r[2 * i + 1]), scale), hi.w, lo.w);
            const int at = i * 256 + (((h & 7) ^ (2 * i + ky)) << 4);
            *reinterpret_cast<uint4*>(dst + at) = hi;
            *reinterpret_cast<uint4*>(dst + sizeof(sm.k[0][0]) + at) = lo;
          }
          if (lane < 8) sm.ksc[t & 3][g * 8 + lane] = inverse;
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) bar_arrive(&sm.kfull[s]);
        } else {
          const int s = t % 3;
          float2 z = make_float2(0.f, 0.f);  // NaN unless all are finite
          float m[8], scale;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            z = fma2(lo2(r[i]), make_float2(0.f, 0.f), z);
            z = fma2(hi2(r[i]), make_float2(0.f, 0.f), z);
            m[i] = mag4(0.0f, r[i]);
          }
          unsigned bad = 0;
          if (__builtin_expect(__any_sync(kFull, !(z.x + z.y == 0.0f)), 0)) {
            // 0 * inf must not reach the rows that do not see the key: its value row leaves the
            // product (0) and the rows that see it add it one by one
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const bool x = finite(r[i].x), y = finite(r[i].y), zz = finite(r[i].z), w = finite(r[i].w);
              m[i] = mag4(0.0f, make_float4(x ? r[i].x : 0.f, y ? r[i].y : 0.f, zz ? r[i].z : 0.f, w ? r[i].w : 0.f));
              if (__any_sync(kFull, !(x && y && zz && w))) {
                r[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                bad |= 1u << i;
              }
            }
          }
          const float inverse = row_scales<8>(r, m, scale, 127 - kKtLeastShare);
          if (t >= 3 && !dead) dead = !bar_wait(&sm.vfree[s], (t / 3 - 1) & 1, abort);
          // dimension 4 lane + e sits in row 32 e + lane, the group's 8 keys in one piece of it
          uint8_t* dst = &sm.v[s][0][lane * 128 + ((g ^ (lane & 7)) << 4)];
          auto put = [&](int e, float2 w0, float2 w1, float2 w2, float2 w3, float2 w4, float2 w5, float2 w6, float2 w7) {
            const float2 w[8] = {times(w0, scale), times(w1, scale), times(w2, scale), times(w3, scale),
                                 times(w4, scale), times(w5, scale), times(w6, scale), times(w7, scale)};
            uint32_t h0[4], h1[4], l0[4], l1[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 u = w[2 * i], v = w[2 * i + 1];
              split_f16(make_float2(u.x, v.x), h0[i], l0[i]);
              split_f16(make_float2(u.y, v.y), h1[i], l1[i]);
            }
            constexpr int low = sizeof(sm.v[0][0]);
            *reinterpret_cast<uint4*>(dst + e * 4096) = make_uint4(h0[0], h0[1], h0[2], h0[3]);
            *reinterpret_cast<uint4*>(dst + e * 4096 + 4096) = make_uint4(h1[0], h1[1], h1[2], h1[3]);
            *reinterpret_cast<uint4*>(dst + low + e * 4096) = make_uint4(l0[0], l0[1], l0[2], l0[3]);
            *reinterpret_cast<uint4*>(dst + low + e * 4096 + 4096) = make_uint4(l1[0], l1[1], l1[2], l1[3]);
          };
          put(0, lo2(r[0]), lo2(r[1]), lo2(r[2]), lo2(r[3]), lo2(r[4]), lo2(r[5]), lo2(r[6]), lo2(r[7]));
          put(2, hi2(r[0]), hi2(r[1]), hi2(r[2]), hi2(r[3]), hi2(r[4]), hi2(r[5]), hi2(r[6]), hi2(r[7]));
          if (lane < 8) {
            sm.vsc[t & 3][g * 8 + lane] = inverse;
            sm.vlog[t & 3][g * 8 + lane] = (float)((int)(__float_as_uint(inverse) >> 23) - 127);
          }
          if (lane == 0) sm.vbad[t & 3][g] = (uint8_t)bad;
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            bar_arrive(&sm.vfull[s]);
            bar_arrive(&sm.vinfo[t & 3]);
          }
        }
      }
    }
  } else if (warp == kKtMmaWarp) {
    // ---------------- MMA issue ----------------
    constexpr uint32_t id_qk = kt_idesc(kKvTileKeys), id_pv = kt_idesc(kKvD);
    bool ok = true;
    int units = 0;
    KtCursor cur = start;
    for (; ok && cur.seek<MASK>(a); cur.pass(a), ++units) {
      ok = bar_wait(&sm.qfull, units & 1, abort);
      // step i: S of tile i, then O of the tile before
      for (int i = 0; ok && i <= cur.n; ++i) {
        if (i < cur.n) {
          // S = Q K^T; its buffer is free: P of tile t - 2 was waited for
          const int t = cur.t0 + i, s = t & 1;
          ok = bar_wait(&sm.kfull[s], (t >> 1) & 1, abort);
          if (!ok) break;
          if (lane == 0) bar_arrive(&sm.sfull[s]);  // passes on what the converters wrote beside the tile
          tc_after();
          __syncwarp();
          if (elected()) {
            mma_pairs<8, sizeof(sm.k[0][0][0])>(tmem + kTmS + 64 * s, tmem + kTmQ, tmem + kTmQ + 64, sm.k[s][0][0],
                                                sm.k[s][1][0], id_qk);
            mma_commit(&sm.kfree[s]);
            mma_commit(&sm.sfull[s]);
          }
          __syncwarp();
        }
        if (i > 0) {
          // O = P V, once every warp wrote its P and has the O before
          const int w = cur.t0 + i - 1, s = w & 1, vs = w % 3;
          ok = bar_wait(&sm.vfull[vs], (w / 3) & 1, abort) && bar_wait(&sm.pfull[s], (w >> 1) & 1, abort) &&
               (w == 0 || bar_wait(&sm.ofree, (w - 1) & 1, abort));
          if (!ok) break;
          tc_after();
          __syncwarp();
          if (elected()) {
            mma_pairs<4, 0>(tmem + kTmO, tmem + kTmP + 64 * s, tmem + kTmP + 64 * s + 32, sm.v[vs][0], sm.v[vs][1], id_pv);
            mma_commit(&sm.vfree[vs]);
            mma_commit(&sm.ofull);
          }
          __syncwarp();
        }
      }
    }
    // nothing of this CTA's may be at work in shared memory or TMEM when it ends
    if (elected()) mma_commit(&sm.done);
    __syncwarp();
    mb_wait_ns(su32(&sm.done), 0, kDrainLimitNs, nullptr);
  } else {
    // ---------------- softmax, output ----------------
    // thread (row, half): keys 32 half .. + 32 of a tile, output columns 64 half .. + 64, which are
    // dimensions 4 i + 2 half and 4 i + 2 half + 1 (i < 32)
    const int row = tid & 127, half = tid >> 7;
    const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    int t = 0;
    // after a wait that ran out the loops go on without waiting (the two warps of a row meet at
    // named barriers) and the rows get NaN
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (ok) ok = bar_wait(bar, parity, abort);
    };
    auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(2 + (warp & 3)) : "memory"); };
    if (!a.split)  // units without keys have no tiles
      for (int u = blockIdx.x; u < a.units; u += kKvGrid) {
        const KvUnit x = kv_unit<MASK>(a, KtCursor::in_order(a, u));
        if (x.chunks > 0 || row >= x.nrows || half > 0) continue;
        float4* dst = reinterpret_cast<float4*>(a.out + kv_row_offset<MASK>(a, x, row));
#pragma unroll 1
        for (int i = 0; i < kKvD / 4; ++i) dst[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (a.norm) a.norm[kv_row_number(a, x, row)] = make_float2(INFINITY, 0.0f);
      }
    // The warp's cursor is one object of its 32 lanes: one of them moves it on, between the others' last
    // look at the unit behind and their first at the next.
    KtCursor& cur = sm.cursor[warp];
    auto forward = [&](bool begin) {
      int more = 0;
      __syncwarp();
      if (lane == 0) {
        if (begin)
          cur = start;
        else
          cur.pass(a);
        more = cur.seek<MASK>(a);
      }
      __syncwarp();
      return __shfl_sync(kFull, more, 0) != 0;
    };
    for (bool begin = true; forward(begin); begin = false) {
      const KvUnit& x = cur.x;
      // half of the query row: scaled hi / lo to TMEM, dimensions in the order of the K tiles (32
      // half .. + 32 and 64 + 32 half .. + 32).  A thread that reads its own row takes 32 memory
      // transactions an access (that cost 10 us a unit), so the warp reads rows and turns them.
      float qinv;
      {
        float4 mine4[16];
        float4* turn = reinterpret_cast<float4*>(&sm.turn[half][warp & 3][0][0]);
        const int row0 = (warp & 3) * 32;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = row0 + 4 * i + (lane >> 3);
          const float4* src = reinterpret_cast<const float4*>(a.q + kv_row_offset<MASK>(a, x, min(r, x.nrows - 1))) +
                              half * 8 + (lane & 7);
          mine4[i] = src[0];
          mine4[8 + i] = src[16];
        }
#pragma unroll
        for (int part = 0; part < 2; ++part) {  // the two stretches of 32 dimensions
#pragma unroll
          for (int i = 0; i < 8; ++i) turn[(4 * i + (lane >> 3)) * 9 + (lane & 7)] = mine4[part * 8 + i];
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) mine4[part * 8 + i] = turn[lane * 9 + i];
          __syncwarp();
        }
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) m = mag(mag(mag(mag(m, mine4[i].x), mine4[i].y), mine4[i].z), mine4[i].w);
        sm.top[0][half][row].x = m;
        meet();
        m = fmaxf(m, sm.top[0][half ^ 1][row].x);
        meet();
        float scale;
        scale_of(__float_as_uint(m), scale, qinv);
        if (a.norm && cur.off == 0 && half == 0 && row < x.nrows) a.qscale[kv_row_number(a, x, row)] = scale;
        const float2 sc = make_float2(scale, scale);
#pragma unroll
        for (int part = 0; part < 4; ++part) {
          uint32_t hi[8], lo[8];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float4 v = mine4[part * 2 + i], w = mine4[8 + part * 2 + i];
            split_f16(mul2(lo2(v), sc), hi[4 * i], lo[4 * i]);
            split_f16(mul2(hi2(v), sc), hi[4 * i + 1], lo[4 * i + 1]);
            split_f16(mul2(lo2(w), sc), hi[4 * i + 2], lo[4 * i + 2]);
            split_f16(mul2(hi2(w), sc), hi[4 * i + 3], lo[4 * i + 3]);
          }
          tm_st8(mine + kTmQ + 32 * half + 8 * part, hi);
          tm_st8(mine + kTmQ + 64 + 32 * half + 8 * part, lo);
        }
        tm_wait_st();
        tc_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&sm.qfull);
      }
      float2 o[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = make_float2(0.f, 0.f);
      // o stands for sum p v 2^(14 - share) against the maximum m, l for sum p
      float m = -INFINITY, share = kKtLeastShare, l = 0.0f, corr = 0.0f;
      const float cq = fmaxf(a.c * qinv, kLeastFactor);
      // tiles from this one on hold a key that some row of the unit does not see
      const int tend = cur.t0 + cur.n, tmask = cur.t0 - cur.off + (MASK == kMaskTree ? x.p : x.p + x.i0 + 1) / kKvTileKeys;
      // o = o * f + the O tile of tile w, whose P stood against the maximum and the share of then
      // (the tile's scales are still in place: their next writer waits for the PV after this)
      auto add_o = [&](int w, float f) {
        wait(&sm.ofull, w & 1);
        tc_after();
        const float2 f2 = make_float2(f, f);
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          uint32_t r[32];
          tm_ld32(mine + kTmO + 64 * half + 32 * part, r);
          tm_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i)
            o[part * 16 + i] =
                fma2(o[part * 16 + i], f2, make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])));
        }
        if (const unsigned long long bad = *reinterpret_cast<const unsigned long long*>(&sm.vbad[w & 3][0])) {
          const float2* vb = reinterpret_cast<const float2*>(
              a.v + (((size_t)x.b * a.hkv + x.hk) * (size_t)a.max_t + (size_t)(cur.off + w - cur.t0) * kKvTileKeys) * kKvD);
#pragma unroll 1
          for (int key = 0; key < kKvTileKeys; ++key) {
            if (!((bad >> key) & 1)) continue;
            const uint32_t hi = tm_ld1(mine + kTmP + 64 * (w & 1) + (key >> 1));
            const uint32_t lo = tm_ld1(mine + kTmP + 64 * (w & 1) + 32 + (key >> 1));
            tm_wait_ld();
            const int sh = (key & 1) * 16;
            float p = __half2float(__ushort_as_half((unsigned short)(hi >> sh))) +
                      __half2float(__ushort_as_half((unsigned short)(lo >> sh)));
            p *= __uint_as_float((254u << 23) - __float_as_uint(sm.vsc[w & 3][key]));  // over a power of 2
            if (p != 0.0f) {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float2 v = vb[(size_t)key * 64 + 4 * i + half], w2 = vb[(size_t)key * 64 + 4 * i + 2 + half];
                o[i].x = fmaf(p, v.x, o[i].x);
                o[i].y = fmaf(p, w2.x, o[i].y);
                o[16 + i].x = fmaf(p, v.y, o[16 + i].x);
                o[16 + i].y = fmaf(p, w2.y, o[16 + i].y);
              }
            }
            __syncwarp();
          }
        }
        tc_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&sm.ofree);
      };
      for (;; ++t) {
        float next = 1.0f;
        if (t < tend) {
        const int s = t & 1;
        const uint32_t sat = mine + kTmS + 64 * s + 32 * half;
        uint32_t see;
        auto look = [&]() { see = kv_sees<MASK>(a, x, row, (cur.off + t - cur.t0) * kKvTileKeys + 32 * half); };
        if (MASK == kMaskTree && t >= tmask) look();  // its loads beside the wait
        wait(&sm.sfull[s], (t >> 1) & 1);
        tc_after();
        wait(&sm.vinfo[t & 3], (t >> 2) & 1);
        float top = -INFINITY, heavy = -INFINITY;  // of the scores x, and of x - top + log2 w
        if (t >= tmask && MASK != kMaskTree) look();
#pragma unroll 1
        for (int part = 0; part < 2; ++part) {
          uint32_t r[16];
          float2 x[8];
          tm_ld16(sat + 16 * part, r);
          tm_wait_ld();
          if (t >= tmask) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (!((see >> (16 * part + e)) & 1u)) r[e] = 0xff800000u;  // -inf
          }
          // a key's scale, then the query's: one power of two of both may be 0.  Scores are rounded here, so
          // that the largest is the maximum itself at any size.
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float4 k4 = *reinterpret_cast<const float4*>(&sm.ksc[t & 3][32 * half + 16 * part + 4 * e]);
            x[2 * e] = times(mul2(make_float2(__uint_as_float(r[4 * e]), __uint_as_float(r[4 * e + 1])), lo2(k4)), cq);
            x[2 * e + 1] =
                times(mul2(make_float2(__uint_as_float(r[4 * e + 2]), __uint_as_float(r[4 * e + 3])), hi2(k4)), cq);
          }
          float up = top;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            up = fmaxf(fmaxf(up, x[e].x), x[e].y);
            r[2 * e] = __float_as_uint(x[e].x);
            r[2 * e + 1] = __float_as_uint(x[e].y);
          }
          tm_st16(sat + 16 * part, r);  // for the second pass
          const float h = up == -INFINITY ? 0.0f : -up;
          heavy += top + h;
          top = up;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float4 w4 = *reinterpret_cast<const float4*>(&sm.vlog[t & 3][32 * half + 16 * part + 4 * e]);
            const float2 y = add2(add2(x[2 * e], make_float2(h, h)), lo2(w4));
            const float2 z = add2(add2(x[2 * e + 1], make_float2(h, h)), hi2(w4));
            heavy = fmaxf(fmaxf(heavy, y.x), y.y);
            heavy = fmaxf(fmaxf(heavy, z.x), z.y);
          }
        }
        tm_wait_st();
        sm.top[s][half][row] = make_float2(top, heavy);
        meet();
        // maximum and share in whole powers of two: what stands against them is rescaled without rounding
        const float2 other = sm.top[s][half ^ 1][row];
        const float n_m = fmaxf(m, ceilf(fmaxf(top, other.x)));
        const float base = n_m == -INFINITY ? 0.0f : n_m, fall = m - base;
        const float n_share = fmaxf(fmaxf(share + fall, (float)kKtLeastShare),
                                    ceilf(fmaxf(heavy + (top - base), other.y + (other.x - base))));
        next = ex2(share + fall - n_share);
        l *= ex2(fall);
        m = n_m;
        share = n_share;
        const float2 b2 = make_float2(-base, -base);
        const float lift = ex2(kKtPScale - share);
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll 1
        for (int part = 0; part < 2; ++part) {
          uint32_t r[16], hi[8], lo[8];
          tm_ld16(sat + 16 * part, r);
          tm_wait_ld();
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float4 w4 = *reinterpret_cast<const float4*>(&sm.vsc[t & 3][32 * half + 16 * part + 2 * e]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float2 p = add2(make_float2(__uint_as_float(r[2 * (e + i)]), __uint_as_float(r[2 * (e + i) + 1])), b2);
              p.x = ex2(p.x);
              p.y = ex2(p.y);
              sum = add2(sum, p);
              split_f16(times(mul2(p, i ? hi2(w4) : lo2(w4)), lift), hi[e + i], lo[e + i]);
            }
          }
          tm_st8(mine + kTmP + 64 * s + 16 * half + 8 * part, hi);
          tm_st8(mine + kTmP + 64 * s + 32 + 16 * half + 8 * part, lo);
        }
        tm_wait_st();
        tc_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&sm.pfull[s]);
        l += sum.x + sum.y;
        }
        if (t > cur.t0) add_o(t - 1, corr);
        if (t == tend) break;
        corr = next;
      }
      // the row's sum over both halves (the maxima's place is free: the last tile's was read
      // before its P was given away, and t moves on)
      meet();
      sm.top[0][half][row].x = l;
      meet();
      l = sm.top[0][0][row].x + sm.top[0][1][row].x;
      meet();
      // the row: whole, or this CTA's part of it
      const bool whole = cur.off == 0 && cur.n == x.chunks;
      const size_t slot = 2 * (size_t)blockIdx.x + (cur.off > 0 ? 0 : 1);
      const float nan = __uint_as_float(0x7fffffffu);
      if (!kv_row_valid<MASK>(a, x, row)) m = -INFINITY;
      float f = ex2(share - kKtPScale);
      if (whole) f = m == -INFINITY ? 0.0f : __fdiv_rn(f, l);
      ok = ok && !*abort;  // another warp that went on without its data
      if (!ok) {  // NaN however the parts are joined: an infinite maximum leaves no other part a share
        f = l = nan;
        m = INFINITY;
      }
      {
        // 32 dimensions of the pair's 32 rows at a time, turned back and written by rows
        float* turn = &sm.turn[0][warp & 3][0][0];
        const int r0 = (warp & 3) * 32 + 16 * half + (lane >> 3);
        float4* dst[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = min(r0 + 4 * i, x.nrows - 1);
          dst[i] = reinterpret_cast<float4*>(whole ? a.out + kv_row_offset<MASK>(a, x, r)
                                                   : a.acc + (slot * a.rows + r) * kKvD) + (lane & 7);
        }
#pragma unroll
        for (int part = 0; part < 4; ++part) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int k = part * 8 + i;
            const float e0 = k & 1 ? o[k >> 1].y : o[k >> 1].x, e1 = k & 1 ? o[16 + (k >> 1)].y : o[16 + (k >> 1)].x;
            *reinterpret_cast<float2*>(turn + lane * 36 + 4 * i + 2 * half) =
                f == 0.0f ? make_float2(0.f, 0.f) : make_float2(e0 * f, e1 * f);
          }
          meet();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 v = *reinterpret_cast<const float4*>(turn + (16 * half + 4 * i + (lane >> 3)) * 36 + 4 * (lane & 7));
            if (r0 + 4 * i < x.nrows) dst[i][part * 8] = v;
          }
          meet();
        }
      }
      if (a.split && tid == 0 && cur.off == 0)  // for the merge: the first CTA, and how many there are
        a.begun[cur.u] = make_int2(blockIdx.x, 1 + (x.chunks - cur.n + sm.find.quota - 1) / sm.find.quota);
      if (row < x.nrows) {
        if (half == 0) {
          if (!whole) {
            a.stat[slot * 2 * a.rows + row] = m;
            a.stat[(slot * 2 + 1) * a.rows + row] = l;
          }
          if (a.norm && whole) a.norm[kv_row_number(a, x, row)] = row_norm(m, l);
        }
      }
    }
  }
  tc_before();
  __syncthreads();
  tc_after();
  if (warp == kKtMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kKtTmemCols) : "memory");
}

// After a split: the parts of the units that more than one CTA worked on, in the order of the CTAs, and
// zeros for units without keys.  A CTA has at most two parts: the rest of a unit that began before it (slot
// 2 cta) and the beginning of one that ends after it (slot 2 cta + 1).  A warp takes EACH rows of
// unit blockIdx.x and has eight parts' rows in flight.
constexpr int kKtMergeWarps = 8;
template <int MASK, int EACH>
__global__ void __launch_bounds__(kKtMergeWarps * 32) kv_tile_merge_kernel(const KvArgs a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r0 = (blockIdx.y * kKtMergeWarps + warp) * EACH;
  pdl_launch_dependents();
  pdl_wait();
  const KvUnit x = kv_unit<MASK>(a, blockIdx.x);
  if (r0 >= x.nrows) return;
  if (x.chunks == 0) {  // no CTA came by
    for (int r = r0; r < min(r0 + EACH, x.nrows); ++r) {
      reinterpret_cast<float4*>(a.out + kv_row_offset<MASK>(a, x, r))[lane] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (a.norm && lane == 0) a.norm[kv_row_number(a, x, r)] = make_float2(INFINITY, 0.0f);
    }
    return;
  }
  const int2 d = a.begun[blockIdx.x];
  const int parts = d.y;
  if (parts == 1) return;
  auto slot = [&](int s) { return 2 * ((size_t)d.x + s) + (s == 0 ? 1 : 0); };
  int row[EACH];
  float M[EACH], L[EACH];
  float4 A[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    row[i] = min(r0 + i, x.nrows - 1);
    M[i] = -INFINITY;
    L[i] = 0.0f;
    A[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int s = lane; s < parts; s += 32)
#pragma unroll
    for (int i = 0; i < EACH; ++i) M[i] = fmaxf(M[i], a.stat[slot(s) * 2 * a.rows + row[i]]);
#pragma unroll
  for (int i = 0; i < EACH; ++i)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M[i] = fmaxf(M[i], __shfl_xor_sync(kFull, M[i], o));
  for (int s0 = 0; s0 < parts; s0 += 32) {  // a lane per part for the factors, then a part at a time
    float f[EACH];
    const int s1 = s0 + lane;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      f[i] = 0.0f;
      if (s1 < parts && M[i] != -INFINITY) {
        f[i] = exp2f(a.stat[slot(s1) * 2 * a.rows + row[i]] - M[i]);
        if (f[i] != 0.0f) L[i] = fmaf(a.stat[(slot(s1) * 2 + 1) * a.rows + row[i]], f[i], L[i]);
      }
    }
    const int n = min(32, parts - s0);
    constexpr int kAhead = 8 / EACH;  // parts whose rows are loaded before one is used
    for (int s = 0; s < n; s += kAhead) {
      float4 v[kAhead][EACH];
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
#pragma unroll
        for (int i = 0; i < EACH; ++i)
          if (s + j < n)
            v[j][i] = ld_row(reinterpret_cast<const float4*>(a.acc + (slot(s0 + s + j) * a.rows + row[i]) * kKvD) + lane);
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
          const float fs = __shfl_sync(kFull, f[i], (s + j) & 31);
          if (s + j < n && fs != 0.0f)  // an empty part's sums stay out
            A[i] = make_float4(fmaf(v[j][i].x, fs, A[i].x), fmaf(v[j][i].y, fs, A[i].y), fmaf(v[j][i].z, fs, A[i].z),
                               fmaf(v[j][i].w, fs, A[i].w));
        }
    }
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const float sum = warp_sum(L[i]);
    if (r0 + i >= x.nrows) break;
    if (M[i] != -INFINITY)
      A[i] = make_float4(__fdiv_rn(A[i].x, sum), __fdiv_rn(A[i].y, sum), __fdiv_rn(A[i].z, sum), __fdiv_rn(A[i].w, sum));
    reinterpret_cast<float4*>(a.out + kv_row_offset<MASK>(a, x, row[i]))[lane] = A[i];
    if (a.norm && lane == 0) a.norm[kv_row_number(a, x, row[i])] = row_norm(M[i], sum);
  }
}

// ---------------------------------------------------------------------------------
// Column sums of the softmax of causal rows: weight[j] += sum over the rows that see key j of
// 2^(s_rj - m_r) / l_r, m_r and l_r the rows' maxima and sums, from every score once more.  The scores
// are the tile kernel's bit for bit: the same scale for every row and key, the same products in the same
// order, the same roundings.  (Any others, however exact, would give a row of large scores more or less
// than one unit in all: at scores of 2^24 a rounding is a factor of two.)  Keys are the M side
// (128 a CTA, hi / lo in TMEM, a thread owns a key), tiles of 64 rows the N side, so a key's sum
// stays in one register.  grid (key tiles, batch * hkv, splits): split z takes row tiles z, z +
// splits, ... and leaves its sums in part[z]; kv_column_add_kernel adds them in split order.
// Two CTAs per SM: 4 warps exponentials, 8 converters, 1 MMA; 24 MMAs of N = 64 a tile, about
// 820 cycles, beside 512 cycles of exponentials; what it waits for is the converters' chain of load,
// scale, split and hand-over.  4 x 1024 tokens, 16 heads on 2: 74 us, tensor pipe 24 % busy.
constexpr int kKcThreads = 416, kKcConvertWarp = 4, kKcMmaWarp = 12;
constexpr uint32_t kKcTmemCols = 256;
constexpr int kKcKeys = 128, kKcRows = 64;

struct KcSmem {
  alignas(1024) uint8_t q[2][2][2][kKcRows * 128];  // [stage][hi, lo][64 dims][row][128 B]
  alignas(16) float factor[4][kKcRows];             // from a product under the row's scale to its score
  alignas(16) float top[4][kKcRows], inv[4][kKcRows];  // the rows' -maxima and 1 / sums
  alignas(16) int last[4][kKcRows];                 // the last key a row sees
  alignas(16) float turn[4][32 * 20];               // rows of a warp's keys: memory <-> a thread per key
  alignas(8) uint64_t qfull[2], qfree[2], info[4], sfull[2], sfree[2], kfull, done;
  uint32_t tmem;
  int abort;
};

__global__ void __launch_bounds__(kKcThreads, 2)
kv_column_tile_kernel(const KvArgs a, float* weight, float* __restrict__ part, uint64_t wait_ns) {
  extern __shared__ uint8_t kt_raw[];
  KcSmem& sm = *reinterpret_cast<KcSmem*>(kt_raw + ((1024 - (su32(kt_raw) & 1023)) & 1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort = &sm.abort;
  if (tid == 0) {
    s_kt_wait_ns = wait_ns;
    for (int i = 0; i < 2; ++i) {
      bar_init(&sm.qfull[i], 8);
      bar_init(&sm.qfree[i], 1);
      bar_init(&sm.sfull[i], 1);
      bar_init(&sm.sfree[i], 4);
    }
    for (int i = 0; i < 4; ++i) bar_init(&sm.info[i], 8);
    bar_init(&sm.kfull, 4);
    bar_init(&sm.done, 1);
    sm.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kKcMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(&sm.tmem)),
                 "r"(kKcTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.y / a.hkv, hk = blockIdx.y - b * a.hkv;
  const int p = a.pos[b], rows = a.n * a.group;
  const int keys = (p < 0 || p >= a.max_t) ? 0 : min(p + a.n, a.max_t);
  const int j0 = blockIdx.x * kKcKeys;
  // row tiles first, first + splits, ...: from the one that holds the first row to see a key
  const int splits = gridDim.z;
  const int seen = j0 < keys ? (int)(((int64_t)max(0, j0 - p) * a.group) / kKcRows) : 0;
  const int first = seen + blockIdx.z;
  const int tiles = j0 < keys ? (rows + kKcRows - 1) / kKcRows : 0;
  const int n = first < tiles ? (tiles - 1 - first) / splits + 1 : 0;
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = sm.tmem;
  const size_t bh = blockIdx.y;

  if (warp >= kKcConvertWarp && warp < kKcMmaWarp) {
    // ---------------- converters: query rows 8 cw .. + 8 of every tile ----------------
    const int cw = warp - kKcConvertWarp, h = lane & 15, ky = lane >> 4;
    const float4* qb = reinterpret_cast<const float4*>(a.q + ((size_t)b * a.n * a.hq + hk * a.group) * kKvD) + h;
    const int there = keys - p <= 0 ? 0 : min(rows, (keys - p) * a.group);  // rows inside the cache
    float4 qr[8];
    const unsigned row0 = blockIdx.y * (unsigned)rows;  // all rows together are fewer than 2^31
    float constant;  // of row lane % 8: maximum (lanes below 8), 1 / sum (16), scale (24)
    auto load = [&](int rt) {
      const int rl = rt * kKcRows + cw * 8 + (lane & 7);
      constant = lane < 8 ? INFINITY : lane < 16 ? 0.0f : 1.0f;
      if (rl < there)
        constant = lane < 16 ? reinterpret_cast<const float*>(a.norm)[2 * (row0 + rl) + (lane >> 3)] : a.qscale[row0 + rl];
      const int r = rt * kKcRows + cw * 8 + ky;
      int tok = r / a.group, head = r - tok * a.group;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        qr[2 * i] = qr[2 * i + 1] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r + 2 * i < there) {
          const float4* row = qb + ((size_t)tok * a.hq + head) * (kKvD / 4);
          qr[2 * i] = row[0];
          qr[2 * i + 1] = row[16];
        }
        head += 2;  // the row after the next, with no division
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (head >= a.group) {
            head -= a.group;
            ++tok;
          }
      }
    };
    bool dead = false;
    if (n > 0) load(first);
    for (int t = 0; t < n; ++t) {
      const int s = t & 1, rt = first + t * splits;
      if (t >= 2 && !dead) dead = !bar_wait(&sm.qfree[s], ((t >> 1) - 1) & 1, abort);
      uint8_t* dst = &sm.q[s][0][h >> 3][(cw * 8 + ky) * 128];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float scale = __shfl_sync(kFull, constant, 16 + 2 * i + ky);
        uint4 hi, lo;
        split_f16(times(lo2(qr[2 * i]), scale), hi.x, lo.x);
        split_f16(times(hi2(qr[2 * i]), scale), hi.y, lo.y);
        split_f16(times(lo2(qr[2 * i + 1]), scale), hi.z, lo.z);
        split_f16(times(hi2(qr[2 * i + 1]), scale), hi.w, lo.w);
        const int at = i * 256 + (((h & 7) ^ (2 * i + ky)) << 4);
        *reinterpret_cast<uint4*>(dst + at) = hi;
        *reinterpret_cast<uint4*>(dst + sizeof(sm.q[0][0]) + at) = lo;
      }
      const int at = cw * 8 + (lane & 7);
      if (lane < 8) {
        sm.top[t & 3][at] = -constant;
        sm.last[t & 3][at] = p + (rt * kKcRows + at) / a.group;
      } else if (lane < 16) {
        sm.inv[t & 3][at] = constant;
      } else if (lane < 24) {
        sm.factor[t & 3][at] = fmaxf(a.c * __uint_as_float((254u << 23) - __float_as_uint(constant)), kLeastFactor);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        bar_arrive(&sm.qfull[s]);
        bar_arrive(&sm.info[t & 3]);
      }
      if (t + 1 < n) load(rt + splits);
    }
  } else if (warp == kKcMmaWarp) {
    constexpr uint32_t id = kt_idesc(kKcRows);
    bool ok = n == 0 || bar_wait(&sm.kfull, 0, abort);
    for (int t = 0; ok && t < n; ++t) {
      const int s = t & 1;
      ok = bar_wait(&sm.qfull[s], (t >> 1) & 1, abort);
      if (ok && t >= 2) ok = bar_wait(&sm.sfree[s], ((t >> 1) - 1) & 1, abort);
      if (!ok) break;
      tc_after();
      __syncwarp();
      if (elected()) {
        mma_pairs<8, sizeof(sm.q[0][0][0]), true>(tmem + 128 + 64 * s, tmem, tmem + 64, sm.q[s][0][0], sm.q[s][1][0], id);
        mma_commit(&sm.qfree[s]);
        mma_commit(&sm.sfull[s]);
      }
      __syncwarp();
    }
    if (elected()) mma_commit(&sm.done);
    __syncwarp();
    mb_wait_ns(su32(&sm.done), 0, kDrainLimitNs, nullptr);
  } else if (warp < kKcConvertWarp) {
    // ---------------- a key per thread ----------------
    const uint32_t mine = tmem + ((uint32_t)(warp * 32) << 16);
    const int j = j0 + tid;
    float kinv = 0.0f;
    if (n > 0) {
      // the warp reads its 32 rows and turns them (see the tile kernel's query rows)
      const float4* kr = reinterpret_cast<const float4*>(a.k + bh * a.max_t * kKvD);
      const int row0 = j0 + warp * 32;
      unsigned m = 0;
#pragma unroll 8
      for (int i = 0; i < 32; ++i) {
        const float4 v = kr[(size_t)min(row0 + i, keys - 1) * 32 + lane];
        const unsigned top = __reduce_max_sync(kFull, __float_as_uint(mag(mag(mag(mag(0.0f, v.x), v.y), v.z), v.w)));
        if (i == lane) m = top;
      }
      // the scale that row_scales gives the key
      if (j >= keys) m = 0;
      unsigned top = m;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(kFull, top, o));
      const bool even = (__ballot_sync(kFull, m >= near_of(top)) >> (lane & 24) & 255u) == 255u && top < 0x7f800000u;
      float scale;
      scale_of(even ? top : m, scale, kinv);
      const float2 sc = make_float2(scale, scale);
      float4* turn = reinterpret_cast<float4*>(&sm.turn[warp][0]);
#pragma unroll
      for (int part = 0; part < 8; ++part) {  // dimensions 8 part .. + 8 and 64 + 8 part .. + 8
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 8 * i + (lane >> 2), c = lane & 3;
          turn[r * 5 + c] = kr[(size_t)min(row0 + r, keys - 1) * 32 + (c >> 1) * 16 + part * 2 + (c & 1)];
        }
        __syncwarp();
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 v = turn[lane * 5 + i], w = turn[lane * 5 + 2 + i];
          split_f16(mul2(lo2(v), sc), hi[4 * i], lo[4 * i]);
          split_f16(mul2(hi2(v), sc), hi[4 * i + 1], lo[4 * i + 1]);
          split_f16(mul2(lo2(w), sc), hi[4 * i + 2], lo[4 * i + 2]);
          split_f16(mul2(hi2(w), sc), hi[4 * i + 3], lo[4 * i + 3]);
        }
        tm_st8(mine + 8 * part, hi);
        tm_st8(mine + 64 + 8 * part, lo);
        __syncwarp();
      }
      tm_wait_st();
      tc_before();
      __syncwarp();
      if (lane == 0) bar_arrive(&sm.kfull);
    }
    bool ok = true;
    float2 sum = make_float2(0.f, 0.f);
    for (int t = 0; ok && t < n; ++t) {
      const int s = t & 1;
      ok = bar_wait(&sm.info[t & 3], (t >> 2) & 1, abort) && bar_wait(&sm.sfull[s], (t >> 1) & 1, abort);
      if (!ok) break;
      tc_after();
      // rows from this one on see the whole key tile
      const bool masked = p + (first + t * splits) * kKcRows / a.group < j0 + kKcKeys - 1;
#pragma unroll 1
      for (int part = 0; part < 2; ++part) {
        uint32_t r[32];
        tm_ld32(mine + 128 + 64 * s + 32 * part, r);
        tm_wait_ld();
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float4 c4 = *reinterpret_cast<const float4*>(&sm.factor[t & 3][32 * part + 4 * e]);
          const float4 m4 = *reinterpret_cast<const float4*>(&sm.top[t & 3][32 * part + 4 * e]);
          const float4 v4 = *reinterpret_cast<const float4*>(&sm.inv[t & 3][32 * part + 4 * e]);
          // the product is rounded to the score, as in the tile kernel; the key's scale, a power of two, passes
          // through the sum exactly
          float2 x = mul2(make_float2(__uint_as_float(r[4 * e]), __uint_as_float(r[4 * e + 1])), lo2(c4));
          float2 y = mul2(make_float2(__uint_as_float(r[4 * e + 2]), __uint_as_float(r[4 * e + 3])), hi2(c4));
          x = fma2(x, make_float2(kinv, kinv), lo2(m4));
          y = fma2(y, make_float2(kinv, kinv), hi2(m4));
          x = make_float2(ex2(x.x), ex2(x.y));
          y = make_float2(ex2(y.x), ex2(y.y));
          if (masked) {
            const int4 la = *reinterpret_cast<const int4*>(&sm.last[t & 3][32 * part + 4 * e]);
            x.x = j <= la.x ? x.x : 0.0f;
            x.y = j <= la.y ? x.y : 0.0f;
            y.x = j <= la.z ? y.x : 0.0f;
            y.y = j <= la.w ? y.y : 0.0f;
          }
          sum = fma2(x, lo2(v4), sum);
          sum = fma2(y, hi2(v4), sum);
        }
      }
      tc_before();
      __syncwarp();
      if (lane == 0) bar_arrive(&sm.sfree[s]);  // after the last look at the tile's constants too
    }
    if (j < keys) {
      const float w = ok && !*abort ? sum.x + sum.y : __uint_as_float(0x7fffffffu);
      if (part)
        part[((size_t)blockIdx.z * gridDim.y + bh) * a.max_t + j] = w;
      else
        weight[bh * a.max_t + j] += w;
    }
  }
  tc_before();
  __syncthreads();
  tc_after();
  if (warp == kKcMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kKcTmemCols) : "memory");
}

__global__ void __launch_bounds__(256)
kv_column_add_kernel(const float* __restrict__ part, const int* __restrict__ pos, int n, int hkv, int max_t, int splits,
                     float* __restrict__ weight) {
  pdl_launch_dependents();
  pdl_wait();
  const int bh = blockIdx.y, p = pos[bh / hkv], j = blockIdx.x * 256 + threadIdx.x;
  if (p < 0 || p >= max_t || j >= min(p + n, max_t)) return;
  float s = 0.0f;
  for (int z = 0; z < splits; ++z) s += part[((size_t)z * gridDim.y + bh) * max_t + j];
  weight[(size_t)bh * max_t + j] += s;
}

// Row splits of the column sums: about 592 CTAs (two for each of two places on an SM) over the
// keys of the new rows alone, 8 row tiles a CTA at least (its start costs as much as some tiles).
// (4 x 1024 tokens with 256, 444 and 592 CTAs: 198, 193 and 190 us for the whole call.)
int column_splits(int batch, int n, int hkv, int group) {
  const int64_t tiles = ((int64_t)n * group + kKcRows - 1) / kKcRows;
  const int64_t places = (int64_t)batch * hkv * ((n + kKcKeys - 1) / kKcKeys);
  const int64_t want = (592 + places - 1) / places;
  const int64_t most = tiles / 8 > 64 ? 64 : tiles / 8;
  return (int)(want < most ? want : most < 1 ? 1 : most);
}

template <int MASK>
cudaError_t launch_tile(const KvArgs& a, int device, cudaStream_t s) {
  static int configured[128] = {0};
  const size_t smem = sizeof(KtSmem) + 1024;
  cudaError_t e = ensure_smem((const void*)kv_tile_kernel<MASK>, configured, device, smem, false);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kKvGrid);
  cfg.blockDim = dim3(kKtThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, kv_tile_kernel<MASK>, a, wait_limit_ns());
  if (e != cudaSuccess || !a.split) return e;
  // Few units have few rows, of many parts each: a warp per row.  With many, the CTAs' starts count.
  // (A tree over 2 units of 63 parts 68 us with four rows a warp, 33 with one; 30 units of 4 parts 37
  // and 33; 64 units of 3 parts 157 and 159.)
  const int rows = a.units > a.batch * a.hkv ? kKvTileRows : a.n * a.group;  // of the largest unit
  const int each = a.units <= kKvGrid / 4 ? 1 : 4;
  cfg.gridDim = dim3((unsigned)a.units, (unsigned)((rows + kKtMergeWarps * each - 1) / (kKtMergeWarps * each)));
  cfg.blockDim = dim3(kKtMergeWarps * 32);
  cfg.dynamicSmemBytes = 0;
  return each == 1 ? cudaLaunchKernelEx(&cfg, kv_tile_merge_kernel<MASK, 1>, a)
                   : cudaLaunchKernelEx(&cfg, kv_tile_merge_kernel<MASK, 4>, a);
}

}  // namespace

cudaError_t launch_kv_tile(const KvArgs& a, int mask, int device, cudaStream_t s) {
  return mask == kMaskTree ? launch_tile<kMaskTree>(a, device, s) : launch_tile<kMaskCausal>(a, device, s);
}

size_t kv_column_tile_bytes(int batch, int n, int hq, int hkv, int max_t) {
  const int splits = column_splits(batch, n, hkv, hq / hkv);
  return splits > 1 ? (size_t)splits * batch * hkv * max_t * 4 : 0;
}

cudaError_t launch_kv_column_tile(const KvArgs& a, float* weight, float* part, int device, cudaStream_t s) {
  static int configured[128] = {0};
  const size_t smem = sizeof(KcSmem) + 1024;
  cudaError_t e = ensure_smem((const void*)kv_column_tile_kernel, configured, device, smem, true);
  if (e != cudaSuccess) return e;
  const int splits = column_splits(a.batch, a.n, a.hkv, a.group);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.max_t + kKcKeys - 1) / kKcKeys), (unsigned)(a.batch * a.hkv), (unsigned)splits);
  cfg.blockDim = dim3(kKcThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, kv_column_tile_kernel, a, weight, splits > 1 ? part : nullptr, wait_limit_ns());
  if (e != cudaSuccess || splits == 1) return e;
  cfg.gridDim = dim3((unsigned)((a.max_t + 255) / 256), (unsigned)(a.batch * a.hkv));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, kv_column_add_kernel, (const float*)part, a.pos, a.n, a.hkv, a.max_t, splits, weight);
}

cudaError_t read_kv_tile_fault(unsigned int* flags, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(flags, g_kv_tile_fault, sizeof(unsigned int));
  if (e == cudaSuccess && clear) {
    const unsigned int z = 0;
    e = cudaMemcpyToSymbol(g_kv_tile_fault, &z, sizeof(z));
  }
  return e;
}

}  // namespace q8lin
