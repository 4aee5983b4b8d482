// Attention of new tokens over a paged cache on tcgen05 (bf16 activations, heads of 64 or 128; pages in bf16, e4m3, int8 or 4 bits), and
// of whole prompts, whose keys and values are packed rows (KIND PG_ROWS).
// Mathematics and division of the work: paged_attend.cu, paged.cuh.
//
// One persistent CTA an SM; two softmax warpgroups X = 0, 1 of a row per thread.  An item is a block of (token, head of the group)
// rows of a sequence against the key tiles of 128 that they see:
//   chunks:  up to 256 rows, X = rows 0..127 and 128..255 against the same key tile; 128 rows or fewer: X = the even and the odd tiles;
//   steps (FEW, where a sequence has few rows): up to 32 rows, X = the even and the odd tiles, and the rows lie in the 128 of the
//     query tile four times (or eight, see below): warp w of a warpgroup has a row per thread as well, but only keys 32 w ..
//     32 w + 31 of a tile (its probabilities of the others are 0), with a maximum, a sum and an O of its own.  One warp of four
//     would have all the work otherwise, and a tile's softmax would be the longest link of the chain.
// Parts of a row with sums of their own are joined through shared memory when the item ends.
// P is rounded to bf16, which adds to a result about as much as its own rounding does.  Steps of up to 16 rows leave 16 lanes of each
// warp idle; there the rows lie in the tile eight times, and the other copy multiplies what the rounding of the first one left: the
// output's rounding alone remains, at no cost.
// Roles: warp 0 copies pages by TMA (128-byte swizzle) into a ring of K and V tiles, in the order in which they are used; warp 1
// issues  S_X = Q_X K^T  (M = N = 128) into 128 columns of tensor memory and  O_X += P_X V  with P_X, written by the softmax over
// S_X's columns, as the operand from tensor memory and V as an MN-major operand from the same kind of tile (tcgen05.mma of one CTA
// complete in the order of issue, so S_X of the next tile may follow P_X V); warps 2 and 3 fetch the next item's queries, with 8-bit
// pages its scales too, but in steps over bf16 pages warp 2 copies the values' pages and warp 0 the keys'.
// 8-bit pages: four more warps turn the copied payloads into bf16 tiles (exactly: a payload has at most 7 bits of mantissa;
// only e4m3's codes of NaN become 480, and where a tile has one the rows that may see it are summed again);
// a row's scale multiplies its logit, or its probability before that is rounded to bf16.
// 4-bit pages: the same warps make the values themselves, a scale for 32 channels included ((u - 8) s with s of 5 bits has 8 bits at most:
// exact), so that the softmax has no scales to apply.  Packed rows: a tile is a box of a tensor map over tokens, and what follows a
// sequence in it is the next one's: masked, its values cleared like those behind the end in a last page.
// Both of these (OPEN) take blocks of whole tokens, 128 / G * G rows a warpgroup, whose queries are two or four copies of a tensor map (through two
// warps they came 5000 clocks after the item before had been stored), count the ends of items in the division (paged.cuh), and leave out
// masks, and halves of a tile, where a warp's rows have no edge.
//
// The running maximum of a row is raised, and O_X rescaled, only when a tile exceeds it by 2^8: probabilities up to 256 lose
// nothing in bf16 or in the fp32 sums, and the accumulator makes its way through registers only a few times a row.
//
// Keys behind a sequence's end read as zeros where a whole page is missing (an out-of-range coordinate of the copy); in its last page
// the softmax clears the value rows behind it, whatever earlier tokens left there.  A key that only some rows of a tile see has
// p = 0 in the others, which is no mask for an infinity or a NaN: O shows it, and such a row is summed again key by key, reading only
// what it sees (pt_slow_row).  Every wait is bounded (status word, see kch_device_status).
//
// Measured, 16 heads of 128 on 4.  Steps of 64 sequences over 8192 tokens, pages of 64: 169 us, 6.4 TB/s, the memory's rate; 500 to
// 16000 tokens, pages of 16 and more 176 us, of 8 198 (a tile is 16 or 32 copies then: with one warp copying keys and values pages of
// 16 and 8 took 196 and 322, and with each page asked for where it was needed and not a tile ahead pages of 16 took 263).
// A chunk of 4096 tokens behind 28672: 827 us, 1247 TFLOP/s, in a burst, and 1000 us in a long run, where the power limit holds the
// clock at 1.6 GHz.  A step of it is 3500 clocks, 2048 of them products: scores 512, maximum 350, powers 1500 (a pair of four by FMAs then), value product 512,
// hand-overs 500, and two warpgroups that take turns.  Powers by FMAs (POLY) help heads of 64 alone, whose products are half as long: 32 of
// them 1486 us with one pair of four, 1579 with none, 1623 with two; heads of 128 827 with none, 825 with one, 932 against 878 with two.
// Neither did P handed over in halves (883 where the rest took 878) shorten it, nor the maximum and P in one pass (996, registers).  fp8
// pages: 1210 us, the conversion's ALU operations and the scales' products (6000 clocks a step; all powers are the special-function unit's, for
// the FMAs have the scales: 1281 with one pair of four, and 124 against 119 for a ragged batch of 24 sequences with a window of 1000).
// Short items cost their ends: 37 x 16 items of 256 rows and 9 tiles take 117 us, four to a CTA, of which steps are 75: 10000 clocks
// until a CTA's first scores, as many for the first end (its code comes from memory), then 6000 an end and 3000 until the next item's
// scores (its queries: 12000 clocks for two warps' copies, most of them behind the last softmax).
// Prompts, 16 heads of 128 on 4 (OPEN; before the three measures above): one of 8192 tokens 257 us (351), 37 of 20 to 1500 184 (316), 64 of 512 147
// (188); two of 8300 and 14001 on 2 key heads 1042 (1317), 1200 TFLOP/s in a burst.  An item's first scores are there 600 clocks after the one before it, its end
// takes 5000 (900 until the last product, 3700 to store its rows); a step of a long prompt is 3430, a masked one up to 5000.  Chunks over 4-bit pages: 1024
// tokens behind 15360 155 us, where bf16 pages take 142.
#include <cuda.h>
#include <math.h>

#include <atomic>
#include <type_traits>

#include "paged.cuh"
#include "tc5_utils.cuh"

#define PT_KT 128
// Polls of a wait, eight seconds: a warp that sums its 32 rows again makes the others wait 5 us a key, so that the limit is 1.6 million keys
// in the part that a CTA has of them.
#define PT_SPIN (1u << 28)

template <int D, int KIND, int FEW>
struct PtCfg {
  static constexpr int R = FEW ? FEW : 256, TWO = FEW ? FEW : 128, COPIES = FEW ? 128 / FEW : 1;
  static constexpr bool ROWS = KIND == PG_ROWS, Q4 = KIND == KCH_INT4, Q8 = KIND == KCH_FP8_E4M3 || KIND == KCH_INT8;
  static constexpr bool OPEN = ROWS || Q4;               // blocks of whole tokens (a.bt.rows), whose queries a tensor map's copies fetch
  static constexpr bool CODES = Q8 || Q4;                // pages hold codes, which a warpgroup turns into tiles
  static constexpr bool APART = FEW && !CODES;           // keys' and values' pages are copied by a warp each
  static constexpr int PANELS = D / 64, TILE = PT_KT * D * 2, RAW = Q4 ? PT_KT * D / 2 : PT_KT * D, GROUPS = D / 32;      // (GROUPS: scales of a row, Q4)
  static constexpr int RAW_ALL = RAW + (Q4 ? PT_KT * GROUPS * 2 : 0);      // with 4 bits' scales behind them
  static constexpr int STAGES = Q8 ? (D == 128 ? 3 : 6) : Q4 ? (D == 128 ? 4 : 7) : (D == 128 ? 5 : 8), RAWS = CODES ? (D == 128 ? 3 : 6) : 0;
  // of 4 pairs: how many powers are FMAs' and not the special-function unit's
  static constexpr int POLY = D == 64 && !FEW && !CODES ? 1 : 0;
  static constexpr int SCALES = 4;                       // key tiles whose scales are held
  static constexpr int THREADS = CODES ? 512 : 384;
  // registers of the warpgroups, and of a thread at launch
  static constexpr int REG_FEED = CODES ? 80 : 88, REG_SOFT = CODES ? 168 : 208, REG_CONV = 88, REG_LAUNCH = 65536 / THREADS / 8 * 8;
  static_assert(128 * (REG_FEED + 2 * REG_SOFT + (CODES ? REG_CONV : 0)) <= THREADS * REG_LAUNCH, "register split");
};

// 32 bytes of a row.  (The lanes' rows are as many lines, one a cycle: half of 16 bytes' stores.)
__device__ __forceinline__ void pt_store8(void* p, const uint32_t* v, bool wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
                 "r"(v[6]), "r"(v[7]) : "memory");
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(v[0], v[1], v[2], v[3]);
    *(reinterpret_cast<uint4*>(p) + 1) = make_uint4(v[4], v[5], v[6], v[7]);
  }
}

template <int D, int KIND, int FEW>
struct PtSmem {
  typedef PtCfg<D, KIND, FEW> C;
  alignas(1024) uint8_t q[2][128 * D * 2];
  alignas(1024) uint8_t kv[C::STAGES][C::TILE];
  alignas(C::CODES ? 1024 : 16) uint8_t raw[C::RAWS ? C::RAWS : 1][C::RAWS ? C::RAW_ALL : 16];
  alignas(16) float scale[C::Q8 ? C::SCALES : 1][2][C::Q8 ? PT_KT : 4];
  float ml[2][256];                                      // maxima and sums of the parts of an item's keys
  float factor[2][32];                                   // of its rows: 1 / the denominator
  uint32_t odd[2];                                       // rows of it that are not finite, by column half
  uint32_t nan_code;                                     // e4m3: a code of NaN among the tiles so far
  alignas(8) uint64_t full[C::STAGES], empty[C::STAGES];
  uint64_t raw_full[C::RAWS ? C::RAWS : 1], raw_empty[C::RAWS ? C::RAWS : 1];
  uint64_t sc_full[C::SCALES], sc_empty[C::SCALES];
  uint64_t q_full, q_empty, s_full[2], p_full[2], pv_done[2];
  uint32_t tmem;
};
static_assert(sizeof(PtSmem<128, KCH_BF16, 0>) <= 232448 && sizeof(PtSmem<128, KCH_INT8, 0>) <= 232448 && sizeof(PtSmem<128, KCH_INT4, 0>) <= 232448, "shared memory of the paged attention");
static_assert(PG_PLAN_BYTES(PG_MAX_B) <= 4 * 16384, "the plan lies in the ring of tiles");

__device__ __forceinline__ void pt_tma_4d(void* dst, const void* map, int c0, int c1, int c2, int c3, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_addr_u32(dst)), "l"(map), "r"(smem_addr_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}
__device__ __forceinline__ void pt_tma_3d(void* dst, const void* map, int c0, int c1, int c2, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_addr_u32(dst)), "l"(map), "r"(smem_addr_u32(bar)), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void pt_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void pt_arrive_n(uint64_t* bar, uint32_t n) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr_u32(bar)), "r"(n) : "memory");
}
__device__ __forceinline__ void pt_st(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void pt_st(uint32_t taddr, const uint32_t (&r)[32]) { t5_st32(taddr, r); }
__device__ __forceinline__ void pt_ld(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void pt_ld(uint32_t taddr, uint32_t (&r)[32]) { t5_ld32(taddr, r); }
// pairs of fp32 values: one issue slot for two of them
__device__ __forceinline__ uint64_t pt_pack(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void pt_unpack(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t pt_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t pt_mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ void pt_scale2(uint32_t& x0, uint32_t& x1, uint64_t f) {
  float a, b;
  pt_unpack(pt_mul2(pt_pack(__uint_as_float(x0), __uint_as_float(x1)), f), a, b);
  x0 = __float_as_uint(a);
  x1 = __float_as_uint(b);
}
__device__ __forceinline__ uint64_t pt_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 2^x of a pair by FMAs: x = n + f, |f| <= 1/2, 2^f by the polynomial of degree 4 whose largest relative error is smallest (2.6e-6;
// Remez exchange), times 2^n.  A NaN stays one through the clamp and the product (added to the exponent, n would make a number of it),
// and 2^-127, for everything below -126.5 and -inf too, is an exponent of 0: a key that is masked or weighs nothing gets 0.
__device__ __forceinline__ float pt_clamp(float x) {
  float r;
  asm("max.NaN.f32 %0, %1, 0fC2FE0000;" : "=f"(r) : "f"(x));      // -127
  return r;
}
__device__ __forceinline__ void pt_ex2_fma(float& x0, float& x1) {
  const uint64_t big = pt_pack(12583039.f, 12583039.f), x = pt_pack(pt_clamp(x0), pt_clamp(x1));      // 1.5 * 2^23 + 127
  const uint64_t t = pt_add2(x, big), n = pt_add2(t, pt_pack(-12583039.f, -12583039.f)), f = pt_fma2(n, pt_pack(-1.f, -1.f), x);
  uint64_t p = pt_fma2(f, pt_pack(0.009570102207362652f, 0.009570102207362652f), pt_pack(0.05591785907745361f, 0.05591785907745361f));
  p = pt_fma2(p, f, pt_pack(0.240247443318367f, 0.240247443318367f));
  p = pt_fma2(p, f, pt_pack(0.6931217908859253f, 0.6931217908859253f));
  p = pt_fma2(p, f, pt_pack(0.9999992847442627f, 0.9999992847442627f));
  float t0, t1;
  pt_unpack(t, t0, t1);
  pt_unpack(pt_mul2(p, pt_pack(__uint_as_float(__float_as_uint(t0) << 23), __uint_as_float(__float_as_uint(t1) << 23))), x0, x1);
}
// bits [lo, hi) of a 32-bit word (any lo, hi)
__device__ __forceinline__ uint32_t pt_range(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 32);
  return hi > lo ? (0xFFFFFFFFu >> (32 - (hi - lo))) << lo : 0u;
}
// two bf16 values from two 8-bit codes, exactly (but see `most`)
// (as FMAs: mul and sub of bf16 pairs become conversions to fp32 and back, and 4500 cycles for a tile of 128 x 128 instead of ~900)
__device__ __forceinline__ uint32_t pt_bf16_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// most: e4m3, the largest of the codes without their signs; a NaN's (which comes out as 480) is the largest of all, 0x7F0
template <int KIND>
__device__ __forceinline__ void pt_codes4(uint32_t w, uint32_t& lo, uint32_t& hi, uint32_t& most) {
  if (KIND == KCH_FP8_E4M3) {
    // sign, exponent and mantissa moved to their places are 2^-120 of the value (subnormal codes become subnormal bf16 values)
    const uint32_t a = __byte_perm(w, 0u, 0x1404), b = __byte_perm(w, 0u, 0x3424), sa = (a >> 4) & 0x07F007F0u, sb = (b >> 4) & 0x07F007F0u;
    lo = pt_bf16_fma((a & 0x80008000u) | sa, 0x7B807B80u, 0x80008000u);
    hi = pt_bf16_fma((b & 0x80008000u) | sb, 0x7B807B80u, 0x80008000u);
    most = __vimax3_u16x2(most, sa, sb);
  } else {
    // 128 + the low 7 bits, less 256 or 128 by the sign
    const uint32_t a = __byte_perm(w, 0x43434343u, 0x5140), b = __byte_perm(w, 0x43434343u, 0x7362);
    lo = pt_bf16_fma(a & 0xFF80FF80u, 0xBF80BF80u, a & 0xFF7FFF7Fu);
    hi = pt_bf16_fma(b & 0xFF80FF80u, 0xBF80BF80u, b & 0xFF7FFF7Fu);
  }
}

// 8 channels in bf16 from a word of 4-bit codes, times their scale: the code's place in the mantissa of 16 makes 16 + u of it, and
// (16 + u) s - 24 s = (u - 8) s has at most 8 bits where s has 5: exact.  s, s24: pairs of the scale and -24 times it.
__device__ __forceinline__ void pt_nibbles8(uint32_t w, uint32_t s, uint32_t s24, uint4& x) {
  const uint32_t even = w << 3, odd = w >> 1;            // (of each byte the lower and the upper code, in its bits 3 .. 6)
  x.x = pt_bf16_fma((__byte_perm(even, odd, 0x4400) & 0x00780078u) | 0x41804180u, s, s24);
  x.y = pt_bf16_fma((__byte_perm(even, odd, 0x5511) & 0x00780078u) | 0x41804180u, s, s24);
  x.z = pt_bf16_fma((__byte_perm(even, odd, 0x6622) & 0x00780078u) | 0x41804180u, s, s24);
  x.w = pt_bf16_fma((__byte_perm(even, odd, 0x7733) & 0x00780078u) | 0x41804180u, s, s24);
}

// Is there a code of NaN (0x7F, 0xFF) among the keys [from, to) of a sequence, or their values?  A warp's.
template <int D>
__device__ __noinline__ bool pt_nan_among(const PgAttend& a, int b, int h, int from, int to) {
  constexpr int PIECES = D / 16;
  const int lane = threadIdx.x & 31;
  uint32_t x = 0u;
#pragma unroll 4
  for (int j = from + lane / PIECES; j < to; j += 32 / PIECES) {
    const int page = __ldg(a.bt.table + b * a.bt.ld_table + (j >> a.bt.shift));
    if ((unsigned)page >= (unsigned)a.bt.num_pages) continue;
    const int64_t at = (((int64_t)page * a.bt.n_kv + h) * a.page + (j & (a.page - 1))) * PIECES + lane % PIECES;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(kv ? a.v : a.k) + at);
      x |= ((u.x & 0x7F7F7F7Fu) + 0x01010101u) | ((u.y & 0x7F7F7F7Fu) + 0x01010101u) | ((u.z & 0x7F7F7F7Fu) + 0x01010101u) | ((u.w & 0x7F7F7F7Fu) + 0x01010101u);
    }
  }
  return __any_sync(0xffffffffu, (x & 0x80808080u) != 0u);
}

// One row on one warp over the keys [from, to), reading only those: sum_j round(p_j) v_j, p_j = 2^(s_j sc - shift); columns
// c0 .. c1 of it go to `dst` (fp32, a part) or `out` (times f, rounded).  16 keys at a time (4 bits, whose scales take
// registers too: 8), a lane with D / 32 channels of each; their pages are asked for as many keys ahead, and the sums of the lanes are halved
// over and over until lane l has that of key l mod 16: 0.15 us a key on
// all warps.  (With each key's page asked for where it is needed, and a sum of its own, 0.5 us.)
template <int D, int KIND>
__device__ __noinline__ void pt_slow_row(const PgAttend& a, int b, int row0, int h, const bf16* q, int from, int to, float sc, float shift,
                                         float f, bf16* out, float* dst, int c0, int c1) {
  typedef PtCfg<D, KIND, 0> C;
  constexpr bool Q8 = C::Q8, Q4 = C::Q4, ROWS = C::ROWS;
  constexpr int E = D / 32, BYTES = Q4 ? E / 2 : Q8 ? E : 2 * E, U = Q4 ? 8 : 16;      // channels and bytes of a lane, keys in flight
  typedef typename std::conditional<BYTES == 8, uint2, typename std::conditional<BYTES == 4, uint32_t,
          typename std::conditional<BYTES == 2, uint16_t, uint8_t>::type>::type>::type Raw;
  const int lane = threadIdx.x & 31, own = lane & (U - 1);
  float qv[E], o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) { qv[e] = ldf(q + lane * E + e); o[e] = 0.f; }
  auto value = [](const Raw& x, int e) -> float {
    uint32_t w;
    if constexpr (BYTES == 8) w = e < 2 ? x.x : x.y;
    else w = x;
    if constexpr (Q4) return (float)((int)(w >> (4 * e) & 15u) - 8);
    if constexpr (!C::CODES) return __uint_as_float(e & 1 ? w & 0xFFFF0000u : w << 16);
    const uint8_t code = (uint8_t)(w >> (8 * e));
    if constexpr (KIND == KCH_INT8) return (float)(int8_t)code;
    __nv_fp8_e4m3 v;
    v.__x = code;
    return float(v);
  };
  auto ask = [&](int j0) { return ROWS ? 0 : j0 < to ? pg_page(a.bt, b, min(j0 + own, to - 1) >> a.bt.shift) : -1; };
  int page = ask(from);
#pragma unroll 1
  for (int j0 = from; j0 < to; j0 += U) {
    const int next = ask(j0 + U);
    Raw k[U], v[U];
    uint32_t sf[Q4 ? U : 1];                             // 4 bits: the scales of the lane's channels, the key's and the value's
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int pg = __shfl_sync(0xffffffffu, page, u), j = min(j0 + u, to - 1);
      int64_t at_k, at_v;
      if constexpr (ROWS) {
        at_k = ((row0 + j) * a.ld_k + h * D) * 2 + lane * BYTES;
        at_v = ((row0 + j) * a.ld_v + h * D) * 2 + lane * BYTES;
      } else {
        at_k = at_v = ((((int64_t)max(pg, 0) * a.bt.n_kv + h) * a.page + (j & (a.page - 1))) * 32 + lane) * BYTES;
      }
      if constexpr (Q4) {
        sf[u] = 0u;
        if (pg >= 0) {
          const int64_t at = (((int64_t)pg * a.bt.n_kv + h) * a.page + (j & (a.page - 1))) * C::GROUPS + lane * E / 32;
          sf[u] = __ldg((const uint16_t*)a.ks + at) | (uint32_t)__ldg((const uint16_t*)a.vs + at) << 16;
        }
      }
      k[u] = v[u] = Raw{};                               // (a page that is missing: zeros)
      if (pg >= 0) {
        k[u] = __ldg(reinterpret_cast<const Raw*>((const uint8_t*)a.k + at_k));
        v[u] = __ldg(reinterpret_cast<const Raw*>((const uint8_t*)a.v + at_v));
      }
    }
    float ks = 1.f, vs = 1.f;
    if (Q8 && page >= 0) {
      const int64_t row = ((int64_t)page * a.bt.n_kv + h) * a.page + (min(j0 + own, to - 1) & (a.page - 1));
      ks = __ldg((const float*)a.ks + row);
      vs = __ldg((const float*)a.vs + row);
    }
    float s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s[u] = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s[u] = fmaf(qv[e], Q4 ? value(k[u], e) * __uint_as_float(sf[Q4 ? u : 0] << 16) : value(k[u], e), s[u]);
    }
#pragma unroll
    for (int n = U / 2; n > 0; n >>= 1) {
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float keep = lane & n ? s[i + n] : s[i], give = lane & n ? s[i] : s[i + n];
        s[i] = keep + __shfl_xor_sync(0xffffffffu, give, n);
      }
    }
#pragma unroll
    for (int n = U; n < 32; n <<= 1) s[0] += __shfl_xor_sync(0xffffffffu, s[0], n);
    const float p = round_to<bf16>(ex2_fast(fmaf(s[0] * ks, sc, -shift)) * vs);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float pu = __shfl_sync(0xffffffffu, p, u);
      if (j0 + u < to) {
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(pu, Q4 ? value(v[u], e) * __uint_as_float(sf[Q4 ? u : 0] & 0xFFFF0000u) : value(v[u], e), o[e]);
      }
    }
    page = next;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane * E + e;
    if (d < c0 || d >= c1) continue;
    if (dst) dst[d] = o[e]; else stf(out + d, o[e] * f);
  }
}

template <int D, int KIND, int FEW>
__global__ void __launch_bounds__(PtCfg<D, KIND, FEW>::THREADS, 1)
paged_attend_tc5_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CUtensorMap qmap,
                        const __grid_constant__ PgAttend a) {
  typedef PtCfg<D, KIND, FEW> C;
  typedef PgWalk<C::OPEN ? 0 : C::R, PT_KT, C::TWO, C::OPEN ? PG_EXTRA : 0, C::ROWS> Walk;
  extern __shared__ __align__(1024) uint8_t pt_raw[];    // (no room to align it by hand; every block begins its memory there)
  PtSmem<D, KIND, FEW>& sm = *reinterpret_cast<PtSmem<D, KIND, FEW>*>(pt_raw);
  if (smem_addr_u32(pt_raw) & 1023) {
    if (threadIdx.x == 0) atomicCAS(a.bt.status, 0u, (unsigned)KCH_STATUS_PAGED_ATTEND);
    return;
  }
  const int tid = threadIdx.x, warp = t5_warp_index(), lane = tid & 31, G = a.bt.G, n_kv = a.bt.n_kv, slot_rows = a.slot_rows;
  const int R = C::OPEN ? a.bt.rows : C::R, TWO = C::OPEN ? a.bt.rows / 2 : C::TWO;      // rows of an item, and of either warpgroup
  if (tid == 0) {
    for (int i = 0; i < C::STAGES; ++i) { mbarrier_init(&sm.full[i], C::CODES ? 4 : 1); mbarrier_init(&sm.empty[i], 1); }
    for (int i = 0; i < C::RAWS; ++i) { mbarrier_init(&sm.raw_full[i], 1); mbarrier_init(&sm.raw_empty[i], 4); }
    for (int i = 0; i < C::SCALES; ++i) { mbarrier_init(&sm.sc_full[i], 64); mbarrier_init(&sm.sc_empty[i], 8); }
    mbarrier_init(&sm.q_full, C::APART || (C::OPEN && a.q_map) ? 1 : 2);
    mbarrier_init(&sm.q_empty, 1);
    sm.odd[0] = sm.odd[1] = sm.nan_code = 0u;
    for (int i = 0; i < 2; ++i) { mbarrier_init(&sm.s_full[i], 1); mbarrier_init(&sm.p_full[i], 4); mbarrier_init(&sm.pv_done[i], 1); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&kmap) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&vmap) : "memory");
    if (C::OPEN && a.q_map) asm volatile("prefetch.tensormap [%0];" ::"l"(&qmap) : "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr_u32(&sm.tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const PgPlace place = pg_plan<C::OPEN ? 0 : C::R, PT_KT, C::TWO, C::OPEN ? PG_EXTRA : 0, C::ROWS>(a.bt, sm.kv, blockIdx.x, gridDim.x);
  pg_zero_rest(a, 2, blockIdx.x, gridDim.x);
  t5_fence_async_smem();                                 // (the plan was read from the ring's memory, which copies write next)
  t5_fence_before();
  __syncthreads();
  t5_fence_after();
  const uint32_t tmem = sm.tmem;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbarrier_wait_bounded(bar, parity & 1, KCH_STATUS_PAGED_ATTEND, PT_SPIN, a.bt.status); };
  // do the warpgroups have rows of their own, or the same rows and every other tile?
  auto paired = [&](const Walk& w) { return !FEW && w.x.rows > TWO; };
  // The ring holds an item's tiles in the order in which they are used.  Rows of both: K0, then V0 K1, V1 K2, ..; rows of one: K0 K1,
  // then V0 K2 V1 K3, V2 K4 V3 K5, ..

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REG_FEED));
    if (warp == 0 || (C::APART && warp == 2)) {
      // ------------------------------ pages into the ring -----------------------------------------------------------------
      // A tile is 128 / rows-of-a-box copies for each panel of 64 channels (8-bit pages: whole rows), a lane each.  In steps
      // over bf16 pages keys and values are a warp's each: small pages are many copies, and a warp issues them one after the other.
      // Otherwise all are one's, which is soon enough, and the other fetches queries (one warp for both: 256 rows of them took so long
      // that a prompt of 8192 tokens was 6 % slower).
      // A warp that comes to fill a place of the ring has filled one at most three places back, so everything N before that has
      // been used, and a barrier's parity cannot be that of two uses ago.
      const int box = min(a.page, PT_KT), boxes = PT_KT / box, panels = C::CODES ? 1 : C::PANELS;
      const int mybox = lane / panels, mypanel = lane % panels;
      const bool mine = lane < boxes * panels;
      constexpr int N = C::CODES ? C::RAWS : C::STAGES;
      uint64_t *fb = C::CODES ? sm.raw_full : sm.full, *eb = C::CODES ? sm.raw_empty : sm.empty;
      int g = 0;
      bool ok = true;
      for (Walk w(a.bt, place); w.valid() && ok; w.next()) {
        const bool pair = paired(w);
        const int per = pair ? 1 : 2, end = (w.first + w.count) * per;
        const int32_t* pages = a.bt.table + (int64_t)w.b * a.bt.ld_table;
        // a box of which some row may see a key: not before the first window, not behind the sequence's end
        auto needed = [&](int tile, int key) { return mine && tile < w.x.tiles && key + box > w.x.lo && key < w.s.kv; };
        // the page of this lane's box of a tile, asked for a tile ahead; -1 where it is not needed
        auto ask = [&](int tile) -> int {
          const int key = w.x.first_key + tile * PT_KT + mybox * box;
          return !C::ROWS && tile < end && needed(tile, key) ? __ldg(pages + (key >> a.bt.shift)) : -1;
        };
        auto copy = [&](int tile, bool v, int id) {
          const int st = g % N, key = w.x.first_key + tile * PT_KT + mybox * box;
          if (C::APART && v != (warp == 2)) {
            ++g;
            return true;
          }
          bool fine = g < N || wait(eb + st, g / N - 1);
          fine = __all_sync(0xffffffffu, fine);
          if (!fine) return false;
          const bool there = mine && (unsigned)id < (unsigned)a.bt.num_pages;
          uint8_t* scales = C::Q4 ? sm.raw[C::Q4 ? st : 0] + (C::Q4 ? C::RAW : 0) + mybox * box * (2 * C::GROUPS) : nullptr;      // 4 bits: of this lane's box
          uint32_t bytes = C::CODES ? C::RAW : C::TILE;
          if constexpr (C::Q4) {
            bytes += __popc(__ballot_sync(0xffffffffu, there)) * box * (2 * C::GROUPS);
            if (mine && !there) {                        // zeros, by hand
              for (int i = 0; i < box * (2 * C::GROUPS); i += 16) *reinterpret_cast<uint4*>(scales + i) = make_uint4(0u, 0u, 0u, 0u);
              t5_fence_async_smem();                     // (a copy writes there next)
            }
            __syncwarp();
          }
          if (lane == 0) mbarrier_expect_tx(fb + st, bytes);
          __syncwarp();
          if (C::ROWS && mine) {
            // (a tile of which no row sees a key: zeros.  The rows behind a sequence's end are the next one's: masked, their values cleared below.)
            pt_tma_3d(sm.kv[st] + mypanel * (PT_KT * 128), v ? &vmap : &kmap, mypanel * 64, w.h, needed(tile, key) ? w.s.row0 + key : a.bt.N, fb + st);
          } else if (mine) {
            if (!there) {                                // out of range: zeros
              if (needed(tile, key)) pg_bad(a.bt);
              id = (int)a.bt.num_pages;
            }
            if constexpr (C::Q4)
              if (there)
                bulk_copy_g2s(scales, (const bf16*)(v ? a.vs : a.ks) + (((int64_t)id * n_kv + w.h) * a.page + (key & (a.page - 1))) * C::GROUPS,
                              box * (2 * C::GROUPS), fb + st);
            uint8_t* dst = C::CODES ? sm.raw[C::CODES ? st : 0] + mybox * box * (C::RAW / PT_KT)
                                    : sm.kv[C::CODES ? 0 : st] + mypanel * (PT_KT * 128) + mybox * box * 128;
            pt_tma_4d(dst, v ? &vmap : &kmap, mypanel * 64, key & (a.page - 1), w.h, id, fb + st);
          }
          ++g;
          return true;
        };
        int t = w.first * per;
        int id0 = ask(t), id1 = ask(t + 1);              // of tiles t and t + 1
        ok = copy(t, false, id0) && (pair || copy(t + 1, false, id1));
        if (pair) {
          for (; t < end && ok; ++t) {
            const int id2 = ask(t + 2);
            ok = copy(t, true, id0) && (t + 1 >= end || copy(t + 1, false, id1));
            id0 = id1;
            id1 = id2;
          }
        } else {
          for (; t < end && ok; t += 2) {
            const int id2 = ask(t + 2), id3 = ask(t + 3);
            ok = copy(t, true, id0) && (t + 2 >= end || copy(t + 2, false, id2)) && copy(t + 1, true, id1) &&
                 (t + 2 >= end || copy(t + 3, false, id3));
            id0 = id2;
            id1 = id3;
          }
        }
      }
      // no copy is in flight when the block ends (after a wait that ran out nobody else may have waited for the last ones)
      for (int i = 1, n = C::CODES ? C::RAWS : C::STAGES; i <= n && i <= g; ++i)
        wait(C::CODES ? &sm.raw_full[C::CODES ? (g - i) % n : 0] : &sm.full[C::CODES ? 0 : (g - i) % n], (g - i) / n);
    } else if (warp == 1) {
      // ------------------------------ MMA issuer --------------------------------------------------------------------------
      if (t5_elect()) {
        const uint32_t id_s = t5_idesc(PT_KT), id_o = t5_idesc(D) | (1u << 16);
        const uint64_t dq = t5_desc(smem_addr_u32(sm.q[0])), dk = t5_desc(smem_addr_u32(sm.kv[0]));
        const uint64_t dv = t5_desc_mn(smem_addr_u32(sm.kv[0]), PT_KT * 128);
        bool ok = true;
        int g = 0, n = 0, c = 0;                         // tiles of the ring; tiles of each softmax; items
        auto scores = [&](int x, int qx, int stage) {    // S_x = Q_qx K^T
          t5_fence_after();
          const uint64_t qd = dq + (uint64_t)(qx * (128 * D * 2 >> 4)), kd = dk + (uint64_t)(stage * (C::TILE >> 4));
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            t5_mma(tmem + 128u * x, qd + (k >> 2) * (128 * 128 >> 4) + 2 * (k & 3), kd + (k >> 2) * (PT_KT * 128 >> 4) + 2 * (k & 3), id_s, k ? 1u : 0u);
          t5_commit(&sm.s_full[x]);
        };
        auto values = [&](int x, int stage, bool first, bool last) {      // O_x (+)= P_x V; last: it frees the tile
          t5_fence_after();
          const uint64_t vd = dv + (uint64_t)(stage * (C::TILE >> 4));
#pragma unroll
          for (int k = 0; k < PT_KT / 16; ++k)
            pt_mma_ts(tmem + 256u + 128u * x, tmem + 128u * x + 8u * k, vd + k * (2048 >> 4), id_o, first && k == 0 ? 0u : 1u);
          if (last) t5_commit(&sm.empty[stage]);
          t5_commit(&sm.pv_done[x]);                     // (behind it no arrival is under way that nobody waits for)
        };
        auto filled = [&](int i) { return wait(&sm.full[i % C::STAGES], i / C::STAGES); };
        for (Walk w(a.bt, place); w.valid() && ok; w.next(), ++c) {
          const bool pair = paired(w);
          ok = wait(&sm.q_full, c);
          for (int x = 0; x < 2 && ok; ++x) {            // the first scores
            if (!(pair && x)) ok = filled(g);
            if (!ok) break;
            scores(x, pair ? x : 0, g % C::STAGES);
            if (!pair || x) { t5_commit(&sm.empty[g % C::STAGES]); ++g; }
          }
          for (int s = 0; s < w.count && ok; ++s, ++n) {
            const bool more = s + 1 < w.count;
            if (!more) t5_commit(&sm.q_empty);           // the queries have been read
            for (int x = 0; x < 2 && ok; ++x) {
              if (!(pair && x)) ok = filled(g) && (!more || filled(g + 1));
              if (ok) ok = wait(&sm.p_full[x], n);
              if (!ok) break;
              values(x, g % C::STAGES, s == 0, !pair || x);
              if (more) {
                scores(x, pair ? x : 0, (g + 1) % C::STAGES);
                if (!pair || x) t5_commit(&sm.empty[(g + 1) % C::STAGES]);
              }
              if (!pair || x) g += more ? 2 : 1;
            }
          }
        }
      }
    } else {
      // ------------------------------ queries ------------------------------------------------------------------------------
      constexpr int FETCH = C::APART ? 32 : 64;          // threads
      const int t = tid - (128 - FETCH);
      int c = 0, kt = 0;
      bool ok = true;
      if (C::OPEN && a.q_map) {
        // whole tokens: their heads of this key head, 64 channels a copy, for either warpgroup's tile.  (The rows behind a sequence's last
        // token are the next one's, or zeros: no row of the item.)
        if (warp == 2) {
          const int tokens = TWO / G, bytes = TWO * 128 * C::PANELS;
          for (Walk w(a.bt, place); w.valid() && ok; w.next(), ++c) {
            if (c) ok = wait(&sm.q_empty, c - 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const bool both = paired(w);
            if (lane == 0) mbarrier_expect_tx(&sm.q_full, both ? 2 * bytes : bytes);
            __syncwarp();
            if (lane < (both ? 2 : 1) * C::PANELS) {
              const int x = lane / C::PANELS, panel = lane % C::PANELS;
              pt_tma_3d(sm.q[x] + panel * (128 * 128), &qmap, panel * 64, w.h * G, w.s.row0 + (w.block * 2 + x) * tokens, &sm.q_full);
            }
          }
          if (c) wait(&sm.q_full, c - 1);                // (no copy is in flight when the block ends)
        }
      }
      if (!(C::OPEN && a.q_map)) for (Walk w(a.bt, place); w.valid() && ok; w.next(), ++c) {
        if (c) ok = wait(&sm.q_empty, c - 1);
        if (!ok) break;
        constexpr int CHUNKS = D / 8, STEP = FETCH / CHUNKS;       // 16 bytes a thread
        static_assert(128 % (4 * STEP) == 0 && 4 * STEP % 8 == 0, "rows of a round");
        const int rows = w.x.rows, k = t % CHUNKS;
        const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;    // (the softmax takes the scale's size: a maximum stays one)
        // Every STEP'th row is a thread's.  Head, source and place in the swizzle are counted on from row to row: computed
        // anew for each they made 256 rows 13000 cycles, more than what is left of an item once its last scores are there.
        const int r0 = t / CHUNKS, skip = pg_token(a.bt, STEP), turn = STEP - skip * G;
        const int row0 = w.block * R + r0, tok0 = pg_token(a.bt, row0);
        int g = row0 - tok0 * G;
        const bf16* src = (const bf16*)a.q + (w.s.row0 + tok0) * a.ld_q + (w.h * G + g) * D + k * 8;
        const int64_t ahead = skip * a.ld_q + turn * D, over = a.ld_q - (int64_t)G * D;
        uint32_t to = smem_addr_u32(sm.q[0]) + (k >> 3) * (128 * 128) + r0 * 128;
        const uint32_t at = ((k & 7) ^ (r0 & 7)) << 4;
#pragma unroll 1
        for (int r = r0; r < rows; r += 4 * STEP, to += 4 * STEP * 128) {
          if (!FEW && !C::OPEN && r == 128 + r0) to += 128 * D * 2 - 128 * 128;      // the second tile
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (r + j * STEP >= rows) break;
            uint32_t dst = to + j * (STEP * 128) + (at ^ ((j * STEP & 7) << 4));
            if constexpr (C::OPEN) {                     // (tiles of TWO rows, which may be no multiple of STEP)
              const int x = r + j * STEP >= TWO ? 1 : 0, i = r + j * STEP - x * TWO;
              dst = smem_addr_u32(sm.q[x]) + (k >> 3) * (128 * 128) + i * 128 + (((k & 7) ^ (i & 7)) << 4);
            }
            if (flip) {
              uint4 u = __ldg(reinterpret_cast<const uint4*>(src));
              u.x ^= flip; u.y ^= flip; u.z ^= flip; u.w ^= flip;
#pragma unroll
              for (int i = 0; i < C::COPIES; ++i)
                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + i * (C::R * 128)), "r"(u.x), "r"(u.y), "r"(u.z), "r"(u.w) : "memory");
            } else {
#pragma unroll
              for (int i = 0; i < C::COPIES; ++i)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + i * (C::R * 128)), "l"(src) : "memory");
            }
            g += turn;
            src += ahead;
            if (g >= G) { g -= G; src += over; }
          }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        t5_fence_async_smem();
        __syncwarp();
        if (lane == 0) mbarrier_arrive(&sm.q_full);
        if constexpr (C::Q8) {
          // the scales of the item's key tiles: two keys a thread, 0 before the window and behind the end (a scale there may be anything); the page is
          // asked for a tile ahead, and the copies report to the barrier by themselves
          const int per = paired(w) ? 1 : 2, end = (w.first + w.count) * per;
          const int32_t* pages = a.bt.table + (int64_t)w.b * a.bt.ld_table;
          auto ask = [&](int tile, int i) -> int {
            const int key = w.x.first_key + tile * PT_KT + t + 64 * i;
            return tile < min(end, w.x.tiles) && key >= w.x.lo && key < w.s.kv ? __ldg(pages + (key >> a.bt.shift)) : -1;
          };
          int id0 = ask(w.first * per, 0), id1 = ask(w.first * per, 1);
          for (int tile = w.first * per; tile < end && ok; ++tile, ++kt) {
            const int n0 = ask(tile + 1, 0), n1 = ask(tile + 1, 1), slot = kt % C::SCALES;
            if (kt >= C::SCALES) ok = wait(&sm.sc_empty[slot], kt / C::SCALES - 1);
            if (!ok) break;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int id = i ? id1 : id0, key = w.x.first_key + tile * PT_KT + t + 64 * i;
              const bool there = (unsigned)id < (unsigned)a.bt.num_pages;
              const int64_t at = there ? ((int64_t)id * n_kv + w.h) * a.page + (key & (a.page - 1)) : 0;
              const int bytes = there ? 4 : 0;           // (none: 4 bytes of zeros)
              asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;"
                           ::"r"(smem_addr_u32(&sm.scale[slot][0][t + 64 * i])), "l"((const float*)a.ks + at), "r"(bytes) : "memory");
              asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;"
                           ::"r"(smem_addr_u32(&sm.scale[slot][1][t + 64 * i])), "l"((const float*)a.vs + at), "r"(bytes) : "memory");
            }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr_u32(&sm.sc_full[slot])) : "memory");
            id0 = n0;
            id1 = n1;
          }
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
  } else if (warp < 12) {
    // ------------------------------ softmax and the items' ends: a row per thread -----------------------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REG_SOFT));
    const int x = (warp >> 2) - 1, r = (warp & 3) * 32 + lane;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + 128u * x + lane_base, tO = tmem + 256u + lane_base;
    const float sc = fmaxf(fabsf(a.scale), 1e-30f);      // (not 0: a masked logit is -inf)
    const float raise = 8.f / sc;
    bool ok = true;
    int n = 0, kt = 0, ring = 0;                         // tiles of this warpgroup; key tiles of the CTA; tiles of the ring before the item
    bool part = false;                                   // the CTA's last item goes on in the next one
    for (Walk w(a.bt, place); w.valid(); w.next()) {
      const bool pair = paired(w);
      constexpr int APART = 128 / C::COPIES;
      const int ri = pair ? x * TWO + r : r % APART, sub = FEW ? r >> 5 : 0;      // row of the item, part of a tile's keys
      const bool live = ri < w.x.rows && (!C::OPEN || r < TWO);
      const int2 keys = pg_sees(a.bt, w.s, w.block * R + ri);           // those of the row
      float m = -INFINITY, l = 0.f;
      for (int s = 0; s < w.count; ++s, ++n) {
        const int tile = pair ? w.first + s : 2 * (w.first + s) + x;
        const int key0 = w.x.first_key + tile * PT_KT, lo = keys.x - key0, hi = keys.y - key0;
        const int from = 32 * sub, to = FEW ? from + 32 : PT_KT;
        const bool whole = __all_sync(0xffffffffu, !live || (lo <= from && hi >= to));
        const bool none = __all_sync(0xffffffffu, !live || min(hi, to) <= max(lo, from));
        const int slot = (pair ? kt : kt + x) % C::SCALES, turn = (pair ? kt : kt + x) / C::SCALES;
        kt += pair ? 1 : 2;
        if (ok) ok = wait(&sm.s_full[x], n);
        if (C::Q8 && ok) ok = wait(&sm.sc_full[slot], turn);
        ok = __all_sync(0xffffffffu, ok);
        t5_fence_after();
        if (none || !ok) {
          const uint32_t zero[32] = {};
          pt_st(tS, zero);
          pt_st(tS + 32u, zero);
        } else {
          // Chunks: the row's scores come from tensor memory twice, in halves: for the maximum, and for P.  Kept in registers they
          // would be 128 of them, and both passes unrolled: the code of all roles then outgrows the instruction cache, and a tile
          // took 3000 cycles (8-bit pages: 7000) where its arithmetic is ~1200.
          const ulonglong2* ks = reinterpret_cast<const ulonglong2*>(sm.scale[C::Q8 ? slot : 0][0]);      // pairs of scales
          const ulonglong2* vs = reinterpret_cast<const ulonglong2*>(sm.scale[C::Q8 ? slot : 0][1]);
          auto fetch = [&](auto& sv, int col) {          // 32 or 64 scores from column `col` on, scaled and masked
            constexpr int N = sizeof(sv) / 4;
#pragma unroll
            for (int k = 0; k < N; k += 32) t5_ld32(tS + col + k, *reinterpret_cast<uint32_t(*)[32]>(sv + k));
            t5_wait_ld();
            if (C::Q8) {
#pragma unroll
              for (int e = 0; e < N / 4; ++e) {
                const ulonglong2 f = ks[col / 4 + e];
                pt_scale2(sv[4 * e], sv[4 * e + 1], f.x);
                pt_scale2(sv[4 * e + 2], sv[4 * e + 3], f.y);
              }
            }
            if (!whole) {
#pragma unroll
              for (int k = 0; k < N; k += 32) {
                // (a chunk's edge lies in one 32 of a tile, or two)
                if (C::OPEN && __all_sync(0xffffffffu, !live || (lo <= col + k && hi >= col + k + 32))) continue;
                const uint32_t mk = pt_range(lo - col - k, hi - col - k);
#pragma unroll
                for (int e = 0; e < 32; ++e) sv[k + e] = mk & (1u << e) ? sv[k + e] : 0xFF800000u;
              }
            }
          };
          float t0 = -INFINITY, t1 = -INFINITY;
          auto highest = [&](const auto& sv) {
#pragma unroll
            for (int e = 0; e < sizeof(sv) / 4; e += 4) {
              t0 = fmaxf(t0, fmaxf(__uint_as_float(sv[e]), __uint_as_float(sv[e + 1])));
              t1 = fmaxf(t1, fmaxf(__uint_as_float(sv[e + 2]), __uint_as_float(sv[e + 3])));
            }
          };
          int begin = 0, end = PT_KT;                    // without the half of a tile of which no row of the warp sees a key
          if (C::OPEN && !whole) {
            if (__all_sync(0xffffffffu, !live || hi <= 64)) end = 64;
            else if (__all_sync(0xffffffffu, !live || lo >= 64)) begin = 64;
          }
          uint32_t few[32];                              // (FEW: 32 keys a warp, which stay)
          if constexpr (FEW != 0) {
            fetch(few, from);
            highest(few);
          } else {
#pragma unroll 1
            for (int col = begin; col < end; col += 64) {
              uint32_t sv[64];
              fetch(sv, col);
              highest(sv);
            }
          }
          const float top = fmaxf(t0, t1);
          if (s == 0) m = top;
          else if (__any_sync(0xffffffffu, live && top > m + raise)) {
            // (each row by itself: neither the other rows nor what lies in unused ones changes a result's bits)
            const float now = top > m + raise ? top : m, keep = now == m ? 1.f : ex2_fast((m - now) * sc);
            m = now;
            l *= keep;
            if (ok) ok = wait(&sm.pv_done[x], n - 1);
            ok = __all_sync(0xffffffffu, ok);
            t5_fence_after();
#pragma unroll 1
            for (int k = 0; k < D / 32; ++k) {
              uint32_t ov[32];
              t5_ld32(tO + 128u * x + 32u * k, ov);
              t5_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * keep);
              t5_st32(tO + 128u * x + 32u * k, ov);
            }
          }
          const float shift = m == -INFINITY ? 0.f : m * sc;
          const uint64_t sc2 = pt_pack(sc, sc), sh2 = pt_pack(-shift, -shift);
          uint64_t sum2 = 0;
          auto weigh = [&](const auto& sv, int col) {    // P of those columns, over scores that have been read
            constexpr int N = sizeof(sv) / 4;
            uint32_t pk[N / 2];
#pragma unroll
            for (int e = 0; e < N / 2; ++e) {
              float x0, x1;
              pt_unpack(pt_fma2(pt_pack(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])), sc2, sh2), x0, x1);
              float p0, p1;                              // (of -inf 0, of a NaN a NaN)
              if ((e & 3) >= 4 - C::POLY) {
                pt_ex2_fma(x0, x1);
                p0 = x0;
                p1 = x1;
              } else {
                p0 = ex2_fast(x0);
                p1 = ex2_fast(x1);
              }
              sum2 = pt_add2(sum2, pt_pack(p0, p1));
              if (C::Q8) {
                const ulonglong2 f = vs[col / 4 + (e >> 1)];
                pt_unpack(pt_mul2(pt_pack(p0, p1), e & 1 ? f.y : f.x), p0, p1);
              }
              pk[e] = pack2_bf16(p0, p1);
              if (FEW == 16 && (r & 16)) pk[e] = pack2_bf16(p0 - __uint_as_float(pk[e] << 16), p1 - __uint_as_float(pk[e] & 0xFFFF0000u));
            }
            pt_st(tS + col / 2, pk);
          };
          if constexpr (FEW != 0) {
            const uint32_t zero[16] = {};
#pragma unroll
            for (int k = 1; k < 4; ++k) pt_st(tS + 16u * ((sub + k) & 3), zero);
            weigh(few, from);
          } else {
#pragma unroll 1
            for (int col = begin; col < end; col += 64) {
              uint32_t sv[64];
              fetch(sv, col);
              weigh(sv, col);
            }
            if (C::OPEN && end - begin < PT_KT) {
              const uint32_t zero[32] = {};
              pt_st(tS + (begin ? 0u : 32u), zero);
            }
          }
          float la, lb;
          pt_unpack(sum2, la, lb);
          l += la + lb;
        }
        if (!C::CODES && w.s.kv > key0 && w.s.kv < key0 + PT_KT) {
          // (codes are numbers by now, or the scales there are 0)
          const int at = pair ? ring + 1 + 2 * s : ring + 2 + 4 * s + (s + 1 < w.count ? 2 : 1) * x;      // of the tile's values in the ring
          if (ok) ok = wait(&sm.full[at % C::STAGES], at / C::STAGES);
          ok = __all_sync(0xffffffffu, ok);
          if (ok && key0 + r >= w.s.kv) {
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
              *reinterpret_cast<uint4*>(sm.kv[at % C::STAGES] + (i >> 3) * (PT_KT * 128) + r * 128 + ((i & 7) << 4)) = make_uint4(0u, 0u, 0u, 0u);
          }
          t5_fence_async_smem();
        }
        t5_wait_st();
        t5_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (C::Q8) pt_arrive_n(&sm.sc_empty[slot], pair ? 1 : 2);
          mbarrier_arrive(&sm.p_full[x]);
        }
      }
      // ---- the item's end: its rows, or its part of them ------------------------------------------------------------------------
      if (ok) ok = wait(&sm.pv_done[x], n - 1);
      ok = __all_sync(0xffffffffu, ok);
      t5_fence_after();
      const bool direct = w.starts() && w.ends();
      float* slot = a.slots + (2 * (int64_t)blockIdx.x + (w.starts() ? 1 : 0)) * pg_slot_floats(slot_rows, D);
      auto out_row = [&](int i) {                        // of the item's row i
        const int rr = w.block * R + i, tk = pg_token(a.bt, rr);
        return (bf16*)a.out + ((int64_t)(w.s.row0 + tk) * (n_kv * G) + w.h * G + rr - tk * G) * D;
      };
      auto factor = [&](int i, float l, float shift) {   // 1 / the row's denominator
        if (!direct) return 1.f;
        float below = l;
        if (a.sink && l > 0.f) {
          const int rr = w.block * R + i;
          below += ex2_fast(ld_any(a.sink, w.h * G + rr - pg_token(a.bt, rr) * G, a.sink_dtype) * PG_LOG2E - shift);
        }
        return l == 0.f ? 0.f : 1.f / below;
      };
      auto redo = [&](int i, float shift, float f, int c0, int c1) {     // a row that is not finite, key by key, on the warp
        const int span = PT_KT * (pair ? 1 : 2), part0 = w.x.first_key + w.first * span, part1 = part0 + w.count * span;
        const int rr = w.block * R + i, tk = pg_token(a.bt, rr);
        const int2 k = pg_sees(a.bt, w.s, rr);
        pt_slow_row<D, KIND>(a, w.b, w.s.row0, w.h, (const bf16*)a.q + (w.s.row0 + tk) * a.ld_q + (w.h * G + rr - tk * G) * D, max(k.x, part0),
                             min(k.y, part1), a.scale < 0.f ? -sc : sc, shift, f, out_row(i), direct ? nullptr : slot + (int64_t)i * D, c0, c1);
      };
      // The parts of a row: its O_0 and O_1 with weights w0, w1 where the warpgroups had other tiles of the same rows (each then
      // stores half of the columns), and with FEW those of four warps.
      const auto sync = [](int bar, int n) { asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(n) : "memory"); };
      float w0 = 1.f, w1 = 0.f, mm = m, ll = l;
      bool none0 = false, none1 = true;                  // a part without a key: what its sums hold does not matter
      if (!pair) {
        sm.ml[0][x * 128 + r] = m;
        sm.ml[1][x * 128 + r] = l;
        sync(1, 256);
        const float m0 = sm.ml[0][r], m1 = sm.ml[0][128 + r];
#pragma unroll
        for (int k = 0; k < 256; k += APART) mm = fmaxf(mm, sm.ml[0][ri + k]);
        const float ref = mm == -INFINITY ? 0.f : mm;
        w0 = ex2_fast((m0 - ref) * sc);
        w1 = ex2_fast((m1 - ref) * sc);
        none0 = m0 == -INFINITY;
        none1 = m1 == -INFINITY;
        if (!FEW || r < APART) {
          ll = 0.f;                                      // (a NaN of a part's sum stays one)
#pragma unroll
          for (int k = 0; k < 256; k += FEW ? 32 : APART) ll += sm.ml[1][ri + k] * ex2_fast((sm.ml[0][ri + k] - ref) * sc);
        }
      }
      const float shift = mm == -INFINITY ? 0.f : mm * sc;
      float f = 1.f;
      if (live && direct && (!FEW || r < APART)) f = factor(ri, ll, shift);
      if (live && !direct && (pair || (x == 0 && r < APART))) {
        slot[(int64_t)slot_rows * D + ri] = mm * sc;
        slot[(int64_t)slot_rows * D + slot_rows + ri] = ll;
      }
      if (FEW && r < APART) sm.factor[x][r] = f;
      const int c0 = pair ? 0 : x * (D / 2), c1 = pair ? D : c0 + D / 2;
      constexpr int CW = FEW ? D / 4 : 32, WORDS = CW / 4;       // columns, and 16-byte words, of a row at a time
      float odd = 0.f;                                   // 0 unless a value of the row is not finite
      bf16* orow = FEW ? nullptr : out_row(ri);
      const bool wide = ((uintptr_t)a.out & 31) == 0;
#pragma unroll 1
      for (int col = c0; col < c1; col += CW) {
        uint32_t o0[CW];
        pt_ld(tO + (pair ? 128u * x : 0u) + col, o0);
        if (pair) {
          t5_wait_ld();
        } else {
          uint32_t o1[CW];
          pt_ld(tO + 128u + col, o1);
          t5_wait_ld();
#pragma unroll
          for (int e = 0; e < CW; ++e) {
            const float a0 = __uint_as_float(o0[e]), a1 = __uint_as_float(o1[e]);
            o0[e] = __float_as_uint((none0 ? 0.f : a0 * w0) + (none1 ? 0.f : a1 * w1));
          }
        }
        float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < CW; ++e) z[e & 3] = fmaf(__uint_as_float(o0[e]), 0.f, z[e & 3]);
        odd += (z[0] + z[1]) + (z[2] + z[3]);
        if constexpr (FEW != 0) {                             // through the second query tile, 128 rows of either warpgroup
          float4* stage = reinterpret_cast<float4*>(sm.q[1]) + x * 128 * WORDS;
          if (live) {
#pragma unroll
            for (int v = 0; v < WORDS; ++v)
              stage[r * WORDS + (v ^ (r & (WORDS - 1)))] = make_float4(__uint_as_float(o0[4 * v]), __uint_as_float(o0[4 * v + 1]),
                                                                       __uint_as_float(o0[4 * v + 2]), __uint_as_float(o0[4 * v + 3]));
            if (col + CW == c1 && ok && odd != 0.f) atomicOr(&sm.odd[x], 1u << ri);
          }
          sync(2 + x, 128);
#pragma unroll 1
          for (int k = r; k < w.x.rows * WORDS && ok; k += 128) {
            const int i = k / WORDS, v = k % WORDS;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int n2 = 0; n2 < 128; n2 += APART) {    // (APART is a multiple of WORDS: one place in the swizzle)
              const float4 p = stage[(n2 + i) * WORDS + (v ^ (i & (WORDS - 1)))];
              o.x += p.x; o.y += p.y; o.z += p.z; o.w += p.w;
            }
            if (direct) {
              const float fi = sm.factor[x][i];
              *reinterpret_cast<uint2*>(out_row(i) + col + 4 * v) = make_uint2(pack2_bf16(o.x * fi, o.y * fi), pack2_bf16(o.z * fi, o.w * fi));
            } else {
              *reinterpret_cast<float4*>(slot + (int64_t)i * D + col + 4 * v) = o;
            }
          }
          sync(2 + x, 128);
        } else if (live && ok) {
          if (direct) {
#pragma unroll
            for (int e = 0; e < CW / 2; ++e) o0[e] = pack2_bf16(__uint_as_float(o0[2 * e]) * f, __uint_as_float(o0[2 * e + 1]) * f);
#pragma unroll
            for (int v = 0; v < CW / 2; v += 8) pt_store8(orow + col + 2 * v, o0 + v, wide);
          } else {
#pragma unroll
            for (int v = 0; v < CW; v += 8) pt_store8(slot + (int64_t)ri * D + col + v, o0 + v, true);
          }
        }
      }
      // e4m3: codes of NaN have counted as 480 so far, which reaches no sum but those that they make NaN.  Where there is one, the rows are
      // summed again as well.
      bool nan = false;
      if (KIND == KCH_FP8_E4M3 && *(volatile uint32_t*)&sm.nan_code != 0u) {
        const int span = PT_KT * (pair ? 1 : 2), part0 = w.x.first_key + w.first * span;
        nan = pt_nan_among<D>(a, w.b, w.h, max(part0, w.x.lo), min(part0 + w.count * span, w.s.kv));
      }
      // rows that are not finite: again, over the columns stored here
      unsigned again;
      if constexpr (FEW != 0) again = (warp & 3) == 0 ? sm.odd[x] : 0u;       // (row i is lane i's of the first warp)
      else again = __ballot_sync(0xffffffffu, live && ok && (odd != 0.f || nan));
      if (again) {
        __syncwarp();
        if (FEW && lane == 0) sm.odd[x] = 0u;
        for (; again; again &= again - 1) {
          const int src = __ffs(again) - 1;
          redo(__shfl_sync(0xffffffffu, ri, src), __shfl_sync(0xffffffffu, shift, src), __shfl_sync(0xffffffffu, f, src), c0, c1);
        }
      }
      t5_fence_before();
      if (!pair) sync(1, 256);                           // both have read O of both, and the maxima and sums
      ring += (pair ? 2 : 4) * w.count;
      if (w.starts() && !w.ends()) {
        part = true;
        if (tid == 128) a.records[blockIdx.x] = {1, w.b, w.h, w.block, w.last(place, blockIdx.x), w.x.rows, w.s.row0};
      }
    }
    if (tid == 128 && !part) a.records[blockIdx.x].valid = 0;
  } else {
    // ------------------------------ codes to bf16 tiles ------------------------------------------------------------------------
    if constexpr (C::CODES) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REG_CONV));
      const int t = tid - 384;
      bool ok = true;
      int g = 0;
      for (Walk w(a.bt, place); w.valid() && ok; w.next()) {
        const bool pair = paired(w);
        const int tiles = 2 * w.count * (pair ? 1 : 2);            // of keys and values
        for (int i = 0; i < tiles && ok; ++i, ++g) {
          ok = wait(&sm.raw_full[g % C::RAWS], g / C::RAWS);
          if (ok && g >= C::STAGES) ok = wait(&sm.empty[g % C::STAGES], g / C::STAGES - 1);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if constexpr (C::Q4) {
            // 32 codes and their scale a thread, a quarter (half) of a row: a warp reads 512 bytes in a row.  The words of 8 channels go to
            // their places two and two about in the second panel, so that 8 threads meet in no bank.  Keys that no row sees, and
            // what lies behind the sequence's end, are zeros (a scale there may be NaN).
            const int piece = t % C::GROUPS, panel = piece >> 1, turn = D == 128 ? 2 * panel : 0;
            const int turns = (i - 2) / 4, rest = (i - 2) % 4;
            const int tile = pair ? w.first + i / 2
                                  : 2 * w.first + (i < 2 ? i : turns == w.count - 1 ? 2 * turns + rest : 2 * turns + (rest & 1) * 2 + (rest >> 1));
            const int key0 = w.x.first_key + tile * PT_KT;
#pragma unroll 1
            for (int row = t / C::GROUPS; row < PT_KT; row += 128 / C::GROUPS) {
              const uint4 u = *reinterpret_cast<const uint4*>(sm.raw[g % C::RAWS] + row * (D / 2) + piece * 16);
              uint32_t s = *reinterpret_cast<const uint16_t*>(sm.raw[g % C::RAWS] + C::RAW + (row * C::GROUPS + piece) * 2);
              const int key = key0 + row;
              s = key >= w.x.lo && key < w.s.kv ? s | s << 16 : 0u;
              const uint32_t s24 = pt_bf16_fma(s, 0xC1C0C1C0u, 0u);      // -24 s
              uint8_t* line = sm.kv[g % C::STAGES] + panel * (PT_KT * 128) + row * 128;
              const uint32_t w4[4] = {turn ? u.z : u.x, turn ? u.w : u.y, turn ? u.x : u.z, turn ? u.y : u.w};
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                uint4 x;
                pt_nibbles8(w4[j], s, s24, x);
                *reinterpret_cast<uint4*>(line + (((((piece & 1) << 2) + (j ^ turn)) ^ (row & 7)) << 4)) = x;
              }
            }
          } else {
            // 16 codes each: 2 words of a tile's row, 4 such pieces a row and panel.  8 threads that meet in the banks have 4 pieces of
            // two rows: one of an even and one of an odd number (whose words lie apart in the tile), and where the codes are
            // swizzled too, numbers that differ in bit 2 as well (5 = 101b: their pieces lie apart there).  A thread's place in
            // both swizzles is the same in every round.
            constexpr int ROWS = D == 128 ? 16 : 32, ROUNDS = PT_KT / ROWS;      // rows between two rounds
            const int k = lane & 3, wq = t >> 5;
            const int row = D == 128 ? (wq >> 1) * 8 + ((lane >> 3) ^ ((lane >> 2) & 1) * 5) : wq * 8 + (lane >> 2), panel = D == 128 ? wq & 1 : 0;
            const uint8_t* src = sm.raw[g % C::RAWS] + row * D + ((D == 128 ? (panel * 4 + k) ^ (row & 7) : k ^ ((row >> 1) & 3)) << 4);
            uint8_t* line = sm.kv[g % C::STAGES] + panel * (PT_KT * 128) + row * 128;
            uint32_t most = 0u;
            uint8_t *to0 = line + (((2 * k) ^ (row & 7)) << 4), *to1 = line + (((2 * k + 1) ^ (row & 7)) << 4);
#pragma unroll 4
            for (int n = 0; n < ROUNDS; ++n) {
              const uint4 u = *reinterpret_cast<const uint4*>(src + n * (ROWS * D));
              uint4 lo, hi;
              pt_codes4<KIND>(u.x, lo.x, lo.y, most);
              pt_codes4<KIND>(u.y, lo.z, lo.w, most);
              pt_codes4<KIND>(u.z, hi.x, hi.y, most);
              pt_codes4<KIND>(u.w, hi.z, hi.w, most);
              *reinterpret_cast<uint4*>(to0 + n * (ROWS * 128)) = lo;
              *reinterpret_cast<uint4*>(to1 + n * (ROWS * 128)) = hi;
            }
            // a code of NaN (an append writes none): at the ends of items from here on it is looked for among what the sequences have
            if (KIND == KCH_FP8_E4M3 && (most >= 0x07F00000u || (most & 0xFFFFu) >= 0x07F0u))
              *(volatile uint32_t*)&sm.nan_code = 1u;
          }
          t5_fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbarrier_arrive(&sm.full[g % C::STAGES]);
            mbarrier_arrive(&sm.raw_empty[g % C::RAWS]);
          }
        }
      }
    }
  }
  __syncthreads();
  if (warp == 0) {
    t5_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// ---- host -------------------------------------------------------------------------------------------------------------------
int kch_make_tensor_map_pages(CUtensorMap* map, const void* base, int elem_bytes, uint64_t pages, uint32_t n_kv, uint32_t page_size, uint32_t c,
                              uint32_t box_rows, bool plain = false);
int kch_make_tensor_map_rows(CUtensorMap* map, const void* base, uint64_t rows, uint32_t heads, uint64_t ld, uint32_t c, uint32_t box_heads, uint32_t box_rows);

bool kch_paged_attend_tc5_supported(int dtype, int c) { return dtype == KCH_BF16 && (c == 64 || c == 128); }

template <int D, int KIND, int FEW>
static int pt_launch(const CUtensorMap& km, const CUtensorMap& vm, const CUtensorMap& qm, const PgAttend& a, int ctas, cudaStream_t s) {
  const int smem = (int)sizeof(PtSmem<D, KIND, FEW>);
  static std::atomic<uint64_t> done{0};                  // devices on which the kernel has its shared memory
  int dev = 0;
  KCH_CUDA_OK(cudaGetDevice(&dev));
  if (dev > 63 || !((done.load(std::memory_order_relaxed) >> dev) & 1)) {
    KCH_CUDA_OK(cudaFuncSetAttribute(paged_attend_tc5_kernel<D, KIND, FEW>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (dev <= 63) done.fetch_or(1ULL << dev, std::memory_order_relaxed);
  }
  paged_attend_tc5_kernel<D, KIND, FEW><<<ctas, PtCfg<D, KIND, FEW>::THREADS, smem, s>>>(km, vm, qm, a);
  KCH_LAUNCH_OK();
  return KCH_OK;
}

int kch_paged_attend_tc5(PgAttend& a, int kind, int rows, int ctas, cudaStream_t s) {
  CUtensorMap km, vm, qm = {};
  // (a negative scale's sign goes to the queries on their way: no plain copies)
  a.q_map = (kind == PG_ROWS || kind == KCH_INT4) && a.bt.G <= 128 && a.scale >= 0.f;
  if (a.q_map) {
    const int rc = kch_make_tensor_map_rows(&qm, a.q, a.bt.N, (uint32_t)a.bt.n_kv * a.bt.G, a.ld_q, a.c, a.bt.G, a.bt.rows / 2 / a.bt.G);
    if (rc != KCH_OK) return rc;
  }
  if (kind == PG_ROWS) {
    int rc = kch_make_tensor_map_rows(&km, a.k, a.bt.N, a.bt.n_kv, a.ld_k, a.c, 1, PT_KT);
    if (rc == KCH_OK) rc = kch_make_tensor_map_rows(&vm, a.v, a.bt.N, a.bt.n_kv, a.ld_v, a.c, 1, PT_KT);
    if (rc != KCH_OK) return rc;
    return a.c == 64 ? pt_launch<64, PG_ROWS, 0>(km, vm, qm, a, ctas, s) : pt_launch<128, PG_ROWS, 0>(km, vm, qm, a, ctas, s);
  }
  const bool q4 = kind == KCH_INT4;
  const int es = kind == KCH_BF16 ? 2 : 1, box = a.page < PT_KT ? a.page : PT_KT, wide = q4 ? a.c / 2 : a.c;
  int rc = kch_make_tensor_map_pages(&km, a.k, es, (uint64_t)a.bt.num_pages, a.bt.n_kv, a.page, wide, box, q4);
  if (rc == KCH_OK) rc = kch_make_tensor_map_pages(&vm, a.v, es, (uint64_t)a.bt.num_pages, a.bt.n_kv, a.page, wide, box, q4);
  if (rc != KCH_OK) return rc;
#define PT_GO(D_, K_, F_) pt_launch<D_, K_, F_>(km, vm, qm, a, ctas, s)
#define PT_KIND(D_)                                                                            \
  (kind == KCH_FP8_E4M3 ? PT_GO(D_, KCH_FP8_E4M3, 0) : kind == KCH_INT8 ? PT_GO(D_, KCH_INT8, 0) : q4 ? PT_GO(D_, KCH_INT4, 0) \
   : rows == 16 ? PT_GO(D_, KCH_BF16, 16) : rows == 32 ? PT_GO(D_, KCH_BF16, 32) : PT_GO(D_, KCH_BF16, 0))
  return a.c == 64 ? PT_KIND(64) : PT_KIND(128);
#undef PT_KIND
#undef PT_GO
}
