// Attention of few new tokens a sequence over 8-bit pages (e4m3, int8; bf16 activations, heads of 64 or 128).
// Mathematics and division of the work: paged_attend.cu, paged.cuh.
//
// A step of a few tokens is bound by the pages' bytes, and on its heels follows the arithmetic that turns codes into bf16: 2 ALU
// operations a code (at 64 lanes a clock, 2048 clocks for the 256 keys and values that an SM gets from memory in 2850).  So codes are
// converted once, in the registers of the warp that multiplies them (mma.sync; the rows are far too few for the tensor core's rate to
// matter): through tiles of tcgen05 the same step took twice as long, for the tiles are written, fenced and read back.
//
// An item is up to 32 (token, head of the group) rows of a sequence; a tile is 128 keys, its payloads and scales copied into a ring by
// one warp (TMA, 128-byte or 64-byte swizzle; scales by bulk copies).  Four warps share a tile, 32 keys each, and the other four take
// the next one (32 rows: eight share it); a warp has a maximum, a sum and an O of its own, so that nothing but the ring is waited for,
// and they are joined when the item ends.  (With 16 keys a warp and tile there were too few instructions that do not wait for one another: 2900 clocks a tile.)
//   S = Q K^T: the order of the contraction is free, so thread (g, t) of a fragment takes 32 (16) consecutive channels of key g, four of
//     them a product: a row is read in 16-byte words, and the queries' fragments are loaded in the same order.
//   O += P V:  the order of the columns is free, so thread (g, t) takes 16 (8) consecutive channels of keys 2t, 2t + 1, 2t + 8, 2t + 9,
//     one of them a product; pairs of keys meet by a byte permutation.  P comes from S in place.
// A key's scale multiplies its logit, and its probability before that is rounded to bf16; masked keys are taken out after that, so
// that a scale that is not finite stays where it is seen.  e4m3's codes of NaN (an append writes none, but a pool that existed before may
// hold some) convert to 480; the largest code of a tile is kept, an instruction more for four codes, and where it is one of them the
// item's keys are looked through when it ends and what sees one is made NaN (5 % of a step; a test of each word for such bytes took 7 to 10).
//
// Measured, 64 sequences, 16 heads of 128 on 4, pages of 64: 8192 tokens, e4m3, 143 us (3.9 TB/s of pages); 500 to 16000 tokens, e4m3 158,
// int8 163, and on one key head 58 and 59.  Bound by what two warps of a scheduler have in flight (half of the issue slots are used).
// Through tcgen05 tiles 8192 tokens took 179 us and one key head 65; with sixteen warps of 104 registers (they spill) 166.
#include <cuda.h>
#include <math.h>

#include <atomic>

#include "paged.cuh"
#include "tc5_utils.cuh"

#define PM_KT 128
#define PM_SPIN (1u << 26)

// R rows an item: 8, 16 or 32, by what a sequence has.  8 (one token of up to 8 heads): the lower half of the scores' fragments is
// empty, and that of P has what its rounding left (paged_attend_tc5.cu has the reason; 16 rows: in products of their own, 7 %; 32:
// none).  32: two fragments a warp, which then takes 16 keys of every tile, for the registers' sake.
template <int R>
struct PmCfg {
  static constexpr int WARPS = 8, THREADS = 128 + 32 * WARPS;                   // that compute; the first warpgroup copies
  static constexpr int SHARE = R == 32 ? 8 : 4, SLICE = PM_KT / SHARE, H = SLICE / 8;      // warps of a tile; a warp's keys; in eights
  static constexpr int MT = R == 32 ? 2 : 1, F = R == 8 ? 2 : 4, HF = R / 8;    // fragments; scores of one a thread has; rows of a thread
  static constexpr int REG_FEED = R == 32 ? 56 : 64, REG_WORK = R == 32 ? 224 : 216, REG_LAUNCH = 65536 / THREADS / 8 * 8;
  static_assert(128 * REG_FEED + 32 * WARPS * REG_WORK <= THREADS * REG_LAUNCH, "register split");
};
template <int D, int R>
struct PmSmem {
  typedef PmCfg<R> C;
  static constexpr int STAGES = D == 128 ? 4 : 8;        // (even: a stage is always the same warps')
  alignas(1024) uint8_t k[STAGES][PM_KT * D], v[STAGES][PM_KT * D];
  alignas(16) float ks[STAGES][PM_KT], vs[STAGES][PM_KT];
  alignas(16) float stage[C::WARPS][8 * D];
  alignas(16) uint4 q[D / 16][C::MT][32];                // fragments of the queries: contraction step, fragment, lane
  float ml[2][C::WARPS][R];
  uint32_t nan_code, nan[R][D / 32];                     // e4m3: a code of NaN among the item's tiles; the channels that it makes NaN, by row
  alignas(8) uint64_t full[STAGES], empty[STAGES];
};
static_assert(sizeof(PmSmem<128, 16>) <= 232448 && sizeof(PmSmem<128, 32>) <= 232448, "shared memory of the paged attention over 8-bit pages");
static_assert(PG_PLAN_BYTES(PG_MAX_B) <= 4 * PM_KT * 64, "the plan lies in the ring of tiles");

__device__ __forceinline__ void pm_tma_4d(void* dst, const void* map, int c0, int c1, int c2, int c3, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_addr_u32(dst)), "l"(map), "r"(smem_addr_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}
__device__ __forceinline__ uint32_t pm_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// e4m3: a code in the high byte of either half; sign, exponent and mantissa moved to their places are 2^-120 of the value (subnormal
// codes become subnormal bf16 values).  int8: a code in the low byte; 128 + its low 7 bits, less 256 or 128 by the sign.  Exact, but that
// e4m3's codes of NaN come out as 480.
template <int KIND>
__device__ __forceinline__ uint32_t pm_value2(uint32_t t, uint32_t& size) {      // size: e4m3, of the codes without their signs
  if (KIND == KCH_FP8_E4M3) {
    size = (t >> 4) & 0x07F007F0u;
    return pm_fma((t & 0x80008000u) | size, 0x7B807B80u, 0x80008000u);
  }
  return pm_fma((t & 0x00800080u) | 0x43004300u, 0xBF80BF80u, (t & 0x007F007Fu) | 0x43004300u);
}
// byte I of x and byte J of y as a pair of values
template <int KIND>
__device__ __forceinline__ uint32_t pm_pair(uint32_t x, uint32_t y, int i, int j, uint32_t& size) {
  const uint32_t sel = KIND == KCH_FP8_E4M3 ? (i << 4) | ((4 + j) << 12) : i | ((4 + j) << 8);
  return pm_value2<KIND>(__byte_perm(x, y, sel), size);
}
// the largest size of two pairs and `most`; a NaN's is the largest of all, 0x7F0
template <int KIND>
__device__ __forceinline__ void pm_most(uint32_t& most, uint32_t s0, uint32_t s1) {
  if (KIND == KCH_FP8_E4M3) most = __vimax3_u16x2(most, s0, s1);
}
__device__ __forceinline__ bool pm_has_nan(uint32_t most) { return most >= 0x07F00000u || (most & 0xFFFFu) >= 0x07F0u; }
// (not volatile: products, conversions and the softmax of a tile may be mixed)
__device__ __forceinline__ void pm_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void pm_mma(float (&d)[2], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {      // rows 8 .. 15: zeros
  float x, y;
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%5}, {%7,%8}, {%9,%10,%11,%11};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(x), "=f"(y)
      : "r"(a[0]), "r"(0), "r"(a[2]), "r"(b0), "r"(b1), "f"(d[0]), "f"(d[1]), "f"(0.f));
}
// which bytes of w are e4m3 codes of NaN (0x7F, 0xFF): their top bits
__device__ __forceinline__ uint32_t pm_nan(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ uint4 pm_lds(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }

// The codes of NaN among the keys [from, to) of a sequence: which channels of which of the item's rows see one (all of them, where it is a
// key's).  Of 256 threads.
template <int D>
__device__ __noinline__ void pm_find_nan(const PgAttend& a, int b, int h, int row0, int rows, PgSeq s, int from, int to, uint32_t (*nan)[D / 32], int tid) {
  constexpr int PIECES = 2 * D / 16;                     // of a key: its own and its value's
  for (int64_t i = tid; i < (int64_t)(to - from) * PIECES; i += 256) {
    const int key = from + (int)(i / PIECES), piece = (int)(i % (D / 16)), page = __ldg(a.bt.table + b * a.bt.ld_table + (key >> a.bt.shift));
    const bool value = i % PIECES >= D / 16;
    if ((unsigned)page >= (unsigned)a.bt.num_pages) continue;
    const int64_t row = ((int64_t)page * a.bt.n_kv + h) * a.page + (key & (a.page - 1));
    const uint4 u = __ldg(reinterpret_cast<const uint4*>((const uint8_t*)(value ? a.v : a.k) + row * D) + piece);
    const uint32_t w[4] = {pm_nan(u.x), pm_nan(u.y), pm_nan(u.z), pm_nan(u.w)};
    uint32_t bits = 0u;
    for (int e = 0; e < 16; ++e) bits |= (w[e >> 2] >> (8 * (e & 3) + 7) & 1u) << e;
    if (!bits) continue;
    for (int r = 0; r < rows; ++r) {
      const int2 keys = pg_sees(a.bt, s, row0 + r);
      if (key < keys.x || key >= keys.y) continue;
      if (value) atomicOr(&nan[r][piece / 2], bits << (16 * (piece & 1)));
      else for (int k = 0; k < D / 32; ++k) atomicOr(&nan[r][k], 0xFFFFFFFFu);
    }
  }
}

template <int D, int KIND, int R>
__global__ void __launch_bounds__(PmCfg<R>::THREADS, 1)
paged_attend_mma_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PgAttend a) {
  typedef PmSmem<D, R> S;
  typedef PmCfg<R> C;
  typedef PgWalk<R, PM_KT, 0> Walk;
  extern __shared__ __align__(1024) uint8_t pm_raw[];
  S& sm = *reinterpret_cast<S*>(pm_raw);
  if (smem_addr_u32(pm_raw) & 1023) {                    // (every block begins its memory there)
    if (threadIdx.x == 0) atomicCAS(a.bt.status, 0u, (unsigned)KCH_STATUS_PAGED_ATTEND);
    return;
  }
  const int tid = threadIdx.x, warp = t5_warp_index(), lane = tid & 31, G = a.bt.G, n_kv = a.bt.n_kv;
  if (tid == 0) {
    for (int i = 0; i < S::STAGES; ++i) { mbarrier_init(&sm.full[i], 4); mbarrier_init(&sm.empty[i], C::SHARE); }
    sm.nan_code = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&kmap) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&vmap) : "memory");
  }
  const PgPlace place = pg_plan<R, PM_KT, 0>(a.bt, sm.k, blockIdx.x, gridDim.x);
  pg_zero_rest(a, 2, blockIdx.x, gridDim.x);
  t5_fence_async_smem();                                 // (the plan was read from the ring's memory, which copies write next)
  __syncthreads();
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbarrier_wait_bounded(bar, parity & 1, KCH_STATUS_PAGED_ATTEND, PM_SPIN, a.bt.status); };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REG_FEED));
    // ------------------------------ pages into the ring: keys, values and the scales of either a warp, a box each lane ------------
    // (one warp that issued all four took 180 us for 64 sequences in pages of 16 whose bytes are 45 us)
    const int box = min(a.page, PM_KT), boxes = PM_KT / box;
    const bool mine = lane < boxes, scales = warp >= 2, values = warp & 1;
    int g = 0;
    bool ok = true;
    for (Walk w(a.bt, place); w.valid() && ok; w.next()) {
      const int end = w.first + w.count;
      const int32_t* pages = a.bt.table + (int64_t)w.b * a.bt.ld_table;
      // a box of which some row may see a key: not before the first window, not behind the sequence's end
      auto needed = [&](int tile, int key) { return mine && tile < w.x.tiles && key + box > w.x.lo && key < w.s.kv; };
      // asked for a tile ahead; -1 where it is not needed
      auto ask = [&](int tile) -> int {
        const int key = w.x.first_key + tile * PM_KT + lane * box;
        return tile < end && needed(tile, key) ? __ldg(pages + (key >> a.bt.shift)) : -1;
      };
      int id = ask(w.first);
      for (int tile = w.first; tile < end && ok; ++tile, ++g) {
        const int next = ask(tile + 1), st = g % S::STAGES, key = w.x.first_key + tile * PM_KT + lane * box;
        ok = g < S::STAGES || wait(&sm.empty[st], g / S::STAGES - 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const bool there = mine && (unsigned)id < (unsigned)a.bt.num_pages;
        const unsigned some = __ballot_sync(0xffffffffu, there);
        if (mine && !there) {                            // zeros: codes by a coordinate out of range, scales by hand
          if (needed(tile, key)) pg_bad(a.bt);
          if (scales) {
            float4* to = reinterpret_cast<float4*>((values ? sm.vs[st] : sm.ks[st]) + lane * box);
            for (int i = 0; i < box / 4; ++i) to[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            t5_fence_async_smem();                       // (a copy writes there next)
          }
        }
        __syncwarp();
        if (lane == 0) mbarrier_expect_tx(&sm.full[st], scales ? __popc(some) * box * 4 : PM_KT * D);
        __syncwarp();
        const int r0 = key & (a.page - 1);
        if (scales) {
          if (there)
            bulk_copy_g2s((values ? sm.vs[st] : sm.ks[st]) + lane * box, (const float*)(values ? a.vs : a.ks) + ((int64_t)id * n_kv + w.h) * a.page + r0, box * 4,
                          &sm.full[st]);
        } else if (mine) {
          pm_tma_4d((values ? sm.v[st] : sm.k[st]) + lane * box * D, values ? &vmap : &kmap, 0, r0, w.h, there ? id : (int)a.bt.num_pages, &sm.full[st]);
        }
        id = next;
      }
    }
    // no copy is in flight when the block ends (after a wait that ran out nobody else may have waited for the last ones)
    for (int i = 1; i <= S::STAGES && i <= g; ++i) wait(&sm.full[(g - i) % S::STAGES], (g - i) / S::STAGES);
    return;
  }

  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REG_WORK));
  // ------------------------------ the warps that compute ---------------------------------------------------------------------------------
  constexpr int KS = D / 16, NT = D / 8, RUN = D / 4;    // contraction steps; column tiles; channels of a key a thread has
  const int g = lane >> 2, t = lane & 3, cw = warp - 4, ct = tid - 128;      // (counted from the first of them)
  const float sc = fmaxf(fabsf(a.scale), 1e-30f);        // (not 0: a masked logit is -inf)
  const float raise = 8.f / sc;
  const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;      // the sign goes to the queries: a maximum stays one
  const auto sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(32 * C::WARPS) : "memory"); };
  // byte of the tile at which the 16-byte word `c` of row r lies (D = 128: words swizzled by the row; D = 64: by every second)
  const auto word = [](int r, int c) { return r * D + ((D == 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3)) << 4); };
  int n = 0;                                             // tiles of the ring
  bool ok = true, part = false;
  for (Walk w(a.bt, place); w.valid(); w.next()) {
    // queries: of step i the lane (g, t) has channels RUN t + 4 i .. + 3 of rows g and g + 8 of each fragment
    for (int i = ct; i < KS * C::MT * 32; i += 32 * C::WARPS) {
      const int ln = i & 31, mt = (i >> 5) % C::MT, step = (i >> 5) / C::MT, d = RUN * (ln & 3) + 4 * step;
      uint2 u[2] = {};
#pragma unroll
      for (int hf = 0; hf < C::F / 2; ++hf) {
        const int r = 16 * mt + (ln >> 2) + 8 * hf, row = w.block * R + r, tok = pg_token(a.bt, row);
        if (r < w.x.rows)
          u[hf] = __ldg(reinterpret_cast<const uint2*>((const bf16*)a.q + (w.s.row0 + tok) * a.ld_q + (w.h * G + row - tok * G) * D + d));
      }
      sm.q[step][mt][ln] = make_uint4(u[0].x ^ flip, u[1].x ^ flip, u[0].y ^ flip, u[1].y ^ flip);
    }
    sync();
    constexpr int HF = C::HF, MT = C::MT, F = C::F;      // (value e of fragment mt: row 16 mt + 8 (e / 2) + g, one of two columns)
    int2 keys[HF];
#pragma unroll
    for (int hf = 0; hf < HF; ++hf)
      keys[hf] = g + 8 * hf < w.x.rows ? pg_sees(a.bt, w.s, w.block * R + g + 8 * hf) : make_int2(0, 0);
    const int2 k0 = pg_sees(a.bt, w.s, w.block * R), k1 = pg_sees(a.bt, w.s, w.block * R + w.x.rows - 1);      // first and last row's
    float m[HF], l[HF], o[NT][MT][4];
#pragma unroll
    for (int hf = 0; hf < HF; ++hf) { m[hf] = -INFINITY; l[hf] = 0.f; }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < MT * 4; ++e) o[j][e / 4][e % 4] = 0.f;
    for (int tile = w.first; tile < w.first + w.count; ++tile, ++n) {
      if (n % (C::WARPS / C::SHARE) != cw / C::SHARE) continue;
      const int st = n % S::STAGES, base = C::SLICE * (cw % C::SHARE), key0 = w.x.first_key + tile * PM_KT + base;      // the warp's keys
      if (ok) ok = wait(&sm.full[st], n / S::STAGES);
      ok = __all_sync(0xffffffffu, ok);
      if (ok && key0 < k1.y && key0 + C::SLICE > k0.x) {
        const uint8_t *tk = sm.k[st], *tv = sm.v[st];
        float s[C::H][MT][F] = {};
        uint32_t most = 0u;                              // e4m3: the largest code
#pragma unroll
        for (int i4 = 0; i4 < KS; i4 += 4) {             // 16 bytes of each key's run
          uint4 kc[C::H];
#pragma unroll
          for (int h = 0; h < C::H; ++h) kc[h] = pm_lds(tk + word(base + 8 * h + g, RUN / 16 * t + (i4 >> 2)));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t q[MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              const uint4 u = sm.q[i4 + i][mt][lane];
              q[mt][0] = u.x; q[mt][1] = u.y; q[mt][2] = u.z; q[mt][3] = u.w;
            }
#pragma unroll
            for (int h = 0; h < C::H; ++h) {
              const uint32_t c = i == 0 ? kc[h].x : i == 1 ? kc[h].y : i == 2 ? kc[h].z : kc[h].w;
              uint32_t s0, s1;
              const uint32_t b0 = pm_pair<KIND>(c, c, 0, 1, s0), b1 = pm_pair<KIND>(c, c, 2, 3, s1);
              pm_most<KIND>(most, s0, s1);
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) pm_mma(s[h][mt], q[mt], b0, b1);
            }
          }
        }
        if (KIND == KCH_FP8_E4M3 && pm_has_nan(most)) *(volatile uint32_t*)&sm.nan_code = 1u;      // (checked behind either product: one word held to the tile's end takes 2 % more)
        // scaled; what a row does not see is -inf
        const bool whole = key0 >= k1.x && key0 + C::SLICE <= k0.y && w.x.rows == R;
        constexpr int E = MT * F;                        // values of a thread in 8 keys; bit E h + e of `sees`
        uint32_t sees = 0xFFFFFFFFu;
        static_assert(C::H * E <= 32, "a bit each");
        if (!whole) {
          sees = 0u;
#pragma unroll
          for (int h = 0; h < C::H; ++h)
#pragma unroll
            for (int e = 0; e < E; ++e) {
              const int key = key0 + 8 * h + 2 * t + (e & 1);
              if (key >= keys[e >> 1].x && key < keys[e >> 1].y) sees |= 1u << (E * h + e);
            }
        }
        float top[HF];
#pragma unroll
        for (int hf = 0; hf < HF; ++hf) top[hf] = -INFINITY;
#pragma unroll
        for (int h = 0; h < C::H; ++h) {
          const float2 f = *reinterpret_cast<const float2*>(&sm.ks[st][base + 8 * h + 2 * t]);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            float& x = s[h][e / F][e % F];
            x = sees & (1u << (E * h + e)) ? x * (e & 1 ? f.y : f.x) : -INFINITY;
            top[e >> 1] = fmaxf(top[e >> 1], x);
          }
        }
        bool up[HF], any = false;                        // a row's maximum is raised only when it is exceeded by 2^8
#pragma unroll
        for (int hf = 0; hf < HF; ++hf) {
          top[hf] = fmaxf(top[hf], __shfl_xor_sync(0xffffffffu, top[hf], 1));
          top[hf] = fmaxf(top[hf], __shfl_xor_sync(0xffffffffu, top[hf], 2));
          up[hf] = m[hf] == -INFINITY ? top[hf] > m[hf] : top[hf] > m[hf] + raise;
          any = any || up[hf];
        }
        if (__any_sync(0xffffffffu, any)) {
#pragma unroll
          for (int hf = 0; hf < HF; ++hf) {
            const float f = up[hf] ? ex2_fast((m[hf] - top[hf]) * sc) : 1.f;
            if (up[hf]) m[hf] = top[hf];
            l[hf] *= f;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              o[j][hf / 2][2 * (hf % 2)] *= f; o[j][hf / 2][2 * (hf % 2) + 1] *= f;
              if (R == 8) { o[j][0][2] *= f; o[j][0][3] *= f; }
            }
          }
        }
        float shift[HF];
#pragma unroll
        for (int hf = 0; hf < HF; ++hf) shift[hf] = m[hf] == -INFINITY ? 0.f : m[hf] * sc;
        uint32_t p[C::H / 2][MT][4] = {}, rest[R == 16 ? C::H / 2 : 1][4] = {};      // P, and what its rounding leaves
#pragma unroll
        for (int h = 0; h < C::H; ++h) {
          const float2 f = *reinterpret_cast<const float2*>(&sm.vs[st][base + 8 * h + 2 * t]);
          float x[E];
#pragma unroll
          for (int e = 0; e < E; ++e) {
            x[e] = ex2_fast(fmaf(s[h][e / F][e % F], sc, -shift[e >> 1]));
            l[e >> 1] += x[e];
            x[e] = sees & (1u << (E * h + e)) ? x[e] * (e & 1 ? f.y : f.x) : 0.f;
          }
#pragma unroll
          for (int hf = 0; hf < HF; ++hf) {
            const uint32_t u = pack2_bf16(x[2 * hf], x[2 * hf + 1]);
            const uint32_t left = pack2_bf16(x[2 * hf] - __uint_as_float(u << 16), x[2 * hf + 1] - __uint_as_float(u & 0xFFFF0000u));
            p[h >> 1][hf / 2][2 * (h & 1) + hf % 2] = u;
            if (R == 8) p[h >> 1][0][2 * (h & 1) + 1] = left;
            if (R == 16) rest[h >> 1][2 * (h & 1) + hf] = left;
          }
        }
        // of the values channels NT g .. NT g + NT - 1 of keys 2t, 2t + 1, 2t + 8, 2t + 9 of either half of the 32
        most = 0u;
#pragma unroll
        for (int b = 0; b < C::H / 2; ++b) {
          uint32_t c[4][NT / 4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = base + 16 * b + 2 * t + (i & 1) + 8 * (i >> 1);
            if constexpr (D == 128) {
              const uint4 u = pm_lds(tv + word(r, g));
              c[i][0] = u.x; c[i][1] = u.y; c[i][2] = u.z; c[i][3] = u.w;
            } else {
              const uint2 u = *reinterpret_cast<const uint2*>(tv + word(r, g >> 1) + 8 * (g & 1));
              c[i][0] = u.x; c[i][1] = u.y;
            }
          }
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            uint32_t s0, s1;
            const uint32_t b0 = pm_pair<KIND>(c[0][j >> 2], c[1][j >> 2], j & 3, j & 3, s0), b1 = pm_pair<KIND>(c[2][j >> 2], c[3][j >> 2], j & 3, j & 3, s1);
            pm_most<KIND>(most, s0, s1);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              pm_mma(o[j][mt], p[b][mt], b0, b1);
              if constexpr (R == 16) pm_mma(o[j][mt], rest[b], b0, b1);
            }
          }
        }
        if (KIND == KCH_FP8_E4M3 && pm_has_nan(most)) *(volatile uint32_t*)&sm.nan_code = 1u;
      }
      __syncwarp();
      if (lane == 0) mbarrier_arrive(&sm.empty[st]);
    }
    if (R == 8) {
#pragma unroll
      for (int j = 0; j < NT; ++j) { o[j][0][0] += o[j][0][2]; o[j][0][1] += o[j][0][3]; }
    }
    // ---- the item's end: the warps' parts of its rows ---------------------------------------------------------------------------
    const bool direct = w.starts() && w.ends();
    float* slot = a.slots + (2 * (int64_t)blockIdx.x + (w.starts() ? 1 : 0)) * pg_slot_floats(a.slot_rows, D);
#pragma unroll
    for (int hf = 0; hf < HF; ++hf) {
      l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 1);
      l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 2);
      if (t == 0) {
        sm.ml[0][cw][g + 8 * hf] = m[hf];
        sm.ml[1][cw][g + 8 * hf] = l[hf];
      }
    }
    sync();
#pragma unroll
    for (int hf = 0; hf < HF; ++hf) {
      if (8 * hf >= w.x.rows) break;                     // (the same for all warps)
      const int i = g + 8 * hf;
      float mm = sm.ml[0][0][i];
#pragma unroll
      for (int k = 1; k < C::WARPS; ++k) mm = fmaxf(mm, sm.ml[0][k][i]);
      const bool none = m[hf] == -INFINITY;              // (a part without a key)
      const float own = none ? 0.f : ex2_fast((m[hf] - mm) * sc);
      float4* mine = reinterpret_cast<float4*>(sm.stage[cw]) + g * (D / 4);
      // 16-byte words of a row, swizzled within runs of 8 so that 8 threads meet in no bank
#pragma unroll
      for (int c = 0; c < RUN / 4; ++c) {
        const int j = 4 * c % NT, mt = hf / 2, e = 2 * (hf % 2) + 4 * c / NT;
        mine[(RUN / 4 * t + c) ^ ((D == 128 ? t : 2 * (t & 1)) + 4 * (g & 1))] =
            none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o[j][mt][e] * own, o[j + 1][mt][e] * own, o[j + 2][mt][e] * own, o[j + 3][mt][e] * own);
      }
      sync();
      for (int k = ct; k < 8 * (D / 4); k += 32 * C::WARPS) {
        const int r = k / (D / 4), c = k % (D / 4), row = 8 * hf + r, tt = c / (RUN / 4);
        if (row >= w.x.rows || !ok) continue;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        const int at = r * (D / 4) + (c ^ ((D == 128 ? tt : 2 * (tt & 1)) + 4 * (r & 1)));
#pragma unroll
        for (int i2 = 0; i2 < C::WARPS; ++i2) {
          const float4 y = reinterpret_cast<const float4*>(sm.stage[i2])[at];
          x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
        }
        float top = sm.ml[0][0][row], sum = 0.f;
#pragma unroll
        for (int i2 = 1; i2 < C::WARPS; ++i2) top = fmaxf(top, sm.ml[0][i2][row]);
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int i2 = 0; i2 < C::WARPS; ++i2) sum += sm.ml[1][i2][row] * ex2_fast((sm.ml[0][i2][row] - ref) * sc);      // (a NaN stays one)
        if (direct) {
          const int rr = w.block * R + row, tok = pg_token(a.bt, rr), head = w.h * G + rr - tok * G;
          float below = sum;
          if (a.sink && sum > 0.f) below += ex2_fast(ld_any(a.sink, head, a.sink_dtype) * PG_LOG2E - ref * sc);
          const float f = sum == 0.f ? 0.f : 1.f / below;
          *reinterpret_cast<uint2*>((bf16*)a.out + ((int64_t)(w.s.row0 + tok) * (n_kv * G) + head) * D + 4 * c) =
              make_uint2(pack2_bf16(x.x * f, x.y * f), pack2_bf16(x.z * f, x.w * f));
        } else {
          *reinterpret_cast<float4*>(slot + (int64_t)row * D + 4 * c) = x;
          if (c == 0) {
            slot[(int64_t)a.slot_rows * D + row] = top * sc;
            slot[(int64_t)a.slot_rows * D + a.slot_rows + row] = sum;
          }
        }
      }
      sync();
    }
    // Codes of NaN (an append writes none) have counted as 480 so far, which reaches no sum but those that they make NaN: all of a row that
    // sees one among the keys, and its channel in a row that sees one among the values.  They are looked for only where there is one.
    if (KIND == KCH_FP8_E4M3 && *(volatile uint32_t*)&sm.nan_code != 0u) {
      sync();                                            // (all have read the word)
      if (ct == 0) *(volatile uint32_t*)&sm.nan_code = 0u;
      for (int i = ct; i < R * (D / 32); i += 32 * C::WARPS) sm.nan[i / (D / 32)][i % (D / 32)] = 0u;
      sync();
      const int part0 = w.x.first_key + w.first * PM_KT;
      pm_find_nan<D>(a, w.b, w.h, w.block * R, w.x.rows, w.s, max(part0, w.x.lo), min(part0 + w.count * PM_KT, w.s.kv), sm.nan, ct);
      sync();
      for (int i = ct; i < w.x.rows * D && ok; i += 32 * C::WARPS) {
        const int row = i / D, d = i % D, rr = w.block * R + row, tok = pg_token(a.bt, rr), head = w.h * G + rr - tok * G;
        if (!(sm.nan[row][d / 32] >> (d & 31) & 1u)) continue;
        if (direct) ((uint16_t*)a.out)[((int64_t)(w.s.row0 + tok) * (n_kv * G) + head) * D + d] = 0x7FC0u;
        else slot[(int64_t)row * D + d] = __uint_as_float(0x7FC00000u);
      }
    }
    if (w.starts() && !w.ends()) {
      part = true;
      if (ct == 0) a.records[blockIdx.x] = {1, w.b, w.h, w.block, w.last(place, blockIdx.x), w.x.rows, w.s.row0};
    }
  }
  if (ct == 0 && !part) a.records[blockIdx.x].valid = 0;
}

// ---- host -------------------------------------------------------------------------------------------------------------------
int kch_make_tensor_map_pages(CUtensorMap* map, const void* base, int elem_bytes, uint64_t pages, uint32_t n_kv, uint32_t page_size, uint32_t c,
                              uint32_t box_rows, bool plain = false);

template <int D, int KIND, int R>
static int pm_launch(const CUtensorMap& km, const CUtensorMap& vm, const PgAttend& a, int ctas, cudaStream_t s) {
  const int smem = (int)sizeof(PmSmem<D, R>);
  static std::atomic<uint64_t> done{0};                  // devices on which the kernel has its shared memory
  int dev = 0;
  KCH_CUDA_OK(cudaGetDevice(&dev));
  if (dev > 63 || !((done.load(std::memory_order_relaxed) >> dev) & 1)) {
    KCH_CUDA_OK(cudaFuncSetAttribute(paged_attend_mma_kernel<D, KIND, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (dev <= 63) done.fetch_or(1ULL << dev, std::memory_order_relaxed);
  }
  paged_attend_mma_kernel<D, KIND, R><<<ctas, PmCfg<R>::THREADS, smem, s>>>(km, vm, a);
  KCH_LAUNCH_OK();
  return KCH_OK;
}

int kch_paged_attend_mma(const PgAttend& a, int kind, int rows, int ctas, cudaStream_t s) {
  CUtensorMap km, vm;
  const int box = a.page < PM_KT ? a.page : PM_KT;
  int rc = kch_make_tensor_map_pages(&km, a.k, 1, (uint64_t)a.bt.num_pages, a.bt.n_kv, a.page, a.c, box);
  if (rc == KCH_OK) rc = kch_make_tensor_map_pages(&vm, a.v, 1, (uint64_t)a.bt.num_pages, a.bt.n_kv, a.page, a.c, box);
  if (rc != KCH_OK) return rc;
#define PM_ROWS(D_, K_)                                                                                      \
  (rows == 8 ? pm_launch<D_, K_, 8>(km, vm, a, ctas, s) : rows == 16 ? pm_launch<D_, K_, 16>(km, vm, a, ctas, s) \
             : pm_launch<D_, K_, 32>(km, vm, a, ctas, s))
#define PM_KIND(D_) (kind == KCH_FP8_E4M3 ? PM_ROWS(D_, KCH_FP8_E4M3) : PM_ROWS(D_, KCH_INT8))
  return a.c == 64 ? PM_KIND(64) : PM_KIND(128);
#undef PM_KIND
#undef PM_ROWS
}
