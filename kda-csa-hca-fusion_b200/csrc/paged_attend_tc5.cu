// Attention of new tokens over a paged cache on tcgen05 (bf16 activations, heads of 64 or 128; pages in bf16, e4m3 or int8).
// Mathematics and division of the work: paged_attend.cu, paged.cuh.
//
// One persistent CTA an SM.  An item is up to 256 (token, head of the group) rows of a sequence against the key tiles of 128 that
// they see; two softmax warpgroups X = 0, 1 of a row per thread work on
//   rows 0..127 and 128..255 against the same key tile, where the item has more than 128 rows, or
//   the same rows against the even and the odd key tiles (joined in tensor memory when the item ends), where it has not:
//     a step of single tokens then has two tiles under way as well, and is bound by the loads of its keys.
// Roles: warp 0 copies pages by TMA (128-byte swizzle) into a ring of K and V tiles, in the order in which they are used; warp 1
// issues  S_X = Q_X K^T  (M = N = 128) into 128 columns of tensor memory and  O_X += P_X V  with P_X, written by the softmax over
// S_X's columns, as the operand from tensor memory and V as an MN-major operand from the same kind of tile; warps 2, 3 fetch the
// next item's queries.  tcgen05.mma of one CTA complete in the order of issue, so S_X of the next tile may follow P_X V.
// 8-bit pages: four more warps turn the copied payloads into bf16 tiles (exactly: a payload has at most 7 bits of mantissa);
// a row's scale multiplies its logit, or its probability before that is rounded to bf16.
//
// The running maximum of a row is raised, and O_X rescaled, only when a tile exceeds it by 2^8: probabilities up to 256 lose
// nothing in bf16 or in the fp32 sums, and the accumulator makes its way through registers only a few times a row.
//
// Keys behind a sequence's end read as zeros where a whole page is missing (an out-of-range coordinate of the copy) or are what the
// page holds; p = 0 there, which is no mask for an infinity or a NaN.  O shows it, and such a row is then summed again key by key,
// reading only what it sees (pt_slow_row).  Every wait is bounded (status word, see kch_device_status).
#include <cuda.h>
#include <math.h>

#include "paged.cuh"
#include "tc5_utils.cuh"

#define PT_R 256
#define PT_KT 128
#define PT_SPIN (1u << 22)

template <int D, int KIND>
struct PtCfg {
  static constexpr bool Q8 = KIND >= KCH_FP8_E4M3;
  static constexpr int PANELS = D / 64, TILE = PT_KT * D * 2, RAW = PT_KT * D;
  static constexpr int STAGES = Q8 ? (D == 128 ? 3 : 6) : (D == 128 ? 5 : 8), RAWS = Q8 ? (D == 128 ? 3 : 6) : 0;
  static constexpr int SCALES = 4;                       // key tiles whose scales are held
  static constexpr int THREADS = Q8 ? 512 : 384;
};

template <int D, int KIND>
struct PtSmem {
  typedef PtCfg<D, KIND> C;
  alignas(1024) uint8_t q[2][128 * D * 2];
  alignas(1024) uint8_t kv[C::STAGES][C::TILE];
  alignas(16) uint8_t raw[C::RAWS ? C::RAWS : 1][C::RAWS ? C::RAW : 16];      // (a multiple of 1024 before it)
  alignas(16) float scale[C::Q8 ? C::SCALES : 1][2][C::Q8 ? PT_KT : 4];
  float ml[2][2][128];                                   // maximum and sum of either half of an item's keys
  alignas(8) uint64_t full[C::STAGES], empty[C::STAGES];
  uint64_t raw_full[C::RAWS ? C::RAWS : 1], raw_empty[C::RAWS ? C::RAWS : 1];
  uint64_t sc_full[C::SCALES], sc_empty[C::SCALES];
  uint64_t q_full, q_empty, s_full[2], p_full[2], pv_done[2];
  uint32_t tmem;
};
static_assert(sizeof(PtSmem<128, KCH_BF16>) <= 232448 && sizeof(PtSmem<128, KCH_INT8>) <= 232448, "shared memory of the paged attention");
static_assert(PG_PLAN_BYTES(PG_MAX_B) <= 4 * 16384, "the plan lies in the ring of tiles");

__device__ __forceinline__ void pt_tma_4d(void* dst, const void* map, int c0, int c1, int c2, int c3, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_addr_u32(dst)), "l"(map), "r"(smem_addr_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
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
__device__ __forceinline__ uint64_t pt_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// bits [lo, hi) of a 32-bit word (any lo, hi)
__device__ __forceinline__ uint32_t pt_range(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 32);
  return hi > lo ? (0xFFFFFFFFu >> (32 - (hi - lo))) << lo : 0u;
}
// two bf16 values from two 8-bit codes, exactly
__device__ __forceinline__ uint32_t pt_bf16_mul(uint32_t a, uint32_t b) { uint32_t r; asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ uint32_t pt_bf16_sub(uint32_t a, uint32_t b) { uint32_t r; asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
template <int KIND>
__device__ __forceinline__ void pt_codes4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (KIND == KCH_FP8_E4M3) {
    // sign, exponent and mantissa moved to their places are 2^-120 of the value (subnormal codes become subnormal bf16 values)
    const uint32_t a = __byte_perm(w, 0u, 0x1404), b = __byte_perm(w, 0u, 0x3424);
    lo = pt_bf16_mul((a & 0x80008000u) | ((a >> 4) & 0x07F007F0u), 0x7B807B80u);
    hi = pt_bf16_mul((b & 0x80008000u) | ((b >> 4) & 0x07F007F0u), 0x7B807B80u);
  } else {
    // 128 + the low 7 bits, less 256 or 128 by the sign
    const uint32_t a = __byte_perm(w, 0x43434343u, 0x5140), b = __byte_perm(w, 0x43434343u, 0x7362);
    lo = pt_bf16_sub(a & 0xFF7FFF7Fu, a & 0xFF80FF80u);
    hi = pt_bf16_sub(b & 0xFF7FFF7Fu, b & 0xFF80FF80u);
  }
}

// One row on one warp over the keys [from, to), reading only those: sum_j round(p_j) v_j, p_j = 2^(s_j sc - shift); columns c0 ..
// c1 of it go to `dst` (fp32, a part) or `out` (times f, rounded).
template <int D, int KIND>
__device__ __noinline__ void pt_slow_row(const PgAttend& a, int b, int h, const bf16* q, int64_t from, int64_t to, float sc, float shift,
                                         float f, bf16* out, float* dst, int c0, int c1) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  float qv[E], o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) { qv[e] = ldf(q + lane * E + e); o[e] = 0.f; }
  auto value = [&](const void* p, int64_t i) -> float {
    if (KIND == KCH_BF16) return ldf((const bf16*)p + i);
    if (KIND == KCH_INT8) return (float)((const int8_t*)p)[i];
    return float(((const __nv_fp8_e4m3*)p)[i]);
  };
  for (int64_t j = from; j < to; ++j) {
    const int64_t pg = pg_page(a.bt, b, j >> a.bt.shift);
    const int64_t row = (pg * a.n_kv + h) * a.page + (j & (a.page - 1));
    float s = 0.f;
    if (pg >= 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) s = fmaf(qv[e], value(a.k, row * D + lane * E + e), s);
    }
    s = warp_sum(s);
    float vs = 1.f;
    if (KIND != KCH_BF16 && pg >= 0) { s *= a.ks[row]; vs = a.vs[row]; }
    const float p = round_to<bf16>(ex2_fast(fmaf(s, sc, -shift)) * vs);
    if (pg >= 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(p, value(a.v, row * D + lane * E + e), o[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane * E + e;
    if (d < c0 || d >= c1) continue;
    if (dst) dst[d] = o[e]; else stf(out + d, o[e] * f);
  }
}

template <int D, int KIND>
__global__ void __launch_bounds__(PtCfg<D, KIND>::THREADS, 1)
paged_attend_tc5_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PgAttend a) {
  const int slot_rows = a.slot_rows;
  typedef PtCfg<D, KIND> C;
  extern __shared__ __align__(1024) uint8_t pt_raw[];    // (no room to align it by hand; every block begins its memory there)
  PtSmem<D, KIND>& sm = *reinterpret_cast<PtSmem<D, KIND>*>(pt_raw);
  if (smem_addr_u32(pt_raw) & 1023) {
    if (threadIdx.x == 0) atomicCAS(a.bt.status, 0u, (unsigned)KCH_STATUS_PAGED_ATTEND);
    return;
  }
  const int tid = threadIdx.x, warp = t5_warp_index(), lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < C::STAGES; ++i) { mbarrier_init(&sm.full[i], C::Q8 ? 128 : 1); mbarrier_init(&sm.empty[i], 1); }
    for (int i = 0; i < C::RAWS; ++i) { mbarrier_init(&sm.raw_full[i], 1); mbarrier_init(&sm.raw_empty[i], 4); }
    for (int i = 0; i < C::SCALES; ++i) { mbarrier_init(&sm.sc_full[i], 128); mbarrier_init(&sm.sc_empty[i], 8); }
    mbarrier_init(&sm.q_full, 64);
    mbarrier_init(&sm.q_empty, 1);
    for (int i = 0; i < 2; ++i) { mbarrier_init(&sm.s_full[i], 1); mbarrier_init(&sm.p_full[i], 4); mbarrier_init(&sm.pv_done[i], 1); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr_u32(&sm.tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const PgPlace place = pg_plan<PT_R, PT_KT, true>(a.bt, a.G, a.n_kv, a.window, sm.kv, blockIdx.x, gridDim.x);
  pg_zero_rest(a, 2, blockIdx.x, gridDim.x);
  t5_fence_async_smem();                                 // (the plan was read from the ring's memory, which copies write next)
  t5_fence_before();
  __syncthreads();
  t5_fence_after();
  const uint32_t tmem = sm.tmem;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbarrier_wait_bounded(bar, parity & 1, KCH_STATUS_PAGED_ATTEND, PT_SPIN, a.bt.status); };
  typedef PgWalk<PT_R, PT_KT, true> Walk;
  // the tiles of an item's part in the order in which they are used: f(tile, is it the values)
  auto tiles_of = [](const Walk& w, auto f) {
    const int s0 = w.first, s1 = w.first + w.count;
    if (w.x.rows > PT_R / 2) {
      if (!f(s0, false)) return false;
      for (int s = s0; s < s1; ++s) {
        if (!f(s, true)) return false;
        if (s + 1 < s1 && !f(s + 1, false)) return false;
      }
    } else {
      if (!f(2 * s0, false) || !f(2 * s0 + 1, false)) return false;
      for (int s = s0; s < s1; ++s)
        for (int x = 0; x < 2; ++x) {
          if (!f(2 * s + x, true)) return false;
          if (s + 1 < s1 && !f(2 * s + 2 + x, false)) return false;
        }
    }
    return true;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::Q8 ? 56 : 80));
    if (warp == 0) {
      // ------------------------------ pages into the ring -----------------------------------------------------------------
      // A tile is 128 / rows-of-a-box copies for each panel of 64 channels (8-bit pages: whole rows), a lane each.
      const int box = min(a.page, PT_KT), boxes = PT_KT / box, panels = C::Q8 ? 1 : C::PANELS;
      const int mybox = lane / panels, mypanel = lane % panels;
      const bool mine = lane < boxes * panels;
      int g = 0;
      bool ok = true;
      for (Walk w(a.bt, a.G, a.n_kv, a.window, place); w.valid() && ok; w.next()) {
        ok = tiles_of(w, [&](int tile, bool v) {
          const int64_t key = w.x.first_key + (int64_t)tile * PT_KT + mybox * box;
          int64_t pg = a.bt.num_pages;                   // out of range: zeros
          if (mine && tile < w.x.tiles && key < w.s.kv) {
            pg = pg_page(a.bt, w.b, key >> a.bt.shift);
            if (pg < 0) pg = a.bt.num_pages;
          }
          constexpr int N = C::Q8 ? (C::RAWS ? C::RAWS : 1) : C::STAGES;
          const int st = g % N;
          uint64_t *fb = C::Q8 ? &sm.raw_full[C::Q8 ? st : 0] : &sm.full[C::Q8 ? 0 : st], *eb = C::Q8 ? &sm.raw_empty[C::Q8 ? st : 0] : &sm.empty[C::Q8 ? 0 : st];
          bool fine = true;
          if (g >= N) fine = wait(eb, g / N - 1);
          fine = __all_sync(0xffffffffu, fine);
          if (!fine) return false;
          if (lane == 0) mbarrier_expect_tx(fb, C::Q8 ? C::RAW : C::TILE);
          __syncwarp();
          if (mine) {
            uint8_t* dst = C::Q8 ? sm.raw[C::Q8 ? st : 0] + mybox * box * D : sm.kv[C::Q8 ? 0 : st] + mypanel * (PT_KT * 128) + mybox * box * 128;
            pt_tma_4d(dst, v ? &vmap : &kmap, mypanel * 64, (int)(key & (a.page - 1)), w.h, (int)pg, fb);
          }
          ++g;
          return true;
        });
      }
      // no copy is in flight when the block ends (after a wait that ran out nobody else may have waited for the last ones)
      for (int i = 1, n = C::Q8 ? C::RAWS : C::STAGES; i <= n && i <= g; ++i)
        wait(C::Q8 ? &sm.raw_full[C::Q8 ? (g - i) % n : 0] : &sm.full[C::Q8 ? 0 : (g - i) % n], (g - i) / n);
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
        for (Walk w(a.bt, a.G, a.n_kv, a.window, place); w.valid() && ok; w.next(), ++c) {
          const bool pair = w.x.rows > PT_R / 2;
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
      const int t = tid - 64;
      int c = 0;
      bool ok = true;
      for (Walk w(a.bt, a.G, a.n_kv, a.window, place); w.valid() && ok; w.next(), ++c) {
        if (c) ok = wait(&sm.q_empty, c - 1);
        if (!ok) break;
        const int chunks = D / 8, rows = w.x.rows;
        for (int i = t; i < rows * chunks; i += 64) {
          const int r = i / chunks, k = i % chunks;
          const int64_t row = (int64_t)w.block * PT_R + r, tok = row / a.G;
          const bf16* src = (const bf16*)a.q + (w.s.row0 + tok) * a.ld_q + (int64_t)(w.h * a.G + (int)(row - tok * a.G)) * D + k * 8;
          const uint32_t dst = smem_addr_u32(sm.q[r >> 7]) + (k >> 3) * (128 * 128) + (r & 127) * 128 + (((k & 7) ^ (r & 7)) << 4);
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        t5_fence_async_smem();
        mbarrier_arrive(&sm.q_full);
      }
    }
  } else if (warp < 12) {
    // ------------------------------ softmax and the items' ends: a row per thread -----------------------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::Q8 ? 184 : 208));
    const int x = (warp >> 2) - 1, r = (warp & 3) * 32 + lane;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + 128u * x + lane_base, tO = tmem + 256u + lane_base;
    const bool flip = a.scale < 0.f;
    const float sc = fmaxf(fabsf(a.scale), 1e-30f);      // (not 0: a masked logit is -inf)
    const float raise = 8.f / sc;
    bool ok = true;
    int n = 0, kt = 0;                                   // tiles of this warpgroup; key tiles of the CTA
    PgRecord rec = {};
    for (Walk w(a.bt, a.G, a.n_kv, a.window, place); w.valid(); w.next()) {
      const bool pair = w.x.rows > PT_R / 2;
      const int ri = pair ? x * 128 + r : r;             // row of the item
      const bool live = ri < w.x.rows;
      const int64_t row = (int64_t)w.block * PT_R + ri, tok = row / a.G, pos = w.s.t0 + tok;
      const int64_t key_lo = a.window > 0 ? pos - a.window + 1 : 0, key_hi = min(pos + 1, w.s.kv);      // the keys of the row
      float m = -INFINITY, l = 0.f;
      for (int s = 0; s < w.count; ++s, ++n) {
        const int tile = pair ? w.first + s : 2 * (w.first + s) + x;
        const int64_t key0 = w.x.first_key + (int64_t)tile * PT_KT;
        const int lo = (int)max(min(key_lo - key0, (int64_t)PT_KT), (int64_t)0), hi = (int)max(min(key_hi - key0, (int64_t)PT_KT), (int64_t)0);
        const bool whole = __all_sync(0xffffffffu, !live || (lo == 0 && hi == PT_KT)), none = __all_sync(0xffffffffu, !live || hi <= lo);
        const int slot = (pair ? kt : kt + x) % C::SCALES, turn = (pair ? kt : kt + x) / C::SCALES;
        kt += pair ? 1 : 2;
        if (ok) ok = wait(&sm.s_full[x], n);
        if (C::Q8 && ok) ok = wait(&sm.sc_full[slot], turn);
        ok = __all_sync(0xffffffffu, ok);
        t5_fence_after();
        uint32_t pk[64];
        if (none || !ok) {
#pragma unroll
          for (int e = 0; e < 64; ++e) pk[e] = 0u;
        } else {
          uint32_t sv[128];
#pragma unroll
          for (int k = 0; k < 4; ++k) t5_ld32(tS + 32u * k, *reinterpret_cast<uint32_t(*)[32]>(sv + 32 * k));
          t5_wait_ld();
          if (C::Q8) {
            const float4* ks = reinterpret_cast<const float4*>(sm.scale[slot][0]);
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              const float4 f = ks[k];
              sv[4 * k] = __float_as_uint(__uint_as_float(sv[4 * k]) * f.x);
              sv[4 * k + 1] = __float_as_uint(__uint_as_float(sv[4 * k + 1]) * f.y);
              sv[4 * k + 2] = __float_as_uint(__uint_as_float(sv[4 * k + 2]) * f.z);
              sv[4 * k + 3] = __float_as_uint(__uint_as_float(sv[4 * k + 3]) * f.w);
            }
          }
          if (flip) {
#pragma unroll
            for (int e = 0; e < 128; ++e) sv[e] ^= 0x80000000u;
          }
          if (!whole) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t mk = pt_range(lo - 32 * k, hi - 32 * k);
#pragma unroll
              for (int e = 0; e < 32; ++e) sv[32 * k + e] = mk & (1u << e) ? sv[32 * k + e] : 0xFF800000u;
            }
          }
          float t0 = __uint_as_float(sv[0]), t1 = __uint_as_float(sv[1]), t2 = __uint_as_float(sv[2]), t3 = __uint_as_float(sv[3]);
#pragma unroll
          for (int e = 4; e < 128; e += 4) {
            t0 = fmaxf(t0, __uint_as_float(sv[e]));
            t1 = fmaxf(t1, __uint_as_float(sv[e + 1]));
            t2 = fmaxf(t2, __uint_as_float(sv[e + 2]));
            t3 = fmaxf(t3, __uint_as_float(sv[e + 3]));
          }
          const float top = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3));
          if (s == 0) m = top;
          else if (__any_sync(0xffffffffu, top > m + raise)) {
            const float now = fmaxf(m, top), keep = now == -INFINITY ? 1.f : ex2_fast((m - now) * sc);
            m = now;
            l *= keep;
            if (ok) ok = wait(&sm.pv_done[x], n - 1);
            ok = __all_sync(0xffffffffu, ok);
            t5_fence_after();
#pragma unroll
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
          const float4* vs = reinterpret_cast<const float4*>(sm.scale[C::Q8 ? slot : 0][1]);
#pragma unroll
          for (int e = 0; e < 64; ++e) {
            float x0, x1;
            pt_unpack(pt_fma2(pt_pack(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])), sc2, sh2), x0, x1);
            float p0 = ex2_fast(x0), p1 = ex2_fast(x1);
            sum2 = pt_add2(sum2, pt_pack(p0, p1));
            if (C::Q8) {
              const float4 f = vs[e >> 1];
              p0 *= e & 1 ? f.z : f.x;
              p1 *= e & 1 ? f.w : f.y;
            }
            pk[e] = pack2_bf16(p0, p1);
          }
          float la, lb;
          pt_unpack(sum2, la, lb);
          l += la + lb;
        }
        t5_st32(tS, *reinterpret_cast<const uint32_t(*)[32]>(pk));
        t5_st32(tS + 32u, *reinterpret_cast<const uint32_t(*)[32]>(pk + 32));
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
      float w0 = 1.f, w1 = 0.f;                          // weights of O_0 and O_1 in this row
      float mm = m;
      if (!pair) {
        sm.ml[x][0][r] = m;
        sm.ml[x][1][r] = l;
        asm volatile("bar.sync 1, 256;" ::: "memory");   // (O of both is complete)
        const float m0 = sm.ml[0][0][r], m1 = sm.ml[1][0][r];
        mm = fmaxf(m0, m1);
        const float ref = mm == -INFINITY ? 0.f : mm;
        w0 = ex2_fast((m0 - ref) * sc);
        w1 = ex2_fast((m1 - ref) * sc);
        // (a row without a key in one half has weight 0 there and a NaN of that half's sum stays)
        l = sm.ml[0][1][r] * w0 + sm.ml[1][1][r] * w1;
      }
      t5_fence_after();
      const bool direct = w.starts() && w.ends();
      const float shift = mm == -INFINITY ? 0.f : mm * sc;
      const int head = w.h * a.G + (int)(row - tok * a.G);
      float f = 1.f;
      if (direct && live) {
        float below = l;
        if (a.sink && l > 0.f) below += ex2_fast(ld_any(a.sink, head, a.sink_dtype) * PG_LOG2E - shift);
        f = l == 0.f ? 0.f : 1.f / below;
      }
      float* slot = a.slots + (2 * (int64_t)blockIdx.x + (w.starts() ? 1 : 0)) * pg_slot_floats(slot_rows, D);
      bf16* orow = (bf16*)a.out + ((w.s.row0 + tok) * (int64_t)(a.n_kv * a.G) + head) * D;
      const int c0 = pair ? 0 : x * (D / 2), c1 = pair ? D : c0 + D / 2;
      float odd = 0.f;                                   // 0 unless a value of the row is not finite
      // (a pass before the stores: a row that is not finite is summed again instead of being stored)
      for (int col = c0; col < c1; col += 32) {
        uint32_t ov[32];
        t5_ld32(tO + (pair ? 128u * x : 0u) + col, ov);
        t5_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; ++e) odd += __uint_as_float(ov[e]) * 0.f;
        if (!pair) {
          uint32_t o1[32];
          t5_ld32(tO + 128u + col, o1);
          t5_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            odd += __uint_as_float(o1[e]) * 0.f;
            ov[e] = __float_as_uint(__uint_as_float(ov[e]) * w0 + __uint_as_float(o1[e]) * w1);
          }
        }
        if (live && ok) {
          if (direct) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              uint32_t o4[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) o4[e] = pack2_bf16(__uint_as_float(ov[8 * v + 2 * e]) * f, __uint_as_float(ov[8 * v + 2 * e + 1]) * f);
              *reinterpret_cast<uint4*>(orow + col + 8 * v) = make_uint4(o4[0], o4[1], o4[2], o4[3]);
            }
          } else {
#pragma unroll
            for (int v = 0; v < 8; ++v)
              *reinterpret_cast<uint4*>(slot + (int64_t)ri * D + col + 4 * v) = make_uint4(ov[4 * v], ov[4 * v + 1], ov[4 * v + 2], ov[4 * v + 3]);
          }
        }
      }
      if (!direct && live && (pair || x == 0)) {
        slot[(int64_t)slot_rows * D + ri] = mm * sc;
        slot[(int64_t)slot_rows * D + slot_rows + ri] = l;
      }
      unsigned redo = __ballot_sync(0xffffffffu, live && ok && odd != 0.f);
      if (redo) {
        __syncwarp();
        const int64_t part0 = w.x.first_key + (int64_t)w.first * PT_KT * (pair ? 1 : 2), part1 = part0 + (int64_t)w.count * PT_KT * (pair ? 1 : 2);
        while (redo) {
          const int src = __ffs(redo) - 1;
          redo &= redo - 1;
          const int64_t rr = __shfl_sync(0xffffffffu, row, src), lo = __shfl_sync(0xffffffffu, key_lo, src), hi = __shfl_sync(0xffffffffu, key_hi, src);
          const float sh = __shfl_sync(0xffffffffu, shift, src), ff = __shfl_sync(0xffffffffu, f, src);
          const int64_t tk = rr / a.G;
          const int hd = w.h * a.G + (int)(rr - tk * a.G), ir = (int)(rr - (int64_t)w.block * PT_R);
          pt_slow_row<D, KIND>(a, w.b, w.h, (const bf16*)a.q + (w.s.row0 + tk) * a.ld_q + (int64_t)hd * D, max(max(lo, part0), (int64_t)0), min(hi, part1),
                               flip ? -sc : sc, sh, ff, (bf16*)a.out + ((w.s.row0 + tk) * (int64_t)(a.n_kv * a.G) + hd) * D,
                               direct ? nullptr : slot + (int64_t)ir * D, c0, c1);
        }
      }
      t5_fence_before();
      if (!pair) asm volatile("bar.sync 1, 256;" ::: "memory");        // both have read O of both
      if (w.starts() && !w.ends()) {
        rec.valid = 1; rec.b = w.b; rec.h = w.h; rec.block = w.block; rec.rows = w.x.rows; rec.row0 = w.s.row0;
        rec.last = (int)((place.per * blockIdx.x + (place.left - w.count) + w.x.steps - 1) / place.per);
      }
    }
    if (tid == 128) a.records[blockIdx.x] = rec;
  } else {
    // ------------------------------ 8-bit pages: payloads to bf16 tiles, scales ------------------------------------------------
    if constexpr (C::Q8) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(80));
      const int t = tid - 384;
      bool ok = true;
      int g = 0, kt = 0;
      for (Walk w(a.bt, a.G, a.n_kv, a.window, place); w.valid() && ok; w.next()) {
        ok = tiles_of(w, [&](int tile, bool v) {
          const int64_t key = w.x.first_key + (int64_t)tile * PT_KT + t;
          float fk = 0.f, fv = 0.f;                      // (0 behind the end: a scale there may be anything)
          if (!v && tile < w.x.tiles && key < w.s.kv) {
            const int64_t pg = __ldg(a.bt.table + w.b * a.bt.ld_table + (key >> a.bt.shift));
            if (pg >= 0 && pg < a.bt.num_pages) {
              const int64_t srow = (pg * a.n_kv + w.h) * a.page + (key & (a.page - 1));
              fk = __ldg(a.ks + srow);
              fv = __ldg(a.vs + srow);
            }
          }
          bool fine = wait(&sm.raw_full[g % C::RAWS], g / C::RAWS);
          if (fine && g >= C::STAGES) fine = wait(&sm.empty[g % C::STAGES], g / C::STAGES - 1);
          if (fine && !v && kt >= C::SCALES) fine = wait(&sm.sc_empty[kt % C::SCALES], kt / C::SCALES - 1);
          fine = __all_sync(0xffffffffu, fine);
          if (!fine) return false;
          const uint8_t* src = sm.raw[g % C::RAWS];
          uint8_t* dst = sm.kv[g % C::STAGES];
          constexpr int PIECES = D / 8;                  // 8 codes each: 16 bytes of a tile's row
#pragma unroll 4
          for (int i = t; i < PT_KT * PIECES; i += 128) {
            const int row = i / PIECES, k = i % PIECES;
            const uint2 u = *reinterpret_cast<const uint2*>(src + row * D + k * 8);
            uint4 o;
            pt_codes4<KIND>(u.x, o.x, o.y);
            pt_codes4<KIND>(u.y, o.z, o.w);
            *reinterpret_cast<uint4*>(dst + (k >> 3) * (PT_KT * 128) + row * 128 + (((k & 7) ^ (row & 7)) << 4)) = o;
          }
          if (!v) {
            sm.scale[kt % C::SCALES][0][t] = fk;
            sm.scale[kt % C::SCALES][1][t] = fv;
            mbarrier_arrive(&sm.sc_full[kt % C::SCALES]);
            ++kt;
          }
          t5_fence_async_smem();
          mbarrier_arrive(&sm.full[g % C::STAGES]);
          __syncwarp();
          if (lane == 0) mbarrier_arrive(&sm.raw_empty[g % C::RAWS]);
          ++g;
          return true;
        });
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
                              uint32_t box_rows);

bool kch_paged_attend_tc5_supported(int dtype, int c) { return dtype == KCH_BF16 && (c == 64 || c == 128); }

template <int D, int KIND>
static int pt_launch(const CUtensorMap& km, const CUtensorMap& vm, const PgAttend& a, int ctas, cudaStream_t s) {
  const int smem = (int)sizeof(PtSmem<D, KIND>);
  KCH_CUDA_OK(cudaFuncSetAttribute(paged_attend_tc5_kernel<D, KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  paged_attend_tc5_kernel<D, KIND><<<ctas, PtCfg<D, KIND>::THREADS, smem, s>>>(km, vm, a);
  KCH_LAUNCH_OK();
  return KCH_OK;
}

int kch_paged_attend_tc5(const PgAttend& a, int kind, int ctas, cudaStream_t s) {
  CUtensorMap km, vm;
  const int es = kind == KCH_BF16 ? 2 : 1, box = a.page < PT_KT ? a.page : PT_KT;
  int rc = kch_make_tensor_map_pages(&km, a.k, es, (uint64_t)a.bt.num_pages, a.n_kv, a.page, a.c, box);
  if (rc == KCH_OK) rc = kch_make_tensor_map_pages(&vm, a.v, es, (uint64_t)a.bt.num_pages, a.n_kv, a.page, a.c, box);
  if (rc != KCH_OK) return rc;
#define PT_KIND(D_)                                                                        \
  (kind == KCH_BF16 ? pt_launch<D_, KCH_BF16>(km, vm, a, ctas, s)               \
   : kind == KCH_FP8_E4M3 ? pt_launch<D_, KCH_FP8_E4M3>(km, vm, a, ctas, s)     \
                          : pt_launch<D_, KCH_INT8>(km, vm, a, ctas, s))
  return a.c == 64 ? PT_KIND(64) : PT_KIND(128);
#undef PT_KIND
}
