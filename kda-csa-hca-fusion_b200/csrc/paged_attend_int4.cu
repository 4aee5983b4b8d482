// Attention of few new tokens a sequence over pages in 4 bits (bf16 activations, heads of 64 or 128).
// Mathematics and division of the work: paged_attend.cu, paged.cuh.  A stored value is (u - 8) s, u a code of 4 bits, s the scale of 32 channels.
//
// A step is bound by the pages' bytes, 72 a row of 128 channels, and next to them by the operations that make numbers of the codes: a
// shift, a mask and an FMA for two.  Codes are converted once, in the registers of the warp that multiplies them, whose products
// (mma.sync) take keys, and channels of the values, as their 16 rows and the queries as their 8 columns: half the products that the
// queries as rows would take (paged_attend_mma.cu), and 4 or 8 queries waste nothing.
//   S^T = K Q^T:  a key's code in the mantissa of 16 is 16 + u, and (16 + u) s - 24 s, which is exact (s has 5 bits), an element of the
//     operand.  The order of the contraction is free: thread (g, t) of a fragment has 32 (16) consecutive channels of keys g and g + 8, which
//     are one group's, and the queries' fragments lie in the same order.
//   O^T += V^T P^T:  thread (g, t) has 16 (8) consecutive channels of keys 2t, 2t + 1, 2t + 8, 2t + 9, again one group's; two keys' halves
//     of a word meet by a byte permutation.  P^T comes from S^T by the transposition of 8 x 8 values that the warp has an instruction for.
// A row's maximum is held by the 8 lanes that have its column, who only meet when one of them exceeds it by 2^8; sums stay apart until the end.
// P is rounded to bf16, and what the rounding leaves is multiplied as well, as in the other kinds' steps: up to 4 rows in the other 4 columns, which are the
// same queries again, more rows by products of their own (7 % of the time with 8 rows, 10 % with 16).
// Fragment row g is key rho(g) of its eight, so that keys' words come without meeting in the banks (values' meet two and two).
//
// Measured, 64 sequences, 16 heads of 128 on 4: 8192 tokens in pages of 64 86 us (3.5 TB/s of pages; 89 in pages of 16, 111 of 8), 500 to
// 16000 tokens in pages of 32 90; on two key heads 55, on one 42, of which 20 are the launches, the plan, the first tile and the joining.  Bound by
// issue: by the counters 731 instructions for 32 keys of a warp (all roles), 344 of them the ALU's, which has half the rate and is 53 % busy, 260 the FMA
// pipe's and 32 products, on two warps a scheduler that keep it 56 % busy.
// Tried: 12 warps of 152 registers 86 (and 102 where 8 took 98); a tile's values multiplied while the next one's scores are 92 (registers move); shifts as
// products with powers of two, on the other pipe, 93.  Pages by tensor maps of 64-byte rows: a copy engine's 5 clocks a row are 1280 for a tile.
//
// A scale of NaN (32 channels that were not finite) reaches what sees it: a key's through its logit; a value's is taken for 0 and looked for
// when the item ends, for 0 times it would reach everyone.  So are the scales above 2^123 that no append writes, of which 24 times may be no number:
// what lies behind a sequence's end, or before its window, may hold any bits.
#include <math.h>

#include <atomic>
#include <type_traits>

#include "paged.cuh"
#include "tc5_utils.cuh"

#define P4_KT 128
#define P4_EXTRA 4                     // places of the line before an item's tiles (paged.cuh): its ends take as long as four of them
#define P4_WAIT 4000000000ull          // ns until a wait gives up

// R rows an item: 8 or 16, by what a sequence has.
template <int R>
struct P4Cfg {
  static constexpr int WARPS = 8, THREADS = 128 + 32 * WARPS;       // that compute; the first warpgroup copies
  static constexpr int NT = R / 8;                                  // columns, in eights
  static constexpr int SLICE = 32, SHARE = P4_KT / SLICE, BLOCKS = SLICE / 16;      // a warp's keys of a tile; warps of a tile
  static constexpr int TEAMS = WARPS / SHARE;                       // each takes every TEAMS'th tile
  static constexpr int REG_FEED = 88, REG_WORK = 208, REG_LAUNCH = 65536 / THREADS / 8 * 8;
  static_assert(128 * REG_FEED + 32 * WARPS * REG_WORK <= THREADS * REG_LAUNCH, "register split");
};
template <int D, int R>
struct P4Smem {
  typedef P4Cfg<R> C;
  static constexpr int STAGES = D == 128 ? 8 : 12, ROW = D / 2, GROUPS = D / 32;      // bytes and scales of a row
  alignas(1024) uint8_t k[STAGES][P4_KT * ROW], v[STAGES][P4_KT * ROW];
  alignas(16) uint16_t ks[STAGES][P4_KT * GROUPS], vs[STAGES][P4_KT * GROUPS];
  alignas(16) float stage[C::WARPS][8 * D];
  alignas(16) uint2 q[D / 16][C::NT][32];                // fragments of the queries: contraction step, columns, lane
  float ml[2][C::WARPS][R];
  uint32_t nan_scale, nan[R][GROUPS];                    // a value's odd scale among the keys of the item; the groups that it makes NaN, by row
  alignas(8) uint64_t full[STAGES], empty[STAGES];
};
static_assert(sizeof(P4Smem<128, 16>) <= 232448 && sizeof(P4Smem<64, 16>) <= 232448, "shared memory of the paged attention over 4 bits");
static_assert(PG_PLAN_BYTES(PG_MAX_B) <= 12 * P4_KT * 32, "the plan lies in the ring of tiles");

// A bounded wait that sleeps: a poll returns when the phase is complete, or after 10 us.  (Polls that return at once were an eighth of all
// instructions, on the schedulers that the others compute with.)
__device__ __forceinline__ bool p4_poll(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 10000;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok;
}
__device__ __forceinline__ bool p4_wait_long(uint32_t bar, uint32_t parity, unsigned int* status, unsigned sleep) {
  uint64_t since, now;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(since));
  do {
    if (p4_poll(bar, parity)) return true;
    if (*(volatile unsigned int*)status != 0u) return false;
    if (sleep) __nanosleep(sleep);
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
  } while (now - since < P4_WAIT);
  atomicCAS(status, 0u, (unsigned)KCH_STATUS_PAGED_ATTEND);
  return false;
}
// As a call it keeps the loops short, but the compiler then leaves the registers as they were launched: 8 rows, which have enough of them,
// call (64 sequences of 8192 tokens 86 us, 88 without), 16 do not (38 us where they do 41).
__device__ __noinline__ bool p4_wait_call(uint32_t bar, uint32_t parity, unsigned int* status, unsigned sleep) {
  return p4_wait_long(bar, parity, status, sleep);
}
// What a block that ends waits for: its own copies, whatever the status says (p4_wait_long gives up as soon as another wait has).  10 ms at most.
__device__ __forceinline__ void p4_drain(uint32_t bar, uint32_t parity) {
  for (int i = 0; i < 1000 && !p4_poll(bar, parity); ++i) {}
}
__device__ __forceinline__ uint32_t p4_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// code J of either half of w, as values: J is 0 .. 3, s the scales of both halves, s24 -24 times them; sixteen: 16 in either half, a register
// whose value the compiler does not know (mask and 16 as constants: 64 sequences of 8192 tokens 113 us, 99 so)
template <int J>
__device__ __forceinline__ uint32_t p4_pair(uint32_t w, uint32_t s, uint32_t s24, uint32_t sixteen) {
  uint32_t x = J == 0 ? w << 3 : w >> (4 * J - 3);
  asm("lop3.b32 %0, %1, 0x00780078, %2, 0xEA;" : "=r"(x) : "r"(x), "r"(sixteen));
  return p4_fma(x, s, s24);
}
__device__ __forceinline__ uint32_t p4_s24(uint32_t s) { return p4_fma(s, 0xC1C0C1C0u, 0u); }
__device__ __forceinline__ void p4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t p4_trans(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// which key of its eight a row of the fragments is
__device__ __forceinline__ int p4_rho(int key) { return key ^ (key >> 2 & 1); }
// a scale that no product can take: NaN, an infinity, or above 2^123, of which 24 times still fits bf16 (an append writes up to 2^122)
#define P4_MOST 0x7D00u
__device__ __forceinline__ bool p4_odd(uint32_t s) { return (s & 0x7FFFu) > P4_MOST; }

// Such scales among the values of the keys [from, to) of a sequence: which rows of the item see one, by groups.  Of `threads` threads.
template <int D>
__device__ __noinline__ void p4_find_nan(const PgAttend& a, int b, int h, int row0, int rows, PgSeq s, int from, int to, uint32_t (*nan)[D / 32], int tid,
                                         int threads) {
  constexpr int GROUPS = D / 32;
  for (int64_t i = tid; i < (int64_t)(to - from) * GROUPS; i += threads) {
    const int key = from + (int)(i / GROUPS), group = (int)(i % GROUPS), page = __ldg(a.bt.table + b * a.bt.ld_table + (key >> a.bt.shift));
    if ((unsigned)page >= (unsigned)a.bt.num_pages) continue;
    const int64_t row = ((int64_t)page * a.bt.n_kv + h) * a.page + (key & (a.page - 1));
    if (!p4_odd(__ldg((const uint16_t*)a.vs + row * GROUPS + group))) continue;
    for (int r = 0; r < rows; ++r) {
      const int2 keys = pg_sees(a.bt, s, row0 + r);
      if (key >= keys.x && key < keys.y) *(volatile uint32_t*)&nan[r][group] = 1u;
    }
  }
}

template <int D, int R>
__global__ void __launch_bounds__(P4Cfg<R>::THREADS, 1)
paged_attend_int4_kernel(const __grid_constant__ PgAttend a) {
  typedef P4Smem<D, R> S;
  typedef P4Cfg<R> C;
  typedef PgWalk<R, P4_KT, 0, P4_EXTRA> Walk;
  extern __shared__ __align__(1024) uint8_t p4_raw[];
  S& sm = *reinterpret_cast<S*>(p4_raw);
  if (smem_addr_u32(p4_raw) & 1023) {                    // (every block begins its memory there)
    if (threadIdx.x == 0) atomicCAS(a.bt.status, 0u, (unsigned)KCH_STATUS_PAGED_ATTEND);
    return;
  }
  const int tid = threadIdx.x, warp = t5_warp_index(), lane = tid & 31, G = a.bt.G, n_kv = a.bt.n_kv;
  if (tid == 0) {
    for (int i = 0; i < S::STAGES; ++i) { mbarrier_init(&sm.full[i], 2); mbarrier_init(&sm.empty[i], C::SHARE); }
    sm.nan_scale = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  const PgPlace place = pg_plan<R, P4_KT, 0, P4_EXTRA>(a.bt, sm.k, blockIdx.x, gridDim.x);
  pg_zero_rest(a, 2, blockIdx.x, gridDim.x);
  t5_fence_async_smem();                                 // (the plan was read from the ring's memory, which copies write next)
  __syncthreads();
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (p4_poll(smem_addr_u32(bar), parity & 1)) return true;
    return R == 8 ? p4_wait_call(smem_addr_u32(bar), parity & 1, a.bt.status, warp < 4 ? 300u : 0u)
                  : p4_wait_long(smem_addr_u32(bar), parity & 1, a.bt.status, warp < 4 ? 300u : 0u);
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REG_FEED));
    // ------------------------------ pages into the ring: keys and values of the even and of the odd tiles a warp each, a lane a box of
    // codes (0 .. 15) or of scales (16 .. 31).  (A tile is about a hundred instructions in a row, 1000 cycles beside warps that compute: two
    // warps for all tiles held everyone up.) ------------------------------------------------------------------------------------------------
    const int box = min(a.page, P4_KT), boxes = P4_KT / box, at = lane & 15;
    const bool mine = at < boxes, scales = lane >= 16, values = warp & 1;
    // of this lane's kind: where it lies in the pool, where it goes to (a stage on from there), bytes of a row
    const uint8_t* from = (const uint8_t*)(scales ? (values ? a.vs : a.ks) : values ? a.v : a.k);
    const int bytes = scales ? 2 * S::GROUPS : S::ROW;
    uint8_t* first = (scales ? (uint8_t*)(values ? sm.vs : sm.ks) : (uint8_t*)(values ? sm.v : sm.k)) + at * box * bytes;
    int ahead = warp >> 1, st = ahead, turn = 0, g = 0;  // tiles until this warp's next; its place in the ring, and how often that has been filled; tiles so far
    bool ok = true;
    for (Walk w(a.bt, place); w.valid() && ok; w.next()) {
      const int32_t* pages = a.bt.table + (int64_t)w.b * a.bt.ld_table;
      // a box of which some row may see a key: not before the first window, not behind the sequence's end
      int key0 = w.x.first_key + (w.first + ahead) * P4_KT;
      const int last = min(w.s.kv, w.x.first_key + min(w.first + w.count, w.x.tiles) * P4_KT);
      auto needed = [&](int k) { return mine && k + box > w.x.lo && k < last; };
      // The table is asked for 32 pages at once (those of 2 to 32 tiles), and as many ahead: a page asked for a tile ahead came after 1400 cycles,
      // later than the tile was used up.
      int page0 = key0 >> a.bt.shift;
      auto ask = [&](int from) {
        const int i = from + lane;
        return i >= w.x.lo >> a.bt.shift && i <= (last - 1) >> a.bt.shift ? __ldg(pages + i) : -1;
      };
      int here = ask(page0), then = ask(page0 + 32);
      for (; ahead < w.count && ok; ahead += 2, ++g, key0 += 2 * P4_KT) {
        if ((key0 >> a.bt.shift) - page0 >= 32) {
          page0 += 32;
          here = then;
          then = ask(page0 + 32);
        }
        const int key = key0 + at * box, id = __shfl_sync(0xffffffffu, here, ((key >> a.bt.shift) - page0) & 31);
        ok = turn == 0 || wait(&sm.empty[st], turn - 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const bool there = needed(key) && (unsigned)id < (unsigned)a.bt.num_pages;
        const unsigned some = __ballot_sync(0xffffffffu, there) >> 16;
        uint8_t* to = first + st * (P4_KT * bytes);
        if (mine && !there) {                            // zeros: scales of 0, whatever the codes
          if (needed(key)) pg_bad(a.bt);
          if (scales) {
            for (int j = 0; j < box * bytes; j += 16) *reinterpret_cast<uint4*>(to + j) = make_uint4(0u, 0u, 0u, 0u);
            t5_fence_async_smem();                       // (a copy writes there next)
          }
        }
        __syncwarp();
        if (lane == 0) mbarrier_expect_tx(&sm.full[st], __popc(some) * box * (2 * S::GROUPS + S::ROW));
        __syncwarp();
        if (there) bulk_copy_g2s(to, from + (((int64_t)id * n_kv + w.h) * a.page + (key & (a.page - 1))) * bytes, box * bytes, &sm.full[st]);
        st += 2;
        if (st >= S::STAGES) { st -= S::STAGES; ++turn; }
      }
      ahead -= w.count;
    }
    // no copy is in flight when the block ends (after a wait that ran out nobody else may have waited for the last ones; every other stage
    // is this warp's alone)
    static_assert(S::STAGES % 2 == 0, "stages of two pairs of warps");
    for (int i = 0; i < g && i < S::STAGES / 2; ++i) {
      st -= 2;
      if (st < 0) { st += S::STAGES; --turn; }
      p4_drain(smem_addr_u32(&sm.full[st]), turn & 1);
    }
    return;
  }

  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REG_WORK));
  // ------------------------------ the warps that compute ---------------------------------------------------------------------------------
  constexpr int KS = D / 16, MT = D / 16, RUN = D / 4, NT = C::NT, BL = C::BLOCKS;      // contraction steps; channels in 16s; channels of a key a thread has
  const int g = lane >> 2, t = lane & 3, cw = warp - 4, ct = tid - 128;      // (counted from the first of them)
  const int rho = p4_rho(g);
  uint32_t sixteen;
  asm volatile("mov.b32 %0, 0x41804180;" : "=r"(sixteen));
  const float sc = fmaxf(fabsf(a.scale), 1e-30f);        // (not 0: a masked logit is -inf)
  const float raise = 8.f / sc;
  const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;      // the sign goes to the queries: a maximum stays one
  const auto sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(32 * C::WARPS) : "memory"); };
  int ahead = cw / C::SHARE, st = ahead, turn = 0;       // tiles until this team's next; its place in the ring (TEAMS < STAGES), and how often that has been filled
  bool ok = true, part = false;
  for (Walk w(a.bt, place); w.valid(); w.next()) {
    const bool four = R == 8 && w.x.rows <= 4;           // columns 4 .. 7 are the rows again
    // queries: of step i the lane (g, t) has channels d, d + 4 and d + 1, d + 5 of row g, d = RUN t + 8 (i / 2) + 2 (i % 2)
    for (int i = ct; i < KS * NT * 32; i += 32 * C::WARPS) {
      const int ln = i & 31, nt = (i >> 5) % NT, step = (i >> 5) / NT, d = RUN * (ln & 3) + 8 * (step >> 1) + 2 * (step & 1);
      const int r = 8 * nt + (four ? (ln >> 2) & 3 : ln >> 2), row = w.block * R + r, tok = pg_token(a.bt, row);
      uint2 u = make_uint2(0u, 0u);
      if (r < w.x.rows) {
        const uint32_t* src = reinterpret_cast<const uint32_t*>((const bf16*)a.q + (w.s.row0 + tok) * a.ld_q + (w.h * G + row - tok * G) * D + d);
        const uint32_t x = __ldg(src) ^ flip, y = __ldg(src + 2) ^ flip;      // channels d, d + 1; d + 4, d + 5
        u = make_uint2(__byte_perm(x, y, 0x5410), __byte_perm(x, y, 0x7632));
      }
      sm.q[step][nt][ln] = u;
    }
    sync();
    const int2 k0 = pg_sees(a.bt, w.s, w.block * R), k1 = pg_sees(a.bt, w.s, w.block * R + w.x.rows - 1);      // first and last row's
    // value e of an accumulator: row 8 nt + 2 t + e % 2 of the item (key or channel g, + 8 from e = 2 on)
    float m[NT][2], l[NT][2], o[MT][NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) { m[nt][0] = m[nt][1] = -INFINITY; l[nt][0] = l[nt][1] = 0.f; }
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int e = 0; e < NT * 4; ++e) o[j][e / 4][e % 4] = 0.f;
    const uint2* queries = &sm.q[0][0][lane];
    // The item's tiles, for four rows and for more apart: the same loop for both took the four 97 us where they have 90 (64 sequences of 500 to 16000
    // tokens, 16 heads of 128 on 4).
    auto tiles = [&](auto rows4) {
      constexpr bool twice = decltype(rows4)::value;
      uint2 own[twice ? KS : 1];                         // (four rows' stay in registers; of more, with the rest of P beside it, they would not fit)
      if constexpr (twice) {
#pragma unroll
        for (int i = 0; i < KS; ++i) own[i] = queries[32 * i];
      }
      for (; ahead < w.count; ahead += C::TEAMS) {
        const int base = C::SLICE * (cw % C::SHARE), key0 = w.x.first_key + (w.first + ahead) * P4_KT + base;      // the warp's keys
        if (ok) ok = wait(&sm.full[st], turn);
        ok = __all_sync(0xffffffffu, ok);
        if (ok && key0 < k1.y && key0 + C::SLICE > k0.x) {
          float s[BL][NT][4] = {};
          {
            uint32_t kw[BL][2][RUN / 8], ks[BL][2], k24[BL][2];
#pragma unroll
            for (int x = 0; x < 2 * BL; ++x) {
              const int r = base + 8 * x + rho;
              uint32_t (&to)[RUN / 8] = kw[x >> 1][x & 1];
              if constexpr (D == 128) {
                const uint4 u = *reinterpret_cast<const uint4*>(sm.k[st] + r * S::ROW + 16 * t);
                to[0] = u.x; to[1] = u.y; to[2] = u.z; to[3] = u.w;
              } else {
                const uint2 u = *reinterpret_cast<const uint2*>(sm.k[st] + r * S::ROW + 8 * t);
                to[0] = u.x; to[1] = u.y;
              }
              const uint32_t f = sm.ks[st][r * S::GROUPS + (D == 128 ? t : t >> 1)];
              ks[x >> 1][x & 1] = f | f << 16;
              k24[x >> 1][x & 1] = p4_s24(f | f << 16);
            }
#pragma unroll
            for (int i = 0; i < KS; ++i) {
              uint2 q[NT];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                if constexpr (twice) q[nt] = own[i];
                else q[nt] = queries[32 * (NT * i + nt)];
              }
#pragma unroll
              for (int b = 0; b < BL; ++b) {
                const uint32_t x = kw[b][0][i >> 1], y = kw[b][1][i >> 1], fx = ks[b][0], fy = ks[b][1], gx = k24[b][0], gy = k24[b][1];
                uint32_t a0, a1, a2, a3;
                if (i & 1) {
                  a0 = p4_pair<2>(x, fx, gx, sixteen); a1 = p4_pair<2>(y, fy, gy, sixteen); a2 = p4_pair<3>(x, fx, gx, sixteen); a3 = p4_pair<3>(y, fy, gy, sixteen);
                } else {
                  a0 = p4_pair<0>(x, fx, gx, sixteen); a1 = p4_pair<0>(y, fy, gy, sixteen); a2 = p4_pair<1>(x, fx, gx, sixteen); a3 = p4_pair<1>(y, fy, gy, sixteen);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) p4_mma(s[b][nt], a0, a1, a2, a3, q[nt].x, q[nt].y);
              }
            }
          }
          // what a row does not see is -inf
          if (!(key0 >= k1.x && key0 + C::SLICE <= k0.y)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int r = 8 * nt + 2 * t + e, row = twice ? r & 3 : r;
                const int2 keys = row < w.x.rows ? pg_sees(a.bt, w.s, w.block * R + row) : make_int2(0, 0);
#pragma unroll
                for (int b = 0; b < BL; ++b)
#pragma unroll
                  for (int h = 0; h < 2; ++h) {
                    const int key = key0 + 16 * b + 8 * h + rho;
                    if (!(key >= keys.x && key < keys.y)) s[b][nt][2 * h + e] = -INFINITY;
                  }
              }
          }
          // a row's maximum is raised only when it is exceeded by 2^8
          float top[NT][2];
          bool any = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              top[nt][e] = fmaxf(s[0][nt][e], s[0][nt][2 + e]);
#pragma unroll
              for (int b = 1; b < BL; ++b) top[nt][e] = fmaxf(top[nt][e], fmaxf(s[b][nt][e], s[b][nt][2 + e]));
              any = any || (m[nt][e] == -INFINITY ? top[nt][e] > m[nt][e] : top[nt][e] > m[nt][e] + raise);
            }
          if (__any_sync(0xffffffffu, any)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float& x = top[nt][e];
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                const bool up = m[nt][e] == -INFINITY ? x > m[nt][e] : x > m[nt][e] + raise;
                const float f = up ? ex2_fast((m[nt][e] - x) * sc) : 1.f;
                if (up) m[nt][e] = x;
                l[nt][e] *= f;
#pragma unroll
                for (int j = 0; j < MT; ++j) { o[j][nt][e] *= f; o[j][nt][2 + e] *= f; }
              }
          }
          uint32_t p[BL][NT][2], rest[BL][NT][2];          // P^T: keys 2t, 2t + 1 (and + 8) of row g; what its rounding leaves
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float shift0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0] * sc, shift1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1] * sc;
#pragma unroll
            for (int b = 0; b < BL; ++b)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float x = ex2_fast(fmaf(s[b][nt][2 * h], sc, -shift0)), y = ex2_fast(fmaf(s[b][nt][2 * h + 1], sc, -shift1));
                l[nt][0] += x;
                l[nt][1] += y;
                uint32_t u = pack2_bf16(x, y);
                if constexpr (!twice) rest[b][nt][h] = p4_trans(pack2_bf16(x - __uint_as_float(u << 16), y - __uint_as_float(u & 0xFFFF0000u)));
                else if (t >= 2) u = pack2_bf16(x - __uint_as_float(u << 16), y - __uint_as_float(u & 0xFFFF0000u));
                p[b][nt][h] = p4_trans(u);
              }
          }
          // of the values the lane has channels 16 g .. (8 g ..) of keys 2t, 2t + 1, 2t + 8, 2t + 9
          uint32_t f[BL][4], most = 0u;                    // their scales
#pragma unroll
          for (int i = 0; i < 4 * BL; ++i) {
            f[i >> 2][i & 3] = sm.vs[st][(base + 8 * (i >> 1) + p4_rho(2 * t + (i & 1))) * S::GROUPS + (D == 128 ? g >> 1 : g >> 2)];
            most = max(most, f[i >> 2][i & 3]);
          }
          if (most > P4_MOST) {                            // (or below 0, which an append writes none of)
#pragma unroll
            for (int i = 0; i < 4 * BL; ++i)
              if (p4_odd(f[i >> 2][i & 3])) {
                const int key = key0 + 8 * (i >> 1) + p4_rho(2 * t + (i & 1));
                f[i >> 2][i & 3] = 0u;
                if (key >= w.x.lo && key < w.s.kv) *(volatile uint32_t*)&sm.nan_scale = 1u;      // (else no row sees it)
              }
          }
#pragma unroll
          for (int b = 0; b < BL; ++b) {
            uint32_t vw[4][D / 64];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint8_t* from = sm.v[st] + (base + 16 * b + 8 * (i >> 1) + p4_rho(2 * t + (i & 1))) * S::ROW + D / 16 * g;
              if constexpr (D == 128) {
                const uint2 u = *reinterpret_cast<const uint2*>(from);
                vw[i][0] = u.x; vw[i][1] = u.y;
              } else {
                vw[i][0] = *reinterpret_cast<const uint32_t*>(from);
              }
            }
            const uint32_t fx = f[b][0] | f[b][1] << 16, fy = f[b][2] | f[b][3] << 16, gx = p4_s24(fx), gy = p4_s24(fy);
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
              const uint32_t x0 = __byte_perm(vw[0][i], vw[1][i], 0x5410), x1 = __byte_perm(vw[0][i], vw[1][i], 0x7632);      // channels 0 .. 3, 4 .. 7 of both keys
              const uint32_t y0 = __byte_perm(vw[2][i], vw[3][i], 0x5410), y1 = __byte_perm(vw[2][i], vw[3][i], 0x7632);
#define P4_PV(J_)                                                                                                                        \
    {                                                                                                                                    \
      const uint32_t a0 = p4_pair<J_>(x0, fx, gx, sixteen), a1 = p4_pair<J_>(x1, fx, gx, sixteen), a2 = p4_pair<J_>(y0, fy, gy, sixteen),         \
                     a3 = p4_pair<J_>(y1, fy, gy, sixteen);                                                                                 \
      _Pragma("unroll") for (int nt = 0; nt < NT; ++nt) {                                                                                \
        p4_mma(o[4 * i + J_][nt], a0, a1, a2, a3, p[b][nt][0], p[b][nt][1]);                                                             \
        if constexpr (!twice) p4_mma(o[4 * i + J_][nt], a0, a1, a2, a3, rest[b][nt][0], rest[b][nt][1]);                                 \
      }                                                                                                                                  \
    }
              P4_PV(0) P4_PV(1) P4_PV(2) P4_PV(3)
#undef P4_PV
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbarrier_arrive(&sm.empty[st]);
        st += C::TEAMS;
        if (st >= S::STAGES) { st -= S::STAGES; ++turn; }
      }
    };
    if constexpr (R == 8) {
      if (four) tiles(std::true_type{});
      else tiles(std::false_type{});
    } else {
      tiles(std::false_type{});
    }
    ahead -= w.count;
    if (four) {                                          // (lane t has rows 2 t, 2 t + 1, lane t + 2 what their rounding left)
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][0][e] += __shfl_xor_sync(0xffffffffu, o[j][0][e], 2);
    }
    // ---- the item's end: the warps' parts of its rows ---------------------------------------------------------------------------
    const bool direct = w.starts() && w.ends();
    float* slot = a.slots + (2 * (int64_t)blockIdx.x + (w.starts() ? 1 : 0)) * pg_slot_floats(a.slot_rows, D);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float& x = l[nt][e];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        if (g == 0) {
          sm.ml[0][cw][8 * nt + 2 * t + e] = m[nt][e];
          sm.ml[1][cw][8 * nt + 2 * t + e] = x;
        }
      }
    sync();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (8 * nt >= w.x.rows) break;                     // (the same for all warps)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 2 * t + e;
        float mm = sm.ml[0][0][8 * nt + r];
#pragma unroll
        for (int k = 1; k < C::WARPS; ++k) mm = fmaxf(mm, sm.ml[0][k][8 * nt + r]);
        const bool none = m[nt][e] == -INFINITY;         // (a part without a key)
        const float f = none ? 0.f : ex2_fast((m[nt][e] - mm) * sc);
        float4* to = reinterpret_cast<float4*>(sm.stage[cw]) + r * (D / 4);
        // channels 16 g + 8 i + 4 h .. + 3; words swizzled by the row, so that the lanes of a column do not meet in the banks
#pragma unroll
        for (int i = 0; i < D / 64; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            to[(D / 32 * g + 2 * i + h) ^ t] = none ? make_float4(0.f, 0.f, 0.f, 0.f)
                                                    : make_float4(o[4 * i][nt][2 * h + e] * f, o[4 * i + 1][nt][2 * h + e] * f,
                                                                  o[4 * i + 2][nt][2 * h + e] * f, o[4 * i + 3][nt][2 * h + e] * f);
      }
      sync();
      for (int k = ct; k < 8 * (D / 4); k += 32 * C::WARPS) {
        const int r = k / (D / 4), c = k % (D / 4), row = 8 * nt + r;
        if (row >= w.x.rows || !ok) continue;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        const int at = r * (D / 4) + (c ^ (r >> 1));
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
    // odd scales among the values: the groups of the rows that see one
    if (*(volatile uint32_t*)&sm.nan_scale != 0u) {
      sync();                                            // (all have read the word)
      if (ct == 0) *(volatile uint32_t*)&sm.nan_scale = 0u;
      for (int i = ct; i < R * S::GROUPS; i += 32 * C::WARPS) sm.nan[i / S::GROUPS][i % S::GROUPS] = 0u;
      sync();
      const int part0 = w.x.first_key + w.first * P4_KT;
      p4_find_nan<D>(a, w.b, w.h, w.block * R, w.x.rows, w.s, max(part0, w.x.lo), min(part0 + w.count * P4_KT, w.s.kv), sm.nan, ct, 32 * C::WARPS);
      sync();
      for (int i = ct; i < w.x.rows * D && ok; i += 32 * C::WARPS) {
        const int row = i / D, d = i % D, rr = w.block * R + row, tok = pg_token(a.bt, rr), head = w.h * G + rr - tok * G;
        if (!sm.nan[row][d / 32]) continue;
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
template <int D, int R>
static int p4_launch(const PgAttend& a, int ctas, cudaStream_t s) {
  const int smem = (int)sizeof(P4Smem<D, R>);
  static std::atomic<uint64_t> done{0};                  // devices on which the kernel has its shared memory
  int dev = 0;
  KCH_CUDA_OK(cudaGetDevice(&dev));
  if (dev > 63 || !((done.load(std::memory_order_relaxed) >> dev) & 1)) {
    KCH_CUDA_OK(cudaFuncSetAttribute(paged_attend_int4_kernel<D, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (dev <= 63) done.fetch_or(1ULL << dev, std::memory_order_relaxed);
  }
  paged_attend_int4_kernel<D, R><<<ctas, P4Cfg<R>::THREADS, smem, s>>>(a);
  KCH_LAUNCH_OK();
  return KCH_OK;
}

int kch_paged_attend_int4(const PgAttend& a, int rows, int ctas, cudaStream_t s) {
  if (a.c == 64) return rows == 8 ? p4_launch<64, 8>(a, ctas, s) : p4_launch<64, 16>(a, ctas, s);
  return rows == 8 ? p4_launch<128, 8>(a, ctas, s) : p4_launch<128, 16>(a, ctas, s);
}
