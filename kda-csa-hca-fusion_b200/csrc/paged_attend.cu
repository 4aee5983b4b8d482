// Attention of new tokens over a paged cache on CUDA cores, the kernel that joins parts of items, and the entry point.
//
//   l_j = scale * <q, k_j>,  o = sum_j 2^(l_j log2 e - m) v_j / (sum_j 2^(l_j log2 e - m) + 2^(sink log2 e - m)),  keys j of the
//   sequence with pos(q) - window < j <= pos(q);  a row without keys is 0.
//
// fp32 (whose products the tensor cores would round) and head widths that the tcgen05 kernel does not have.  An item's ROWS x KT
// scores are a register tile of 4 (1) x 4 a thread over rows and keys staged in shared memory in fp32 (stored values times their
// scale), the softmax keeps a running maximum and sum a row, and the sums stay in registers, a row's columns over 16 threads.
// Measured: chunks of 391 to 700 tokens of three sequences, 4 heads of 64 on 2, fp32: 102 us, of which the join is 11: 8 steps
// a CTA, 19500 clocks each where two CTAs share an SM (13000 where one has it), 8200 of which are the products of both at the FMA rate; the
// plan 5500 clocks and the first loads 3000.  16 rows (few tokens): the rows are padded, 64 sequences of 500 to 4000 tokens take 470 us for 608 MB.
#include <math.h>

#include <type_traits>

#include "mma_utils.cuh"
#include "paged.cuh"

// 8 stored values: the words that hold them, and their values as floats
template <typename P>
struct PgStored {
  static constexpr int ES = sizeof(P), W = 2 * ES;
  uint32_t w[W];
  __device__ __forceinline__ void load(const void* base, int64_t i) {
    const P* p = (const P*)base + i;
    if constexpr (W == 2) {
      const uint2 a = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = a.x; w[1] = a.y;
    } else {
#pragma unroll
      for (int k = 0; k < W / 4; ++k) {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(p) + k);
        w[4 * k] = a.x; w[4 * k + 1] = a.y; w[4 * k + 2] = a.z; w[4 * k + 3] = a.w;
      }
    }
  }
  __device__ __forceinline__ void none() {
#pragma unroll
    for (int k = 0; k < W; ++k) w[k] = 0u;
  }
  __device__ __forceinline__ float value(int e) const {
    if constexpr (ES == 4) return __uint_as_float(w[e]);
    else if constexpr (ES == 2) return __uint_as_float(e & 1 ? w[e >> 1] & 0xFFFF0000u : w[e >> 1] << 16);
    else {
      const uint8_t code = (uint8_t)(w[e >> 2] >> (8 * (e & 3)));
      if constexpr (std::is_same<P, int8_t>::value) return (float)(int8_t)code;
      else {
        __nv_fp8_e4m3 v;
        v.__x = code;
        return float(v);
      }
    }
  }
  __device__ __forceinline__ void put(float* to, float f) const {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      reinterpret_cast<float4*>(to)[k] = make_float4(value(4 * k) * f, value(4 * k + 1) * f, value(4 * k + 2) * f, value(4 * k + 3) * f);
  }
};

// a weight of -0: nothing is seen there (a weight that is merely too small is 0, and 0 times a NaN is one)
__device__ __forceinline__ bool pa_none(float weight) { return __float_as_uint(weight) == 0x80000000u; }

#define PA_KT 64
#define PA_THREADS 256
#define PA_CTAS (2 * KCH_SMS)          // at most, of either attention kernel

// steps that a call can have at most, whatever the lengths on the device (of which no two share a row)
static int64_t pa_steps(const PgBatch& a, int rows, int tile) { return ((int64_t)a.N * a.G / rows + a.B) * a.n_kv * (a.cap / tile + 1); }

static constexpr int pa_smem(int ROWS, int DMAX) { return (ROWS * (DMAX + 4) + 2 * PA_KT * (DMAX + 4) + ROWS * (PA_KT + 4) + 3 * ROWS) * 4; }
static_assert(pa_smem(64, 256) <= 232448 && PG_PLAN_BYTES(PG_MAX_B) <= pa_smem(16, 64), "shared memory; the plan lies in the tiles' memory");

// T: activations; P: stored values; DMAX: widths up to this (columns behind the width are 0)
template <typename T, typename P, int ROWS, int DMAX>
__global__ void __launch_bounds__(PA_THREADS) paged_attend_simt_kernel(PgAttend a) {
  constexpr int LD = DMAX + 4, LS = PA_KT + 4, RT = ROWS / 16, CT = DMAX / 64;
  extern __shared__ float4 pa_mem[];
  float* sq = reinterpret_cast<float*>(pa_mem);
  float *sk = sq + ROWS * LD, *sv = sk + PA_KT * LD, *sp = sv + PA_KT * LD, *sm = sp + ROWS * LS, *sl = sm + ROWS, *sa = sl + ROWS;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, c = a.c, c8 = c >> 3;
  const PgPlace place = pg_plan<ROWS, PA_KT, 0>(a.bt, pa_mem, blockIdx.x, gridDim.x);
  pg_zero_rest(a, sizeof(T), blockIdx.x, gridDim.x);
  __syncthreads();
  for (int i = tid; i < (ROWS + 2 * PA_KT) * LD; i += PA_THREADS) sq[i] = 0.f;      // columns c .. DMAX of all three stay 0
  PgRecord rec = {};
  const int G = a.bt.G, n_kv = a.bt.n_kv;
  PgWalk<ROWS, PA_KT, 0> w(a.bt, place);
  for (; w.valid(); w.next()) {
    const int r0 = w.block * ROWS;                             // first (token, head) row of the block in its sequence
    __syncthreads();
    for (int i = tid; i < ROWS * c8; i += PA_THREADS) {
      const int r = i / c8, d = i % c8 * 8;
      PgStored<T> x;
      x.none();
      if (r < w.x.rows) {
        const int t = pg_token(a.bt, r0 + r);
        x.load(a.q, (w.s.row0 + t) * a.ld_q + (int64_t)(w.h * G + r0 + r - t * G) * c + d);
      }
      x.put(sq + r * LD + d, 1.f);
    }
    for (int r = tid; r < ROWS; r += PA_THREADS) { sm[r] = -INFINITY; sl[r] = 0.f; }
    float o[RT][CT][4];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < CT; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
    // A tile's words are asked for while the one before it is multiplied (wide rows would take too many registers: not ahead).
    constexpr int CHUNKS = PA_KT * DMAX / 8 / PA_THREADS;
    PgStored<P> kw[CHUNKS], vw[CHUNKS];
    float fk[CHUNKS], fv[CHUNKS];
    auto ask = [&](int st) {
#pragma unroll
      for (int k = 0; k < CHUNKS; ++k) {
        const int i = tid + k * PA_THREADS, j = i / c8, d = i % c8 * 8, pos = w.x.first_key + st * PA_KT + j;
        kw[k].none();                                          // (0 before the window and behind the sequence's end)
        vw[k].none();
        fk[k] = fv[k] = 1.f;
        if (j < PA_KT && pos >= w.x.lo && pos < w.s.kv) {
          const int64_t pg = pg_page(a.bt, w.b, pos >> a.bt.shift);
          if (pg >= 0) {
            const int64_t row = (pg * n_kv + w.h) * a.page + (pos & (a.page - 1));
            kw[k].load(a.k, row * c + d);
            vw[k].load(a.v, row * c + d);
            if (sizeof(P) == 1) { fk[k] = __ldg(a.ks + row); fv[k] = __ldg(a.vs + row); }
          }
        }
      }
    };
    if (DMAX <= 128) ask(w.first);
    for (int st = w.first; st < w.first + w.count; ++st) {
      const int key0 = w.x.first_key + st * PA_KT;
      if (DMAX > 128) ask(st);
      __syncthreads();
#pragma unroll
      for (int k = 0; k < CHUNKS; ++k) {
        const int i = tid + k * PA_THREADS, j = i / c8, d = i % c8 * 8;
        if (j >= PA_KT) break;
        kw[k].put(sk + j * LD + d, fk[k]);
        vw[k].put(sv + j * LD + d, fv[k]);
      }
      __syncthreads();
      if (DMAX <= 128 && st + 1 < w.first + w.count) ask(st + 1);
      float acc[RT][4];                                        // rows ty + 16 i, keys tx + 16 j
#pragma unroll
      for (int i = 0; i < RT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
      for (int d = 0; d < c; d += 4) {
        float4 kk[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) kk[j] = *reinterpret_cast<const float4*>(sk + (tx + 16 * j) * LD + d);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          const float4 qq = *reinterpret_cast<const float4*>(sq + (ty + 16 * i) * LD + d);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            acc[i][j] = fmaf(qq.x, kk[j].x, acc[i][j]);
            acc[i][j] = fmaf(qq.y, kk[j].y, acc[i][j]);
            acc[i][j] = fmaf(qq.z, kk[j].z, acc[i][j]);
            acc[i][j] = fmaf(qq.w, kk[j].w, acc[i][j]);
          }
        }
      }
      // the 16 threads of a row keep its maximum and sum together
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const int r = ty + 16 * i;
        const int2 keys = r < w.x.rows ? pg_sees(a.bt, w.s, r0 + r) : make_int2(0, 0);
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = key0 + tx + 16 * j;
          acc[i][j] = key >= keys.x && key < keys.y ? acc[i][j] * a.scale : -INFINITY;
          top = fmaxf(top, acc[i][j]);
        }
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float was = sm[r], now = fmaxf(was, top), shift = now == -INFINITY ? 0.f : now;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = key0 + tx + 16 * j;
          const float p = ex2_fast(acc[i][j] - shift);
          sp[r * LS + tx + 16 * j] = key >= keys.x && key < keys.y ? p : -0.f;       // (-0: not seen; 0: seen, but too little for 32 bits)
          sum += p;
        }
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        __syncwarp();
        if (tx == 0) {
          const float keep = ex2_fast(was - shift);               // (0 where nothing was)
          sa[r] = keep;
          sl[r] = sl[r] * keep + sum;
          sm[r] = now;
        }
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const float keep = sa[ty + 16 * i];
#pragma unroll
        for (int j = 0; j < CT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][j][e] *= keep;
      }
      // A key that a row does not see must not reach it: 0 times an infinity or a NaN is no 0.  In a tile where every row
      // sees every key nothing is to be skipped.
      const bool whole = key0 >= pg_sees(a.bt, w.s, r0 + w.x.rows - 1).x && key0 + PA_KT <= pg_sees(a.bt, w.s, r0).y;
      auto product = [&](auto masked) {
#pragma unroll 1
        for (int j = 0; j < PA_KT; j += 4) {                   // four keys at a time: their probabilities in one load a row
          float4 p[RT];
#pragma unroll
          for (int i = 0; i < RT; ++i) p[i] = *reinterpret_cast<const float4*>(sp + (ty + 16 * i) * LS + j);
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int x = 0; x < CT; ++x) {
              const float4 vv = *reinterpret_cast<const float4*>(sv + (j + k) * LD + tx * 4 + 64 * x);
#pragma unroll
              for (int i = 0; i < RT; ++i) {
                const float f = k == 0 ? p[i].x : k == 1 ? p[i].y : k == 2 ? p[i].z : p[i].w;
                if (masked() && pa_none(f)) continue;
                o[i][x][0] = fmaf(f, vv.x, o[i][x][0]);
                o[i][x][1] = fmaf(f, vv.y, o[i][x][1]);
                o[i][x][2] = fmaf(f, vv.z, o[i][x][2]);
                o[i][x][3] = fmaf(f, vv.w, o[i][x][3]);
              }
            }
        }
      };
      if (whole) product([] { return false; });
      else product([] { return true; });
    }
    // ---- the item's end: its rows, or its part of them ---------------------------------------------------------------------
    const bool direct = w.starts() && w.ends();
    float* slot = a.slots + (2 * (int64_t)blockIdx.x + (w.starts() ? 1 : 0)) * pg_slot_floats(a.slot_rows, c);
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int r = ty + 16 * i;
      if (r >= w.x.rows) continue;
      const int t = pg_token(a.bt, r0 + r), h = w.h * G + r0 + r - t * G;
      float f = 1.f;
      if (direct) {
        const float m = sm[r], l = sl[r];
        float below = l;
        if (a.sink && l > 0.f) below += ex2_fast(ld_any(a.sink, h, a.sink_dtype) * PG_LOG2E - m);
        f = l == 0.f ? 0.f : 1.f / below;
      }
      T* orow = (T*)a.out + ((int64_t)(w.s.row0 + t) * (n_kv * G) + h) * c;
#pragma unroll
      for (int x = 0; x < CT; ++x) {
        const int d = tx * 4 + 64 * x;
        if (d >= c) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (direct) stf(orow + d + e, o[i][x][e] * f);
          else slot[(int64_t)r * c + d + e] = o[i][x][e];
        }
      }
      if (!direct && tx == 0) {
        slot[(int64_t)a.slot_rows * c + r] = sm[r];
        slot[(int64_t)a.slot_rows * c + a.slot_rows + r] = sl[r];
      }
    }
    if (w.starts() && !w.ends()) {
      rec.valid = 1; rec.b = w.b; rec.h = w.h; rec.block = w.block; rec.rows = w.x.rows; rec.row0 = w.s.row0;
      rec.last = (int)(((int64_t)place.per * blockIdx.x + (place.left - w.count) + w.x.steps - 1) / place.per);   // (it is the last of the range)
    }
  }
  if (tid == 0) a.records[blockIdx.x] = rec;
}

// ---- joining ----------------------------------------------------------------------------------------------------------------
// The rows of all items that are in parts, one after the other over the blocks, in groups of ROWS of an item: 4, or 1 where that
// gives every row a warp (steps of 64 sequences: 6 us, with 4 they take 7 to 8.5).  Where a row has up to 8 parts a group is a warp's:
// lane 8 j + i weighs part i of its row j, so that maxima, sums and sink of the group are a load each, and then the group's values of
// a part come at once.  (A row at a time, each after a search and three dependent loads, the rows of a chunk's items took 20 to 26 us
// where this takes 12 to 14.)  Else a row is a block's: a thread weighs a part, a warp sums every eighth.  (One long sequence's step gives
// a row 74 or 148 parts: a warp a row took 80 us for them; weighed by the warp that sums them 64 rows of 74 took 10, now 8.)  Either sums
// the parts in one order.  4 (8) columns a lane.  Launched to start while the kernel before it drains.
#define PJ_BLOCKS (4 * KCH_SMS)         // at most: those that the SMs hold
#define PJ_WARPS 8
__device__ __forceinline__ void pj_store4(float* p, float a, float b, float c, float d) { *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d); }
__device__ __forceinline__ void pj_store4(bf16* p, float a, float b, float c, float d) {
  const __nv_bfloat162 x = __floats2bfloat162_rn(a, b), y = __floats2bfloat162_rn(c, d);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}
template <typename T, int W, int ROWS>      // W: columns of a lane, in fours; ROWS: of a group
__global__ void __launch_bounds__(32 * PJ_WARPS) paged_join_kernel(PgJoinArgs a, int ctas) {
  __shared__ int before[PA_CTAS + 1], wide[PA_CTAS], many[PA_CTAS], n_many;      // many: the items whose rows are a block's
  __shared__ alignas(16) float part_o[PJ_WARPS][W * 128];
  __shared__ float part_m[PJ_WARPS], part_l[PJ_WARPS], weight[PA_CTAS];
  constexpr int PER = (PA_CTAS + 32 * PJ_WARPS - 1) / (32 * PJ_WARPS);       // parts of a row that a thread weighs
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  chain_wait();
  for (int i = threadIdx.x; i < ctas; i += 32 * PJ_WARPS) {
    const PgRecord rec = a.records[i];
    wide[i] = rec.valid && rec.last - i >= PJ_WARPS;
    before[i + 1] = rec.valid && !wide[i] ? (rec.rows + ROWS - 1) / ROWS : 0;
  }
  __syncthreads();
  if (warp == 0) {                     // groups of the parted items before each
    int run = 0, wides = 0;
    for (int i0 = 0; i0 < ctas; i0 += 32) {
      const int i = i0 + lane, x = run + pg_scan(i < ctas ? before[i + 1] : 0);
      const unsigned who = __ballot_sync(0xffffffffu, i < ctas && wide[i]);
      if (i < ctas) {
        before[i + 1] = x;
        if (wide[i]) many[wides + __popc(who & ((1u << lane) - 1u))] = i;
      }
      wides += __popc(who);
      run = __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) { before[0] = 0; n_many = wides; }
  }
  __syncthreads();
  const int groups = before[ctas];
  const int64_t size = pg_slot_floats(a.slot_rows, a.c), mat = (int64_t)a.slot_rows * a.c;
  auto slot_of = [&](int i, int first) { return a.slots + (2 * (int64_t)i + (i == first ? 1 : 0)) * size; };
  // (a part without keys: what its sums hold does not matter)
  auto weigh = [](float m, float shift) { return m == -INFINITY ? -0.f : ex2_fast(m - shift); };
  auto add = [](float (&o)[4 * W], int x, const float4& v, float f) {
    const bool none = pa_none(f);
    o[4 * x] = none ? o[4 * x] : fmaf(f, v.x, o[4 * x]);
    o[4 * x + 1] = none ? o[4 * x + 1] : fmaf(f, v.y, o[4 * x + 1]);
    o[4 * x + 2] = none ? o[4 * x + 2] : fmaf(f, v.z, o[4 * x + 2]);
    o[4 * x + 3] = none ? o[4 * x + 3] : fmaf(f, v.w, o[4 * x + 3]);
  };
  auto place = [&](const PgRecord& rec, int r, int& h) {      // of the item's row r in the output; its head
    const int row = rec.block * a.R + r, t = row / a.G;
    h = rec.h * a.G + row - t * a.G;
    return (T*)a.out + ((int64_t)(rec.row0 + t) * a.nh + h) * a.c;
  };
  auto factor = [&](float l, int h, float shift) {            // 1 / the row's denominator
    float below = l;
    if (a.sink && l > 0.f) below += ex2_fast(ld_any(a.sink, h, a.sink_dtype) * PG_LOG2E - shift);
    return l == 0.f ? 0.f : 1.f / below;
  };
  auto store = [&](T* out, const float (&o)[4 * W], float f) {
#pragma unroll
    for (int x = 0; x < W; ++x) {
      const int d = 128 * x + 4 * lane;
      if (d < a.c) pj_store4(out + d, o[4 * x] * f, o[4 * x + 1] * f, o[4 * x + 2] * f, o[4 * x + 3] * f);
    }
  };
  for (int g = blockIdx.x * PJ_WARPS + warp; g < groups; g += gridDim.x * PJ_WARPS) {
    int i = 0, hi = ctas;              // the last i with before[i] <= g
    while (hi - i > 1) {
      const int mid = (i + hi) >> 1;
      if (before[mid] <= g) i = mid; else hi = mid;
    }
    const PgRecord rec = a.records[i];
    const int r0 = (g - before[i]) * ROWS, n = rec.last - i + 1, rows = min(rec.rows - r0, ROWS);
    const int r = r0 + (lane >> 3), part = lane & 7;
    float m = -INFINITY, l = 0.f;
    if (part < n && lane >> 3 < rows) {
      const float* s = slot_of(i + part, i) + mat + r;
      m = s[0];
      l = s[a.slot_rows];
    }
    float shift = m;
#pragma unroll
    for (int k = 4; k > 0; k >>= 1) shift = fmaxf(shift, __shfl_xor_sync(0xffffffffu, shift, k));
    if (shift == -INFINITY) shift = 0.f;
    const float weight = weigh(m, shift);
    l *= weight;
#pragma unroll
    for (int k = 4; k > 0; k >>= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
    int h = 0;
    if (lane >> 3 < rows) place(rec, r, h);
    const float f = factor(l, h, shift);
    float o[ROWS][4 * W] = {};
#pragma unroll 2
    for (int k = 0; k < n; ++k) {
      const float* s = slot_of(i + k, i) + (int64_t)r0 * a.c;
      float4 v[ROWS][W];
#pragma unroll
      for (int j = 0; j < ROWS; ++j)
#pragma unroll
        for (int x = 0; x < W; ++x) {
          const int d = 128 * x + 4 * lane;
          v[j][x] = j < rows && d < a.c ? *reinterpret_cast<const float4*>(s + j * a.c + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
      for (int j = 0; j < ROWS; ++j) {
        const float w = __shfl_sync(0xffffffffu, weight, 8 * j + k);
#pragma unroll
        for (int x = 0; x < W; ++x) add(o[j], x, v[j][x], w);
      }
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const float fj = __shfl_sync(0xffffffffu, f, 8 * j);
      if (j < rows) store(place(rec, r0 + j, h), o[j], fj);
    }
  }
  for (int k = 0; k < n_many; ++k) {
    const int i = many[k];
    const PgRecord rec = a.records[i];
    // (items of few rows: each begins with other blocks)
    for (int r = (int)((blockIdx.x + gridDim.x - (unsigned)(k * a.slot_rows) % gridDim.x) % gridDim.x); r < rec.rows; r += gridDim.x) {
      // a thread weighs one part, or two: weights 2^(m_p - shift)
      const int n = rec.last - i + 1;
      float m[PER], l[PER], top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int q = 0; q < PER; ++q) {
        const int p = threadIdx.x + q * 32 * PJ_WARPS;
        const float* s = slot_of(i + (p < n ? p : 0), i) + mat + r;
        m[q] = p < n ? s[0] : -INFINITY;
        l[q] = p < n ? s[a.slot_rows] : 0.f;
        top = fmaxf(top, m[q]);
      }
      top = warp_max(top);
      __syncthreads();                 // (what the row before left has been read)
      if (lane == 0) part_m[warp] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < PJ_WARPS; ++w) top = fmaxf(top, part_m[w]);
      const float shift = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int q = 0; q < PER; ++q) {
        const int p = threadIdx.x + q * 32 * PJ_WARPS;
        const float f = weigh(m[q], shift);
        if (p < n) weight[p] = f;
        sum = fmaf(f, l[q], sum);
      }
      sum = warp_sum(sum);
      if (lane == 0) part_l[warp] = sum;
      __syncthreads();
      float o[4 * W] = {};
#pragma unroll 8
      for (int p = warp; p < n; p += PJ_WARPS) {
        const float* s = slot_of(i + p, i) + (int64_t)r * a.c;
#pragma unroll
        for (int x = 0; x < W; ++x) {
          const int d = 128 * x + 4 * lane;
          if (d < a.c) add(o, x, *reinterpret_cast<const float4*>(s + d), weight[p]);
        }
      }
#pragma unroll
      for (int x = 0; x < W; ++x) *reinterpret_cast<float4*>(&part_o[warp][128 * x + 4 * lane]) = make_float4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
      __syncthreads();
      const int d = threadIdx.x;       // (at most 256 columns, one a thread)
      if (d < a.c) {
        float all = 0.f, below = 0.f;
#pragma unroll
        for (int w = 0; w < PJ_WARPS; ++w) {
          all += part_o[w][d];
          below += part_l[w];
        }
        int h;
        T* out = place(rec, r, h);
        stf(out + d, all * factor(below, h, shift));
      }
    }
  }
}

int kch_paged_join(const PgJoinArgs& a, int ctas, cudaStream_t s) {
  const int64_t rows = (int64_t)ctas * a.slot_rows, want = (rows + PJ_WARPS - 1) / PJ_WARPS;      // that can be in parts (a block each, where the parts are many)
  const dim3 grid((unsigned)(want < PJ_BLOCKS ? want : PJ_BLOCKS)), block(32 * PJ_WARPS);
  KCH_DISPATCH_FLOAT(a.dtype, T, {
    const bool each = rows <= PJ_BLOCKS * PJ_WARPS;
    if (a.c <= 128) KCH_CUDA_OK(kch_launch_chained(each ? paged_join_kernel<T, 1, 1> : paged_join_kernel<T, 1, 4>, grid, block, 0, s, 1, a, ctas));
    else KCH_CUDA_OK(kch_launch_chained(each ? paged_join_kernel<T, 2, 1> : paged_join_kernel<T, 2, 4>, grid, block, 0, s, 1, a, ctas));
  });
  KCH_LAUNCH_OK();
  return KCH_OK;
}

// ---- entry point --------------------------------------------------------------------------------------------------------------
int kch_paged_check(const kch_paged_cache* p, const kch_paged_batch* b, int dtype, const char* fn);
PgBatch kch_paged_batch_of(const kch_paged_cache* p, const kch_paged_batch* b);

bool kch_paged_attend_tc5_supported(int dtype, int c);
int kch_paged_attend_tc5(const PgAttend& a, int kind, int rows, int ctas, cudaStream_t s);
int kch_paged_attend_mma(const PgAttend& a, int kind, int rows, int ctas, cudaStream_t s);

// How a call is run: the kernel, its rows an item, CTAs, rows of a slot of the workspace.  The host knows the rows of a call and its
// sequences, not who has them: what a sequence has on average decides, and every form takes every batch.  Either side, us, few rows /
// chunks, of 64 sequences over 4000 tokens, 16 heads of 128, pages of 64:
//   rows (tokens x heads of a key head) of a sequence: up to 32, an item of the forms for few rows; behind that they read the keys twice.
//     bf16  8 heads: 1 token 55 / 58, 4 (32 rows) 57 / 60, 5 (40 rows) 100 / 61;  16 heads: 2 tokens 37 / 41, 3 (48 rows) 52 / 42
//     e4m3  8 heads: 1 token 46 / 80, 4 68 / 81, 5 126 / 81;  16 heads: 2 tokens 42 / 47, 3 72 / 48;  int8: 47 / 74, 68 / 74, 125 / 75; 41 / 45, 72 / 46
//   tokens of a sequence: up to 4, so that a long chunk among single tokens cannot be most of a batch's work.  With 190 tokens in one sequence
//     and one in each other (4 on average) 4 heads take 118 / 96 (bf16), 145 / 147 (e4m3), 146 / 141 (int8), 2 heads 191 / 174, 245 / 267, 254 / 254; with
//     448 (8 on average) 127 / 100, 223 / 165, 222 / 156, and 246 / 182, 300 / 277, 302 / 265.  Alike ones would go on to 32 rows: 8 tokens of 4 heads
//     96 / 99, 120 / 141, 119 / 133.
//   CUDA cores, 2000 tokens: items of 16 rows / of 64, 4 fp32 heads of 64 on 2: 16 rows 100 / 161, 24 rows 193 / 162;  256 wide, bf16: 375 / 573, 737 / 575.
enum PaForm { PA_TC5, PA_TC5_FEW, PA_MMA, PA_SIMT };
struct PaPlan { PaForm form; int rows, tile, ctas, slot_rows; bool two; };      // two: items of at most half the rows (FEW: all) take two tiles a step
static PaPlan pa_plan(const kch_paged_attend_args* p) {
  PaPlan x;
  const int64_t B = p->batch.B, rows = p->batch.N * (p->nh / p->cache.n_kv);      // of a key head
  if (!kch_paged_attend_tc5_supported(p->dtype, p->cache.c)) x = {PA_SIMT, rows <= 16 * B ? 16 : 64, PA_KT, PA_CTAS, 0, false};
  else if (rows > 32 * B || p->batch.N > 4 * B) x = {PA_TC5, 256, 128, KCH_SMS, 0, true};
  else if (p->cache.kind == KCH_BF16) x = {PA_TC5_FEW, rows <= 16 * B ? 16 : 32, 128, KCH_SMS, 0, true};
  else x = {PA_MMA, rows <= 8 * B ? 8 : rows <= 16 * B ? 16 : 32, 128, KCH_SMS, 0, false};
  x.slot_rows = (int)(rows < x.rows ? (rows + 7) / 8 * 8 : x.rows);      // (slots are stored to in 16-byte words)
  return x;
}

extern "C" int64_t kch_paged_attend_workspace_bytes(const kch_paged_attend_args* p) {
  if (!p || p->cache.n_kv < 1 || p->nh < 1 || p->cache.c < 1) return 0;
  const PaPlan x = pa_plan(p);
  return pg_workspace_bytes(x.ctas, x.slot_rows, p->cache.c);
}

extern "C" int kch_paged_attend(const kch_paged_attend_args* p, void* stream) {
  KCH_REQUIRE(p != nullptr, "kch_paged_attend: null arguments");
  const int rc = kch_paged_check(&p->cache, &p->batch, p->dtype, "kch_paged_attend");
  if (rc != KCH_OK) return rc;
  const int c = p->cache.c, n_kv = p->cache.n_kv;
  KCH_REQUIRE(p->nh >= 1 && p->nh % n_kv == 0, "kch_paged_attend: nh=%d must be a multiple of n_kv=%d", p->nh, n_kv);
  KCH_REQUIRE(p->sliding_window >= 0, "kch_paged_attend: sliding_window=%d must be >= 0 (0: every key)", p->sliding_window);
  KCH_REQUIRE(isfinite(p->scale * PG_LOG2E), "kch_paged_attend: scale=%g must be finite, times log2(e) too", (double)p->scale);
  KCH_REQUIRE(!p->sink || p->sink_dtype == KCH_F32 || p->sink_dtype == KCH_BF16, "kch_paged_attend: sink dtype tag %d", p->sink_dtype);
  KCH_REQUIRE(p->batch.N * p->nh <= 0x7FFFFE00LL && (int64_t)p->nh * c <= 0x7FFFFFFFLL,       // (rows, a block's end among them, and columns in 32 bits)
              "kch_paged_attend: N * nh = %lld rows of q, nh * c = %lld columns", (long long)(p->batch.N * p->nh), (long long)p->nh * c);
  if (p->batch.N == 0) return KCH_OK;
  const int es = p->dtype == KCH_BF16 ? 2 : 4;
  KCH_REQUIRE(p->q && p->out, "kch_paged_attend: null q or out");
  KCH_REQUIRE(p->ld_q >= (int64_t)p->nh * c && p->ld_q * es % 16 == 0 && ((uintptr_t)p->q & 15) == 0 && ((uintptr_t)p->out & 15) == 0,
              "kch_paged_attend: q and out must be 16-byte aligned, tokens of q (ld_q=%lld elements) at least nh * c apart in multiples of 16 bytes",
              (long long)p->ld_q);
  const int64_t need = kch_paged_attend_workspace_bytes(p);
  KCH_REQUIRE(p->workspace && ((uintptr_t)p->workspace & 255) == 0 && p->workspace_bytes >= need,
              "kch_paged_attend: workspace of %lld bytes (256-byte aligned) is too small: %lld needed", (long long)p->workspace_bytes, (long long)need);
  PgAttend a = {};
  a.bt = kch_paged_batch_of(&p->cache, &p->batch);
  a.q = p->q; a.k = p->cache.k; a.v = p->cache.v; a.ks = p->cache.k_scales; a.vs = p->cache.v_scales;
  a.out = p->out; a.ld_q = p->ld_q; a.c = c; a.page = p->cache.page_size; a.zero_rest = p->zero_rest;
  a.bt.window = p->sliding_window;
  pg_set_group(a.bt, p->nh / n_kv);
  a.scale = p->scale * PG_LOG2E;
  a.sink = p->sink; a.sink_dtype = p->sink_dtype;
  a.records = (PgRecord*)p->workspace;
  const PaPlan x = pa_plan(p);
  KCH_REQUIRE(pa_steps(a.bt, x.rows, x.tile) < PG_MOST, "kch_paged_attend: N=%lld rows against tables of %d pages are more than a call takes",
              (long long)p->batch.N, p->batch.max_pages);
  // (an item's queries may be read again while its rows are stored)
  const uintptr_t q0 = (uintptr_t)p->q, q1 = q0 + ((p->batch.N - 1) * p->ld_q + (int64_t)p->nh * c) * es, o0 = (uintptr_t)p->out;
  KCH_REQUIRE(o0 >= q1 || o0 + p->batch.N * p->nh * c * es <= q0, "kch_paged_attend: out overlaps q");
  KCH_REQUIRE(a.bt.status != nullptr, "kch_paged_attend: cannot resolve the device status word");
  a.slots = (float*)((char*)p->workspace + pg_records_bytes(x.ctas));
  a.slot_rows = x.slot_rows;
  cudaStream_t s = kch_stream(stream);
  // Where no block of rows can have two steps, no item is in parts and there is nothing to join.
  const bool whole = a.bt.cap <= x.tile * (x.two && (x.form == PA_TC5_FEW || (int64_t)a.bt.N * a.bt.G <= x.rows / 2) ? 2 : 1);
  const PgJoinArgs j = {a.out, p->dtype, p->nh, a.bt.G, c, x.rows, x.slot_rows, a.sink, a.sink_dtype, a.records, a.slots};
  if (x.form != PA_SIMT) {
    const int rc5 = x.form == PA_MMA ? kch_paged_attend_mma(a, p->cache.kind, x.rows, x.ctas, s)
                                     : kch_paged_attend_tc5(a, p->cache.kind, x.rows, x.ctas, s);
    return rc5 != KCH_OK || whole ? rc5 : kch_paged_join(j, x.ctas, s);
  }
  const int rows = x.rows, dmax = c <= 64 ? 64 : c <= 128 ? 128 : 256, smem = pa_smem(rows, dmax);
#define PA_GO(T_, P_, R_, D_)                                                                                                 \
  do {                                                                                                                        \
    KCH_CUDA_OK(cudaFuncSetAttribute(paged_attend_simt_kernel<T_, P_, R_, D_>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)); \
    paged_attend_simt_kernel<T_, P_, R_, D_><<<x.ctas, PA_THREADS, smem, s>>>(a);                                            \
  } while (0)
#define PA_WIDTH(T_, P_, R_)                                                                                                  \
  do {                                                                                                                        \
    if (dmax == 64) PA_GO(T_, P_, R_, 64);                                                                                    \
    else if (dmax == 128) PA_GO(T_, P_, R_, 128);                                                                             \
    else PA_GO(T_, P_, R_, 256);                                                                                              \
  } while (0)
#define PA_ROWS(T_, P_)                                                                                                       \
  do {                                                                                                                        \
    if (rows == 16) PA_WIDTH(T_, P_, 16);                                                                                     \
    else PA_WIDTH(T_, P_, 64);                                                                                                \
  } while (0)
  if (p->cache.kind == KCH_FP8_E4M3) { if (p->dtype == KCH_F32) PA_ROWS(float, __nv_fp8_e4m3); else PA_ROWS(bf16, __nv_fp8_e4m3); }
  else if (p->cache.kind == KCH_INT8) { if (p->dtype == KCH_F32) PA_ROWS(float, int8_t); else PA_ROWS(bf16, int8_t); }
  else if (p->dtype == KCH_F32) PA_ROWS(float, float);
  else PA_ROWS(bf16, bf16);
  KCH_LAUNCH_OK();
  return whole ? KCH_OK : kch_paged_join(j, x.ctas, s);
}
