// The paged key / value cache: rows written into their pages (as they are, in 8 bits with a scale a row, or in 4 with one for 32 channels), and
// read back.
//
//   write   s = max_d |x_d| / Q   (Q = 448 for e4m3, 127 for int8; 1 for a row of zeros),   payload_d = round(x_d / s)
//   read    x_d = payload_d * s
//
// One scale a row of c values and key head: it is then a factor of a logit (keys) or of a probability (values), and the products
// of the attention run on payloads, which bf16 holds exactly.  Bound by the bytes: 8 values a thread, a group of threads a row
// (as many as it has such pieces, rounded up to a power of two), the row's maximum over that group by shuffles.  A warp has a token
// and looks its page up once: with the bisection, two lookups and 64-bit divisions for every row of every head, a copy ran at
// half the memory's rate.  Measured: 28708 tokens of 8 key heads of 128 written as bf16 41 us, 5.7 TB/s; 32768 read from e4m3 38 us, 5.4
// TB/s; one token each of 64 sequences, 4 key heads, written as e4m3 and read back 7.6 us for the two launches.
#include <math.h>

#include "paged.cuh"

int kch_paged_check(const kch_paged_cache* p, const kch_paged_batch* b, int dtype, const char* fn) {
  KCH_REQUIRE(dtype == KCH_F32 || dtype == KCH_BF16, "%s: unsupported dtype tag %d", fn, dtype);
  KCH_REQUIRE(p->kind == dtype || p->kind == KCH_FP8_E4M3 || p->kind == KCH_INT8 || p->kind == KCH_INT4,
              "%s: kind=%d: pages hold the activations' type (%d) or one of the 8- and 4-bit kinds", fn, p->kind, dtype);
  KCH_REQUIRE(p->c >= 8 && p->c <= 256 && p->c % 8 == 0, "%s: c=%d must be a multiple of 8 from 8 to 256", fn, p->c);
  KCH_REQUIRE(p->kind != KCH_INT4 || p->c % 32 == 0, "%s: c=%d must be a multiple of 32, the channels of a scale in 4 bits", fn, p->c);
  KCH_REQUIRE(p->page_size >= 8 && p->page_size <= 256 && (p->page_size & (p->page_size - 1)) == 0,
              "%s: page_size=%d must be a power of two from 8 to 256", fn, p->page_size);
  KCH_REQUIRE(p->n_kv >= 1, "%s: n_kv=%d must be >= 1", fn, p->n_kv);
  KCH_REQUIRE(p->num_pages >= 1 && p->num_pages <= 0x7FFFFFFFLL, "%s: num_pages=%lld out of range", fn, (long long)p->num_pages);
  KCH_REQUIRE(b->B >= 1 && b->B <= PG_MAX_B, "%s: B=%d sequences must be from 1 to %d", fn, b->B, PG_MAX_B);
  KCH_REQUIRE(b->N >= 0 && b->N <= 0x7FFFFFFFLL, "%s: N=%lld rows out of range", fn, (long long)b->N);
  KCH_REQUIRE(b->max_pages >= 1 && b->ld_table >= b->max_pages, "%s: max_pages=%d, rows of the table %lld apart", fn, b->max_pages,
              (long long)b->ld_table);
  KCH_REQUIRE(b->table && b->t0 && b->cu_seqlens, "%s: null table, t0 or cu_seqlens", fn);
  KCH_REQUIRE(p->k && p->v && (((uintptr_t)p->k | (uintptr_t)p->v) & 15) == 0, "%s: pages must be 16-byte aligned", fn);
  KCH_REQUIRE(p->kind < KCH_FP8_E4M3 || (p->k_scales && p->v_scales && (((uintptr_t)p->k_scales | (uintptr_t)p->v_scales) & 15) == 0),
              "%s: 8- and 4-bit pages need their scales, 16-byte aligned", fn);
  return KCH_OK;
}

PgBatch kch_paged_batch_of(const kch_paged_cache* p, const kch_paged_batch* b) {
  PgBatch a = {};
  a.n_kv = p->n_kv;
  a.table = b->table; a.ld_table = b->ld_table; a.t0 = b->t0; a.cu = b->cu_seqlens;
  a.B = b->B; a.N = (int)b->N;
  const int64_t cap = (int64_t)b->max_pages * p->page_size;
  a.cap = (int)(cap < 0x7FFFFE00LL ? cap : 0x7FFFFE00LL);      // positions, and the ends of their tiles, in 32 bits
  a.num_pages = p->num_pages;
  a.shift = 0;
  while ((1 << a.shift) < p->page_size) ++a.shift;
  a.status = kch_status_device_ptr();
  return a;
}

struct PgRows {
  PgBatch bt;
  void *x[2]; int64_t ld[2];           // packed rows of k and v, tokens ld elements apart
  void* pages[2]; void* scales[2];
  int n_kv, c, page, kind, zero_rest;
  int tokens;                          // of a warp at a time: 1 or 2
  int parts;                           // warps that share a token's rows
};
#define PC_THREADS 256
#define PC_SMEM_B 2048                 // batches up to this search cu_seqlens in shared memory

// round-to-nearest-even codes of x / s.  The quotient of a product with 1 / s is off by up to 2^-23 of itself: where the codes
// of values 2^-21 to either side differ, the true quotient decides (rounded towards zero with a sticky last bit, so that a
// second rounding cannot fall on the middle between two codes).
__device__ __forceinline__ float pc_quotient(float x, float s) {
  const float q = x / s, r = fmaf(-q, s, x);             // what the rounded quotient leaves, exactly
  uint32_t b = __float_as_uint(q);
  if (r != 0.f) {
    if ((r < 0.f) != (q < 0.f)) --b;                     // |q| was rounded up
    b |= 1u;
  }
  return __uint_as_float(b);
}
__device__ __forceinline__ uint32_t pc_e4m3x2(float lo, float hi) { return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ int pc_int8(float x) { return (int)fminf(fmaxf(rintf(x), -127.f), 127.f); }
__device__ __forceinline__ uint32_t pc_codes2(float x0, float x1, float s, float inv, int kind) {
  const float lo = 1.f - 4.76837158203125e-07f, hi = 1.f + 4.76837158203125e-07f;      // 2^-21
  const float q0 = x0 * inv, q1 = x1 * inv;
  if (kind == KCH_FP8_E4M3) {
    const uint32_t a = pc_e4m3x2(q0 * lo, q1 * lo);
    return a == pc_e4m3x2(q0 * hi, q1 * hi) ? a : pc_e4m3x2(pc_quotient(x0, s), pc_quotient(x1, s));
  }
  int a0 = pc_int8(q0 * lo), a1 = pc_int8(q1 * lo);
  if (a0 != pc_int8(q0 * hi)) a0 = pc_int8(pc_quotient(x0, s));
  if (a1 != pc_int8(q1 * hi)) a1 = pc_int8(pc_quotient(x1, s));
  return ((uint32_t)a0 & 0xFFu) | (((uint32_t)a1 & 0xFFu) << 8);
}

// 4 bits, of 32 channels (4 threads'): the smallest number of 5 bits, 7 times which is `top` or more (top > 0, as bits).  7 s is exact in 32 bits,
// so that the two comparisons are: whether the product with 1 / 7 was rounded up or down does not matter.
#define PC_MOST4 0x7DE00000u           // 7 * 2^122: 24 s, which the attention adds in bf16, stays a number
__device__ __forceinline__ float pc_scale4(uint32_t top) {
  const float most = __uint_as_float(top);
  uint32_t b = (__float_as_uint(most * 0.142857142857142857f) + 0x7FFFFu) & 0xFFF80000u;
  if (7.f * __uint_as_float(b - 0x80000u) >= most) b -= 0x80000u;
  if (7.f * __uint_as_float(b) < most) b += 0x80000u;
  return fmaxf(__uint_as_float(b), 1.17549435e-38f);
}
// The codes of 8 values as a word, the first in its lowest bits: x / s by one Newton step on the residual of x times the reciprocal, plus 1.5 * 2^23 + 8, whose lowest bits
// are then the nearest whole number to the quotient, and 8, ties to even.  A quotient in the middle between two codes comes out exactly;
// bf16 values have no other that is nearer to it than 10^-3 (x has 8 bits, s 5), values in 32 bits have: there the true quotient decides.
template <typename T>
__device__ __forceinline__ uint32_t pc_codes4(const float (&x)[8], float s) {
  float inv;                                             // (within a unit of its last place, which the step makes up for)
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  uint32_t w = 0u;
  float near = 0.f;
#pragma unroll
  for (int e = 7; e >= 0; --e) {
    float q = x[e] * inv;
    q = fmaf(fmaf(-q, s, x[e]), inv, q);
    const float t = q + 12582920.f;
    if constexpr (sizeof(T) == 4) near = fmaxf(near, fabsf(q - (t - 12582920.f)));
    w = w * 16u + __float_as_uint(t);                    // (of 12582912's bits 0x4B400000 is left, shifted: taken off below)
  }
  if constexpr (sizeof(T) == 4) {
    if (near > 0.49999f) {
      w = 0u;
#pragma unroll
      for (int e = 7; e >= 0; --e) w = w * 16u + (uint32_t)((int)rintf(pc_quotient(x[e], s)) + 8);
      return w;
    }
  }
  constexpr uint32_t left = 0x4B400000u * 0x11111111u;
  return w - left;
}

// where packed row t lies: its sequence by bisection of cu_seqlens, then page and row.  Rows (page * n_kv * page_size + row) of the
// pool, -1: it belongs to no sequence, -2: the table has no page for it.
__device__ __forceinline__ int64_t pc_site(const PgRows& a, const int32_t* cu, int t) {
  if (t < cu[0] || t >= cu[a.bt.B]) return -1;
  int lo = 0, hi = a.bt.B;                               // cu[lo] <= t < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid;
  }
  const int before = __ldg(a.bt.t0 + lo);
  const int64_t pos = (int64_t)before + (t - max(cu[lo], 0));      // (a first row in front of the tensor counts as row 0, as in pg_seq)
  if (before < 0 || pos >= a.bt.cap) { pg_bad(a.bt); return -2; }
  const int64_t pg = pg_page(a.bt, lo, (int)pos >> a.bt.shift);
  return pg < 0 ? -2 : pg * a.n_kv * a.page + ((int)pos & (a.page - 1));
}

// 8 activations of a row, as floats
__device__ __forceinline__ void pc_load(const float* p, float (&x)[8]) {
  const float4 a = __ldg((const float4*)p), b = __ldg((const float4*)p + 1);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void pc_load(const bf16* p, float (&x)[8]) {
  const uint4 v = __ldg((const uint4*)p);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) { x[2 * e] = __uint_as_float(w[e] << 16); x[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u); }
}
__device__ __forceinline__ void pc_store(float* p, const float (&x)[8]) {
  *(float4*)p = make_float4(x[0], x[1], x[2], x[3]);
  *((float4*)p + 1) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void pc_store(bf16* p, const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
    w[e] = *reinterpret_cast<const uint32_t*>(&v);
  }
  *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
}
// What a row of c values is in 16-byte words: 8 values a thread.
template <typename T> struct PcWords { uint4 w[sizeof(T) / 2]; };
template <typename T>
__device__ __forceinline__ PcWords<T> pc_words(const void* p) {
  PcWords<T> x;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) x.w[i] = __ldg((const uint4*)p + i);
  return x;
}

// 8 values of 4 bits in bf16, rounded once: 16 + u by the code's place in the mantissa of 16, less 24, times s.
__device__ __forceinline__ uint32_t pc_fma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint4 pc_values4(uint32_t w, uint32_t s) {
  const uint32_t even = w << 3, odd = w >> 1, ss = s | s << 16;      // (of each byte the lower and the upper code, in its bits 3 .. 6)
  uint32_t x[4] = {__byte_perm(even, odd, 0x4400), __byte_perm(even, odd, 0x5511), __byte_perm(even, odd, 0x6622), __byte_perm(even, odd, 0x7733)};
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = pc_fma2(pc_fma2((x[e] & 0x00780078u) | 0x41804180u, 0x3F803F80u, 0xC1C0C1C0u), ss, 0u);
  return make_uint4(x[0], x[1], x[2], x[3]);
}

// A warp has one token, or two where it has lanes for them; GROUP threads a row (key head, k or v) of it.  The page is
// looked up once a token, and four rows a thread are in flight.  Where tokens are few, several warps share one's rows.  READ: pages
// -> packed rows, else packed rows -> pages.
#define PC_FLIGHT 4
template <typename T, int GROUP, bool READ, bool Q8>
__global__ void __launch_bounds__(PC_THREADS) paged_rows_kernel(const __grid_constant__ PgRows a) {
  __shared__ int32_t scu[PC_SMEM_B + 1];
  const int32_t* cu = a.bt.cu;
  if (a.bt.B <= PC_SMEM_B) {
    for (int i = threadIdx.x; i <= a.bt.B; i += PC_THREADS) scu[i] = __ldg(a.bt.cu + i);
    __syncthreads();
    cu = scu;
  }
  const int lane = threadIdx.x & 31, each = 32 / a.tokens, mine = lane & (each - 1);      // lanes of a token, this one among them
  const int d = (mine & (GROUP - 1)) * 8, rows = 2 * a.n_kv, step = each / GROUP * a.parts, row0 = mine / GROUP + each / GROUP * blockIdx.y;
  const bool in_row = d < a.c;
  for (int64_t t0 = ((int64_t)blockIdx.x * (PC_THREADS / 32) + (threadIdx.x >> 5)) * a.tokens; t0 < a.bt.N;
       t0 += (int64_t)gridDim.x * (PC_THREADS / 32) * a.tokens) {
    const int64_t t = t0 + lane / each;
    const int64_t site = t < a.bt.N ? pc_site(a, cu, (int)t) : -1;
    if (!READ && !__any_sync(0xffffffffu, site >= 0)) continue;
    // (k and v of a head one after the other: row 2 h + kv)
    auto packed = [&](int row) { return (T*)a.x[row & 1] + t * a.ld[row & 1] + (int64_t)(row >> 1) * a.c + d; };
    auto pool_row = [&](int row) { return site + (int64_t)(row >> 1) * a.page; };
    if constexpr (!Q8) {
      if ((READ ? t >= a.bt.N : site < 0) || !in_row) continue;
      if (READ && site == -1 && !a.zero_rest) continue;
      for (int r = row0; r < rows; r += step * PC_FLIGHT) {
        PcWords<T> x[PC_FLIGHT] = {};
#pragma unroll
        for (int i = 0; i < PC_FLIGHT; ++i) {
          const int row = r + i * step;
          if (row < rows && site >= 0) x[i] = pc_words<T>(READ ? (const void*)((const T*)a.pages[row & 1] + pool_row(row) * a.c + d) : packed(row));
        }
#pragma unroll
        for (int i = 0; i < PC_FLIGHT; ++i) {
          const int row = r + i * step;
          if (row >= rows) break;
          uint4* to = (uint4*)(READ ? packed(row) : (T*)a.pages[row & 1] + pool_row(row) * a.c + d);
#pragma unroll
          for (int k = 0; k < (int)sizeof(T) / 2; ++k) to[k] = x[i].w[k];
        }
      }
    } else if constexpr (READ) {
      if (t >= a.bt.N || !in_row || (site == -1 && !a.zero_rest)) continue;
      for (int r = row0; r < rows; r += step * PC_FLIGHT) {
        uint2 u[PC_FLIGHT] = {};
        float f[PC_FLIGHT];
#pragma unroll
        for (int i = 0; i < PC_FLIGHT; ++i) {
          const int row = r + i * step;
          f[i] = 0.f;
          if (row < rows && site >= 0) {
            u[i] = __ldg((const uint2*)((const uint8_t*)a.pages[row & 1] + pool_row(row) * a.c + d));
            f[i] = __ldg((const float*)a.scales[row & 1] + pool_row(row));
          }
        }
#pragma unroll
        for (int i = 0; i < PC_FLIGHT; ++i) {
          const int row = r + i * step;
          if (row >= rows) break;
          const uint32_t w[2] = {u[i].x, u[i].y};
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint8_t code = (uint8_t)(w[e >> 2] >> (8 * (e & 3)));
            __nv_fp8_e4m3 v;
            v.__x = code;
            x[e] = (a.kind == KCH_FP8_E4M3 ? float(v) : (float)(int8_t)code) * f[i];
          }
          pc_store(packed(row), x);
        }
      }
    } else {
      const bool here = site >= 0 && in_row;
      // (all lanes of the warp take the same rounds: a row's maximum is found by shuffles)
      for (int r0 = 0; r0 < rows; r0 += step * PC_FLIGHT) {      // (row0 counts from there)
        float x[PC_FLIGHT][8] = {};
#pragma unroll
        for (int i = 0; i < PC_FLIGHT; ++i) {
          const int row = r0 + row0 + i * step;
          if (here && row < rows) pc_load(packed(row), x[i]);
        }
#pragma unroll
        for (int i = 0; i < PC_FLIGHT; ++i) {
          const int row = r0 + row0 + i * step;
          uint32_t top = 0;                              // as bits: a NaN is above an infinity, which is above every number
#pragma unroll
          for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[i][e]) & 0x7FFFFFFFu);
#pragma unroll
          for (int o = GROUP / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
          if (!here || row >= rows) continue;
          const bool finite = top < 0x7F800000u;
          float s = top ? fmaxf(__uint_as_float(top) / (a.kind == KCH_FP8_E4M3 ? 448.f : 127.f), 1.17549435e-38f) : 1.f;
          const float inv = 1.f / s;
          uint32_t w[2];
#pragma unroll
          for (int e = 0; e < 2; ++e)
            w[e] = finite ? pc_codes2(x[i][4 * e], x[i][4 * e + 1], s, inv, a.kind) | pc_codes2(x[i][4 * e + 2], x[i][4 * e + 3], s, inv, a.kind) << 16 : 0u;
          if (!finite) s = __uint_as_float(0x7FC00000u); // a row that is not finite reads as NaN, whichever the kind
          *(uint2*)((uint8_t*)a.pages[row & 1] + pool_row(row) * a.c + d) = make_uint2(w[0], w[1]);
          if (d == 0) ((float*)a.scales[row & 1])[pool_row(row)] = s;
        }
      }
    }
  }
}

// 8-bit pages: one wave of blocks, whose warps walk the tokens; more of them would only wait for the others' end (32768 tokens of 8 heads
// of 128 read from e4m3: 38 us, 42 with 8 to an SM).  Rows that are copied: 8 to an SM, of which it holds 6 (28708 such tokens written
// as bf16: 41 us, 44 in one wave, where an SM that is behind stays so).
template <typename T, int GROUP, bool READ, bool Q8>
static void pc_launch(const PgRows& a, int64_t blocks, cudaStream_t s) {
  static const int resident = [] {
    int n = 0;
    if (!Q8) return 8;
    return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, paged_rows_kernel<T, GROUP, READ, Q8>, PC_THREADS, 0) == cudaSuccess && n > 0 ? n : 4;
  }();
  const int64_t wave = (int64_t)resident * KCH_SMS / a.parts;
  const dim3 grid((unsigned)(blocks < wave ? blocks : wave), (unsigned)a.parts);
  paged_rows_kernel<T, GROUP, READ, Q8><<<grid, PC_THREADS, 0, s>>>(a);
}


// 4 bits.  16 values a thread, so that two of them share a scale; the first rows of a token are asked for before its page is looked up and the next
// ones while these are at work, or (READ) the next token's page behind the rows of this one.  25 609 tokens of 8 key heads of 128, 134 MB either way, which are 20.5 us
// at the copy rate: written in 36.6 us and read in 26.0, call after call; 41.9 and 31.7 with cold caches.  Writing is bound by issue: by the counters 270 instructions for
// 16 values of a thread, look-ups among them, 68 % of the slots.  (With 8 values a thread and each wait behind the other 65 and 36.5 us; two rows of a
// thread in flight, which leaves 24 warps an SM, a tenth more.)
template <typename T> struct Pc16 { uint4 w[sizeof(T)]; };
template <typename T, int GROUP, bool READ>
__global__ void __launch_bounds__(PC_THREADS, (READ || sizeof(T) == 4) ? 1 : 4) paged_rows4_kernel(const __grid_constant__ PgRows a) {
  constexpr int FLIGHT = READ ? 4 : 1;                   // rows of a thread at a time
  __shared__ int32_t scu[PC_SMEM_B + 1];
  const int32_t* cu = a.bt.cu;
  if (a.bt.B <= PC_SMEM_B) {
    for (int i = threadIdx.x; i <= a.bt.B; i += PC_THREADS) scu[i] = __ldg(a.bt.cu + i);
    __syncthreads();
    cu = scu;
  }
  const int lane = threadIdx.x & 31, each = 32 / a.tokens, mine = lane & (each - 1);      // lanes of a token, this one among them
  const int d = (mine & (GROUP - 1)) * 16, rows = 2 * a.n_kv, step = each / GROUP * a.parts, row0 = mine / GROUP + each / GROUP * blockIdx.y;
  const bool in_row = d < a.c;
  const int64_t stride = (int64_t)gridDim.x * (PC_THREADS / 32) * a.tokens;
  int64_t t = ((int64_t)blockIdx.x * (PC_THREADS / 32) + (threadIdx.x >> 5)) * a.tokens + lane / each;
  auto site_of = [&](int64_t t) { return t < a.bt.N ? pc_site(a, cu, (int)t) : -1; };
  int64_t site = READ ? site_of(t) : -1;
  for (; t - lane / each < a.bt.N; t += stride) {
    // (k and v of a head one after the other: row 2 h + kv)
    auto packed = [&](int row) { return (T*)a.x[row & 1] + t * a.ld[row & 1] + (int64_t)(row >> 1) * a.c + d; };
    auto codes = [&](int row) { return (uint2*)((uint8_t*)a.pages[row & 1] + ((site + (int64_t)(row >> 1) * a.page) * a.c + d) / 2); };
    auto mark = [&](int row) { return (uint16_t*)a.scales[row & 1] + (site + (int64_t)(row >> 1) * a.page) * (a.c / 32) + d / 32; };
    if constexpr (READ) {
      const bool fill = t < a.bt.N && in_row && (site != -1 || a.zero_rest);
      int64_t next = -1;
      for (int r = row0; r < rows; r += step * FLIGHT) {
        uint2 u[FLIGHT];
        uint32_t s[FLIGHT];
#pragma unroll
        for (int i = 0; i < FLIGHT; ++i) {
          const int row = r + i * step;
          u[i] = make_uint2(0x88888888u, 0x88888888u);
          s[i] = 0u;
          if (fill && row < rows && site >= 0) {
            u[i] = __ldg(codes(row));
            s[i] = __ldg(mark(row));
          }
        }
        if (r == row0) next = site_of(t + stride);
#pragma unroll
        for (int i = 0; i < FLIGHT; ++i) {
          const int row = r + i * step;
          if (!fill || row >= rows) break;
          if constexpr (sizeof(T) == 2) {
            T* to = packed(row);
            const uint4 x = pc_values4(u[i].x, s[i]), y = pc_values4(u[i].y, s[i]);
            if (((uintptr_t)to & 31) == 0) {             // (in halves, every sector is written twice)
              asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w), "r"(y.x), "r"(y.y),
                           "r"(y.z), "r"(y.w) : "memory");
            } else {
              *(uint4*)to = x;
              *((uint4*)to + 1) = y;
            }
          } else {
            const float f = __uint_as_float(s[i] << 16);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t w = h ? u[i].y : u[i].x;
              float x[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = fmaf((float)((int)((w >> (4 * e)) & 15u) - 8), f, 0.f);      // (0 is +0)
              pc_store(packed(row) + 8 * h, x);
            }
          }
        }
      }
      site = row0 < rows ? next : site_of(t + stride);
    } else {
      // (what belongs to no sequence is not read)
      const bool there = t < a.bt.N && in_row && t >= cu[0] && t < cu[a.bt.B];
      auto ask = [&](int r0, Pc16<T> (&x)[FLIGHT]) {
#pragma unroll
        for (int i = 0; i < FLIGHT; ++i) {
          const int row = r0 + row0 + i * step;
#pragma unroll
          for (int k = 0; k < (int)sizeof(T); ++k) x[i].w[k] = there && row < rows ? __ldg((const uint4*)packed(row) + k) : make_uint4(0u, 0u, 0u, 0u);
        }
      };
      Pc16<T> x[FLIGHT], ahead[FLIGHT];
      ask(0, x);
      site = there ? site_of(t) : -1;
      // (all lanes of the warp take the same rounds: a group's maximum is found by a shuffle)
      for (int r0 = 0; r0 < rows; r0 += step * FLIGHT) {
        if (r0 + step * FLIGHT < rows) ask(r0 + step * FLIGHT, ahead);
#pragma unroll
        for (int i = 0; i < FLIGHT; ++i) {
          const int row = r0 + row0 + i * step;
          float v[2][8];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if constexpr (sizeof(T) == 2) {
              const uint32_t w[8] = {x[i].w[0].x, x[i].w[0].y, x[i].w[0].z, x[i].w[0].w, x[i].w[1].x, x[i].w[1].y, x[i].w[1].z, x[i].w[1].w};
              v[e >> 3][e & 7] = __uint_as_float(e & 1 ? w[e >> 1] & 0xFFFF0000u : w[e >> 1] << 16);
            } else {
              const uint4 w = x[i].w[e >> 2];
              v[e >> 3][e & 7] = __uint_as_float((e & 3) == 0 ? w.x : (e & 3) == 1 ? w.y : (e & 3) == 2 ? w.z : w.w);
            }
          }
          uint32_t top = 0;                              // as bits: a NaN is above an infinity, which is above every number
          if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint4 w = x[i].w[k];
              top = __vimax3_u16x2(top, w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu);
              top = __vimax3_u16x2(top, w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu);
            }
            top = max(top & 0xFFFF0000u, top << 16);
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(v[e >> 3][e & 7]) & 0x7FFFFFFFu);
          }
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
          if (site < 0 || row >= rows) continue;
          const bool number = top <= PC_MOST4;           // (what is not reads as NaN)
          const float s = top && number ? pc_scale4(top) : 1.f;
          *codes(row) = number ? make_uint2(pc_codes4<T>(v[0], s), pc_codes4<T>(v[1], s)) : make_uint2(0x88888888u, 0x88888888u);
          if (d % 32 == 0) *mark(row) = number ? (uint16_t)(__float_as_uint(s) >> 16) : (uint16_t)0x7FC0u;
        }
#pragma unroll
        for (int i = 0; i < FLIGHT; ++i) x[i] = ahead[i];
      }
    }
  }
}

template <typename T, int GROUP, bool READ>
static void pc_launch4(const PgRows& a, int64_t blocks, cudaStream_t s) {
  static const int resident = [] {
    int n = 0;
    return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, paged_rows4_kernel<T, GROUP, READ>, PC_THREADS, 0) == cudaSuccess && n > 0 ? n : 4;
  }();
  const int64_t wave = (int64_t)resident * KCH_SMS / a.parts;
  const dim3 grid((unsigned)(blocks < wave ? blocks : wave), (unsigned)a.parts);
  paged_rows4_kernel<T, GROUP, READ><<<grid, PC_THREADS, 0, s>>>(a);
}

static int rows_impl(const kch_paged_cache* p, const kch_paged_batch* b, void* k, int64_t ld_k, void* v, int64_t ld_v, int dtype,
                     bool read, int zero_rest, void* stream) {
  const char* fn = read ? "kch_paged_read" : "kch_paged_append";
  KCH_REQUIRE(p && b, "%s: null arguments", fn);
  const int rc = kch_paged_check(p, b, dtype, fn);
  if (rc != KCH_OK) return rc;
  if (b->N == 0) return KCH_OK;
  const int es = dtype == KCH_BF16 ? 2 : 4;
  const int64_t width = (int64_t)p->n_kv * p->c;
  KCH_REQUIRE(k && v, "%s: null k or v", fn);
  KCH_REQUIRE(ld_k >= width && ld_v >= width && ld_k * es % 16 == 0 && ld_v * es % 16 == 0 && (((uintptr_t)k | (uintptr_t)v) & 15) == 0,
              "%s: k and v must be 16-byte aligned, their tokens (ld_k=%lld, ld_v=%lld elements) at least n_kv * c apart in multiples of 16 bytes",
              fn, (long long)ld_k, (long long)ld_v);
  PgRows a;
  a.bt = kch_paged_batch_of(p, b);
  KCH_REQUIRE(a.bt.status != nullptr, "%s: cannot resolve the device status word", fn);
  a.x[0] = k; a.x[1] = v; a.ld[0] = ld_k; a.ld[1] = ld_v;
  a.pages[0] = p->k; a.pages[1] = p->v; a.scales[0] = p->k_scales; a.scales[1] = p->v_scales;
  a.n_kv = p->n_kv; a.c = p->c; a.page = p->page_size; a.kind = p->kind; a.zero_rest = zero_rest;
  cudaStream_t s = kch_stream(stream);
  const bool q4 = p->kind == KCH_INT4;
  const int pieces = p->c / (q4 ? 16 : 8), least = q4 ? 4 : 8, group = pieces <= least ? least : pieces <= 2 * least ? 2 * least : 4 * least;
  a.tokens = 2 * p->n_kv * group <= 16 ? 2 : 1;
  const int64_t blocks = ceil_div64(b->N, PC_THREADS / 32 * a.tokens);
  // as many warps to a token as it has rounds of rows, while they are fewer than 16 to an SM
  const int rounds = (int)ceil_div64(2 * p->n_kv * group * a.tokens, 32);
  a.parts = (int)(blocks * (PC_THREADS / 32) >= 16 * KCH_SMS ? 1 : ceil_div64(16 * KCH_SMS, blocks * (PC_THREADS / 32)));
  if (a.parts > rounds) a.parts = rounds;
#define PC_GO(T_, G_, Q_)                                                                                                \
  do {                                                                                                                   \
    if (read) pc_launch<T_, G_, true, Q_>(a, blocks, s);                                                                 \
    else pc_launch<T_, G_, false, Q_>(a, blocks, s);                                                                     \
  } while (0)
#define PC_GO4(T_, G_)                                                                                                   \
  do {                                                                                                                   \
    if (read) pc_launch4<T_, G_, true>(a, blocks, s);                                                                    \
    else pc_launch4<T_, G_, false>(a, blocks, s);                                                                        \
  } while (0)
#define PC_WIDTH4(T_)                                                                                                    \
  do {                                                                                                                   \
    if (group == 4) PC_GO4(T_, 4);                                                                                       \
    else if (group == 8) PC_GO4(T_, 8);                                                                                  \
    else PC_GO4(T_, 16);                                                                                                 \
  } while (0)
#define PC_WIDTH(T_, Q_)                                                                                                 \
  do {                                                                                                                   \
    if (group == 8) PC_GO(T_, 8, Q_);                                                                                    \
    else if (group == 16) PC_GO(T_, 16, Q_);                                                                             \
    else PC_GO(T_, 32, Q_);                                                                                              \
  } while (0)
#define PC_KIND(T_)                                                                                                      \
  do {                                                                                                                   \
    if (q4) PC_WIDTH4(T_);                                                                                               \
    else if (p->kind < KCH_FP8_E4M3) PC_WIDTH(T_, false);                                                                \
    else PC_WIDTH(T_, true);                                                                                             \
  } while (0)
  if (dtype == KCH_BF16) PC_KIND(bf16);
  else PC_KIND(float);
#undef PC_KIND
#undef PC_WIDTH
#undef PC_WIDTH4
#undef PC_GO4
#undef PC_GO
  KCH_LAUNCH_OK();
  return KCH_OK;
}

extern "C" int kch_paged_append(const kch_paged_cache* cache, const kch_paged_batch* batch, const void* k, int64_t ld_k, const void* v,
                                int64_t ld_v, int dtype, void* stream) {
  return rows_impl(cache, batch, const_cast<void*>(k), ld_k, const_cast<void*>(v), ld_v, dtype, false, 0, stream);
}
extern "C" int kch_paged_read(const kch_paged_cache* cache, const kch_paged_batch* batch, void* k, int64_t ld_k, void* v, int64_t ld_v,
                              int dtype, int zero_rest, void* stream) {
  return rows_impl(cache, batch, k, ld_k, v, ld_v, dtype, true, zero_rest, stream);
}
