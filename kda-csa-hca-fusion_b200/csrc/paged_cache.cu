// The paged key / value cache: rows written into their pages (as they are, or in 8 bits with a scale a row), and read back.
//
//   write   s = max_d |x_d| / Q   (Q = 448 for e4m3, 127 for int8; 1 for a row of zeros),   payload_d = round(x_d / s)
//   read    x_d = payload_d * s
//
// One scale a row of c values and key head: it is then a factor of a logit (keys) or of a probability (values), and the products
// of the attention run on payloads, which bf16 holds exactly.  Bound by the bytes: 8 values a thread, a group of threads a row
// (as many as it has such pieces, rounded up to a power of two), the row's maximum over that group by shuffles.
#include <math.h>

#include "paged.cuh"

int kch_paged_check(const kch_paged_cache* p, const kch_paged_batch* b, int dtype, const char* fn) {
  KCH_REQUIRE(dtype == KCH_F32 || dtype == KCH_BF16, "%s: unsupported dtype tag %d", fn, dtype);
  KCH_REQUIRE(p->kind == dtype || p->kind == KCH_FP8_E4M3 || p->kind == KCH_INT8,
              "%s: kind=%d: pages hold the activations' type (%d) or one of the 8-bit kinds", fn, p->kind, dtype);
  KCH_REQUIRE(p->c >= 8 && p->c <= 256 && p->c % 8 == 0, "%s: c=%d must be a multiple of 8 from 8 to 256", fn, p->c);
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
  KCH_REQUIRE(p->kind < KCH_FP8_E4M3 || (p->k_scales && p->v_scales), "%s: 8-bit pages need their scales", fn);
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
  void* pages[2]; float* scales[2];
  int n_kv, c, page, kind, zero_rest;
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

// where packed row t lies: its sequence by bisection of cu_seqlens, then page and row; -1: it belongs to no sequence, -2: the
// table has no page for it
__device__ __forceinline__ int64_t pc_site(const PgRows& a, const int32_t* cu, int64_t t, int h) {
  if (t < cu[0] || t >= cu[a.bt.B]) return -1;
  int lo = 0, hi = a.bt.B;                               // cu[lo] <= t < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid;
  }
  const int64_t pos = max((int64_t)__ldg(a.bt.t0 + lo), (int64_t)0) + (t - cu[lo]);
  if (pos >= a.bt.cap) { pg_bad(a.bt); return -2; }
  const int64_t pg = pg_page(a.bt, lo, (int)(pos >> a.bt.shift));
  return pg < 0 ? -2 : (pg * a.n_kv + h) * a.page + (pos & (a.page - 1));
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
__device__ __forceinline__ void pc_copy(void* to, const void* from, int words) {
  for (int i = 0; i < words; ++i) ((uint4*)to)[i] = __ldg((const uint4*)from + i);
}

// GROUP threads a row (token, key head, k or v); READ: pages -> packed rows, else packed rows -> pages
template <typename T, int GROUP, bool READ>
__global__ void __launch_bounds__(PC_THREADS) paged_rows_kernel(PgRows a) {
  constexpr int W = 8;
  __shared__ int32_t scu[PC_SMEM_B + 1];
  const int32_t* cu = a.bt.cu;
  if (a.bt.B <= PC_SMEM_B) {
    for (int i = threadIdx.x; i <= a.bt.B; i += PC_THREADS) scu[i] = __ldg(a.bt.cu + i);
    __syncthreads();
    cu = scu;
  }
  const int64_t rows = (int64_t)a.bt.N * a.n_kv * 2, groups = (int64_t)gridDim.x * (PC_THREADS / GROUP);
  const int g = threadIdx.x % GROUP, d = g * W;
  const int64_t first = (int64_t)blockIdx.x * (PC_THREADS / GROUP) + threadIdx.x / GROUP;
  // (all threads of a warp take the same number of rounds: the maximum is found by shuffles)
  const int64_t rounds = (rows - (int64_t)blockIdx.x * (PC_THREADS / GROUP) + groups - 1) / groups;
  for (int64_t k = 0; k < rounds; ++k) {
    const int64_t row = first + k * groups;
    const bool in = row < rows;
    const int64_t th = in ? row >> 1 : 0, t = th / a.n_kv;
    const int h = (int)(th - t * a.n_kv), kv = in ? (int)(row & 1) : 0;
    const int64_t site = in ? pc_site(a, cu, t, h) : -1;
    const bool mine = site >= 0 && d < a.c;
    T* px = (T*)a.x[kv] + t * a.ld[kv] + (int64_t)h * a.c + d;
    float x[W] = {};
    if (READ) {
      if (in && d < a.c && (site == -2 || (site == -1 && a.zero_rest))) pc_store(px, x);
      if (!mine) continue;
      if (a.kind < KCH_FP8_E4M3) {
        pc_copy(px, (const T*)a.pages[kv] + site * a.c + d, sizeof(T) / 2);
        continue;
      }
      const float s = __ldg(a.scales[kv] + site);
      const uint8_t* p = (const uint8_t*)a.pages[kv] + site * a.c + d;
      const uint2 u = __ldg((const uint2*)p);
      const uint32_t w[2] = {u.x, u.y};
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const uint8_t code = (uint8_t)(w[e >> 2] >> (8 * (e & 3)));
        __nv_fp8_e4m3 v;
        v.__x = code;
        x[e] = (a.kind == KCH_FP8_E4M3 ? float(v) : (float)(int8_t)code) * s;
      }
      pc_store(px, x);
    } else {
      if (a.kind < KCH_FP8_E4M3) {
        if (mine) pc_copy((T*)a.pages[kv] + site * a.c + d, px, sizeof(T) / 2);
        continue;
      }
      if (mine) pc_load(px, x);
      uint32_t top = 0;                                  // as bits: a NaN is above an infinity, which is above every number
#pragma unroll
      for (int e = 0; e < W; ++e) top = max(top, __float_as_uint(x[e]) & 0x7FFFFFFFu);
#pragma unroll
      for (int o = GROUP / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (!mine) continue;
      const bool finite = top < 0x7F800000u;
      float s = top ? fmaxf(__uint_as_float(top) / (a.kind == KCH_FP8_E4M3 ? 448.f : 127.f), 1.17549435e-38f) : 1.f;
      const float inv = 1.f / s;
      uint32_t w[W / 4];
#pragma unroll
      for (int e = 0; e < W / 4; ++e)
        w[e] = finite ? pc_codes2(x[4 * e], x[4 * e + 1], s, inv, a.kind) | pc_codes2(x[4 * e + 2], x[4 * e + 3], s, inv, a.kind) << 16 : 0u;
      if (!finite) s = __uint_as_float(0x7FC00000u);     // a row that is not finite reads as NaN, whichever the kind
      uint8_t* p = (uint8_t*)a.pages[kv] + site * a.c + d;
      *(uint2*)p = make_uint2(w[0], w[1]);
      if (g == 0) a.scales[kv][site] = s;
    }
  }
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
  const int pieces = p->c / 8;
  const int64_t rows = b->N * p->n_kv * 2;
#define PC_GO(T_, G_)                                                                                                    \
  do {                                                                                                                   \
    const int64_t blocks = ceil_div64(rows, PC_THREADS / G_);                                                            \
    const unsigned grid = (unsigned)(blocks < 64 * KCH_SMS ? blocks : 64 * KCH_SMS);                                     \
    if (read) paged_rows_kernel<T_, G_, true><<<grid, PC_THREADS, 0, s>>>(a);                                            \
    else paged_rows_kernel<T_, G_, false><<<grid, PC_THREADS, 0, s>>>(a);                                                \
  } while (0)
#define PC_WIDTH(T_)                                                                                                     \
  do {                                                                                                                   \
    if (pieces <= 8) PC_GO(T_, 8);                                                                                       \
    else if (pieces <= 16) PC_GO(T_, 16);                                                                                \
    else PC_GO(T_, 32);                                                                                                  \
  } while (0)
  if (dtype == KCH_BF16) PC_WIDTH(bf16);
  else PC_WIDTH(float);
#undef PC_WIDTH
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
