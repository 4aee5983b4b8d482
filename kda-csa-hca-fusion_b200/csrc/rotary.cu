// Rotary positions: pairs of channels of queries and keys turned by an angle that grows with the token's position.
//
//   y_a = x_a cos t - x_b sin t,   y_b = x_b cos t + x_a sin t,   t = pos[token, axis(i)] * f_i   for pair i of r / 2,
//   (a, b) = (i, i + r / 2), or (2 i, 2 i + 1) where neighbours are paired;   channels r .. c - 1 stay;   inverse: -t.
//
// Angles in 64 bits: 32 would leave a position of 10^6 an angle that is off by 0.06.  f_i comes in turns, so that pos f_i less its nearest
// whole number is the angle's remainder, exact to 2^-53 of the product; sine and cosine of that in 32 bits (2^-24 of a turn), the
// rotation in 32 bits, one rounding.
//
// Bound by the bytes of x and y.  A block takes a few tokens: sines and cosines once a token and pair into shared memory, for all heads of
// queries and keys (each head's own would be 45 instructions a pair, more than the memory leaves time for), while the threads' first rows
// are under way; then 8 pairs a thread and row, in 16-byte words, two rows at a time.  Measured: 27 290 tokens of 16 and 8 heads of 128 in bf16,
// three axes, 53.6 us, 6.3 TB/s, 0.95 of the copy rate; 64 tokens 1.7 us in a run of such calls.  Where r is no multiple of 16 a thread has a pair, in accesses
// of 2 or 4 bytes: 9600 tokens of 16 and 4 heads of 64 in bf16 take 22 us with r = 24 and 30 with 40, 15 with 32 and 9 with 64 (fp32 26, 33, 23, 17).
#include "kch_common.cuh"

#define RO_THREADS 256
#define RO_TOKENS 16                   // of a block, at most
#define RO_PAIRS 128                   // of a head, at most

struct RoArgs {
  const void* x[2]; void* y[2];        // queries, keys
  int64_t ldx[2], ldy[2];              // elements between tokens
  const int32_t* pos; int64_t ld_pos;
  const double* turns;
  int64_t N;
  int nh, rows, c, pairs;              // rows: of both
  int ends[3];                         // of the axes before the last
  int tokens, width;                   // tokens of a block; log2 of the threads of a row
  uint32_t by_rows;                    // i / rows = i * by_rows >> 32 for i < tokens * rows, where both are above 1
  float sign;
};

template <typename T> struct RoVec;
template <> struct RoVec<bf16> {
  uint4 w;
  __device__ __forceinline__ void load(const bf16* p) { w = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(bf16* p) const { *reinterpret_cast<uint4*>(p) = w; }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) { x[2 * e] = __uint_as_float(u[e] << 16); x[2 * e + 1] = __uint_as_float(u[e] & 0xFFFF0000u); }
  }
  __device__ __forceinline__ void put(const float (&x)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
      u[e] = *reinterpret_cast<const uint32_t*>(&v);
    }
    w = make_uint4(u[0], u[1], u[2], u[3]);
  }
};
template <> struct RoVec<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) { a = *reinterpret_cast<const float4*>(p); b = *(reinterpret_cast<const float4*>(p) + 1); }
  __device__ __forceinline__ void store(float* p) const { *reinterpret_cast<float4*>(p) = a; *(reinterpret_cast<float4*>(p) + 1) = b; }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
  __device__ __forceinline__ void put(const float (&x)[8]) { a = make_float4(x[0], x[1], x[2], x[3]); b = make_float4(x[4], x[5], x[6], x[7]); }
};

// WORDS: r is a multiple of 16, and a thread's piece 8 pairs in two words of 8 channels; else a pair.  NEXT: neighbours are paired.
template <typename T, bool WORDS, bool NEXT>
__global__ void __launch_bounds__(RO_THREADS) rotary_kernel(const __grid_constant__ RoArgs a) {
  __shared__ alignas(16) float cosine[RO_TOKENS * RO_PAIRS], sine[RO_TOKENS * RO_PAIRS];
  constexpr int P = WORDS ? 8 : 1, FLIGHT = 2;           // pairs of a piece; rows in flight
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int tokens = (int)min((int64_t)a.tokens, a.N - t0), all = tokens * a.rows, step = RO_THREADS >> a.width;
  const int turned = a.pairs / P, pieces = turned + (a.c - 2 * a.pairs) / (WORDS ? 8 : 1);      // of a row: turned, and in all
  const int row0 = threadIdx.x >> a.width, lane = threadIdx.x & ((1 << a.width) - 1);
  struct Place { const T* x; T* y; int token; bool there; };
  auto place = [&](int i) {
    Place p;
    p.there = i < all;
    p.token = !p.there || a.tokens == 1 ? 0 : a.rows == 1 ? i : (int)__umulhi((uint32_t)i, a.by_rows);
    const int row = p.there ? i - p.token * a.rows : 0, k = row >= a.nh, head = row - (k ? a.nh : 0);
    p.x = (const T*)a.x[k] + (t0 + p.token) * a.ldx[k] + (int64_t)head * a.c;
    p.y = (T*)a.y[k] + (t0 + p.token) * a.ldy[k] + (int64_t)head * a.c;
    return p;
  };
  auto angles = [&] {
    for (int i = threadIdx.x; i < tokens * a.pairs; i += RO_THREADS) {
      const int token = i / a.pairs, pair = i - token * a.pairs;
      const int axis = (pair >= a.ends[0]) + (pair >= a.ends[1]) + (pair >= a.ends[2]);
      const double t = (double)__ldg(a.pos + (t0 + token) * a.ld_pos + axis) * __ldg(a.turns + pair);
      float s, c;
      sincospif(2.f * (float)(t - rint(t)), &s, &c);
      cosine[i] = c;
      sine[i] = s * a.sign;
    }
    __syncthreads();
  };
  if constexpr (WORDS) {
    const int first = NEXT ? 16 * lane : 8 * lane, second = first + (NEXT ? 8 : a.pairs);
    bool ready = false;
    for (int i0 = row0; i0 < all || !ready; i0 += FLIGHT * step) {
      Place p[FLIGHT];
      RoVec<T> u[FLIGHT], v[FLIGHT];
#pragma unroll
      for (int f = 0; f < FLIGHT; ++f) {
        p[f] = place(i0 + f * step);
        if (p[f].there && lane < turned) { u[f].load(p[f].x + first); v[f].load(p[f].x + second); }
      }
      if (!ready) { angles(); ready = true; }
      if (lane >= turned) continue;
#pragma unroll
      for (int f = 0; f < FLIGHT; ++f) {
        if (!p[f].there) break;
        float x[8], y[8], c[8], s[8], n[8], m[8];
        u[f].get(x);
        v[f].get(y);
        const int at = p[f].token * a.pairs + 8 * lane;
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          *reinterpret_cast<float4*>(c + e) = *reinterpret_cast<const float4*>(cosine + at + e);
          *reinterpret_cast<float4*>(s + e) = *reinterpret_cast<const float4*>(sine + at + e);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (NEXT) {                                    // pair e: channels 2 e, 2 e + 1 of the 16
            const float q = e < 4 ? x[2 * (e & 3)] : y[2 * (e & 3)], w = e < 4 ? x[2 * (e & 3) + 1] : y[2 * (e & 3) + 1];
            (e < 4 ? n : m)[2 * (e & 3)] = fmaf(q, c[e], -w * s[e]);
            (e < 4 ? n : m)[2 * (e & 3) + 1] = fmaf(w, c[e], q * s[e]);
          } else {
            n[e] = fmaf(x[e], c[e], -y[e] * s[e]);
            m[e] = fmaf(y[e], c[e], x[e] * s[e]);
          }
        }
        u[f].put(n);
        v[f].put(m);
        u[f].store(p[f].y + first);
        v[f].store(p[f].y + second);
      }
    }
    // what is not turned
    if (pieces > turned)
      for (int i = row0; i < all; i += step) {
        const Place p = place(i);
        if (p.x == p.y) continue;
        for (int w = lane; w < pieces - turned; w += 1 << a.width) {
          RoVec<T> u;
          u.load(p.x + 2 * a.pairs + 8 * w);
          u.store(p.y + 2 * a.pairs + 8 * w);
        }
      }
  } else {
    angles();
    for (int i = row0; i < all; i += step) {
      const Place p = place(i);
      for (int w = lane; w < pieces; w += 1 << a.width) {
        if (w < turned) {
          const int first = NEXT ? 2 * w : w, second = NEXT ? first + 1 : w + a.pairs;
          const float x = ldf(p.x + first), y = ldf(p.x + second), c = cosine[p.token * a.pairs + w], s = sine[p.token * a.pairs + w];
          stf(p.y + first, fmaf(x, c, -y * s));
          stf(p.y + second, fmaf(y, c, x * s));
        } else if (p.x != p.y) {
          p.y[a.pairs + w] = p.x[a.pairs + w];
        }
      }
    }
  }
}

// ---- host -------------------------------------------------------------------------------------------------------------------
// Do two column slices [N, width], tokens lda and ldb bytes apart, share a byte?  (Slices of one fused projection lie between one
// another's tokens.)
static bool ro_meet(const void* x, int64_t lda, int64_t wa, const void* y, int64_t ldb, int64_t wb, int64_t N) {
  const int64_t a = (int64_t)(uintptr_t)x, b = (int64_t)(uintptr_t)y;
  if (a >= b + (N - 1) * ldb + wb || b >= a + (N - 1) * lda + wa) return false;
  if (lda != ldb) return true;
  const int64_t d = ((b - a) % lda + lda) % lda;         // of b's columns behind a's
  return d < wa || lda - d < wb;
}

extern "C" int kch_rotary(const kch_rotary_args* p, void* stream) {
  KCH_REQUIRE(p != nullptr, "kch_rotary: null arguments");
  KCH_REQUIRE(p->dtype == KCH_F32 || p->dtype == KCH_BF16, "kch_rotary: unsupported dtype tag %d", p->dtype);
  KCH_REQUIRE(p->c >= 8 && p->c <= 256 && p->c % 8 == 0, "kch_rotary: c=%d must be a multiple of 8 from 8 to 256", p->c);
  KCH_REQUIRE(p->rotary_dim >= 2 && p->rotary_dim <= p->c && p->rotary_dim % 2 == 0, "kch_rotary: rotary_dim=%d must be even, from 2 to c=%d",
              p->rotary_dim, p->c);
  KCH_REQUIRE(p->nh >= 1 && p->n_kv >= 0 && (int64_t)p->nh + p->n_kv <= 65536, "kch_rotary: nh=%d, n_kv=%d", p->nh, p->n_kv);
  KCH_REQUIRE(p->axes >= 1 && p->axes <= 4, "kch_rotary: axes=%d must be from 1 to 4", p->axes);
  int sum = 0;
  for (int i = 0; i < p->axes; ++i) {
    KCH_REQUIRE(p->sections[i] >= 0 && p->sections[i] <= p->rotary_dim / 2, "kch_rotary: sections[%d]=%d", i, p->sections[i]);
    sum += p->sections[i];
  }
  KCH_REQUIRE(sum == p->rotary_dim / 2, "kch_rotary: sections of %d pairs, rotary_dim=%d has %d", sum, p->rotary_dim, p->rotary_dim / 2);
  KCH_REQUIRE(p->N >= 0 && p->N <= 0x7FFFFFFFLL, "kch_rotary: N=%lld rows out of range", (long long)p->N);
  if (p->N == 0) return KCH_OK;
  KCH_REQUIRE(p->positions && p->ld_positions >= p->axes && p->turns, "kch_rotary: null positions or turns, or positions %lld apart",
              (long long)p->ld_positions);
  const int es = p->dtype == KCH_BF16 ? 2 : 4;
  const int64_t wq = (int64_t)p->nh * p->c, wk = (int64_t)p->n_kv * p->c;
  KCH_REQUIRE(p->q && p->q_out && (p->n_kv == 0 || (p->k && p->k_out)), "kch_rotary: null q, k or an output");
  const struct { const void* x; int64_t ld, width; const char* name; } all[4] = {
      {p->q, p->ld_q, wq, "q"}, {p->q_out, p->ld_q_out, wq, "q_out"}, {p->k, p->ld_k, wk, "k"}, {p->k_out, p->ld_k_out, wk, "k_out"}};
  const int operands = p->n_kv ? 4 : 2;
  for (int i = 0; i < operands; ++i)
    KCH_REQUIRE(((uintptr_t)all[i].x & 15) == 0 && all[i].ld >= all[i].width && all[i].ld * es % 16 == 0,
                "kch_rotary: %s must be 16-byte aligned, its tokens (%lld elements) at least heads * c apart in multiples of 16 bytes", all[i].name,
                (long long)all[i].ld);
  for (int o = 1; o < operands; o += 2)                  // an output may be its own input; it meets nothing else
    for (int i = 0; i < operands; ++i) {
      if (i == o || (i == o - 1 && all[i].x == all[o].x && all[i].ld == all[o].ld)) continue;
      KCH_REQUIRE(!ro_meet(all[o].x, all[o].ld * es, all[o].width * es, all[i].x, all[i].ld * es, all[i].width * es, p->N),
                  "kch_rotary: %s overlaps %s", all[o].name, all[i].name);
    }
  RoArgs a = {};
  a.x[0] = p->q; a.x[1] = p->k; a.y[0] = p->q_out; a.y[1] = p->k_out;
  a.ldx[0] = p->ld_q; a.ldx[1] = p->ld_k; a.ldy[0] = p->ld_q_out; a.ldy[1] = p->ld_k_out;
  a.pos = p->positions; a.ld_pos = p->ld_positions; a.turns = p->turns;
  a.N = p->N; a.nh = p->nh; a.rows = p->nh + p->n_kv; a.c = p->c; a.pairs = p->rotary_dim / 2;
  for (int i = 0, end = 0; i < 3; ++i) {
    end += i + 1 < p->axes ? p->sections[i] : 0;
    a.ends[i] = i + 1 < p->axes ? end : 0x7FFFFFFF;
  }
  a.sign = p->inverse ? -1.f : 1.f;
  const bool words = p->rotary_dim % 16 == 0;
  const int lanes = words ? a.pairs / 8 : a.pairs;
  while ((1 << a.width) < lanes) ++a.width;
  // About 8 pieces a thread to a block, but two blocks to an SM where there are tokens for that.  Either side, us, bf16 heads of 128: 27 290 tokens of 24 heads 4 pieces
  // 52.4, 8 53.6, 16 54.7;  9600 of 20 heads 14.7, 17.1, 16.3;  4000 6.9, 8.1, 8.4;  one block an SM at least, two, eight: 4000 tokens 8.1, 8.1, 6.8;  1000
  // 3.8, 3.0, 3.8;  fp32, 8 heads of 64, 1000 tokens 2.8, 2.3, 3.6;  9600 8.9, 8.9, 7.9.
  const int64_t pieces = (int64_t)a.rows << a.width;
  int64_t tokens = 8 * RO_THREADS / pieces;
  if (tokens > p->N / (2 * KCH_SMS)) tokens = p->N / (2 * KCH_SMS);
  a.tokens = (int)(tokens < 1 ? 1 : tokens > RO_TOKENS ? RO_TOKENS : tokens);
  // (with more than one token a block there are 2^10 rows at most: i * rows < 2^32, so that the quotient is exact)
  a.by_rows = (uint32_t)(0x100000000ULL / (uint64_t)(a.rows > 1 ? a.rows : 2)) + 1;
  const dim3 grid((unsigned)ceil_div64(p->N, a.tokens));
  cudaStream_t s = kch_stream(stream);
  KCH_DISPATCH_FLOAT(p->dtype, T, {
    if (words && p->neighbours) rotary_kernel<T, true, true><<<grid, RO_THREADS, 0, s>>>(a);
    else if (words) rotary_kernel<T, true, false><<<grid, RO_THREADS, 0, s>>>(a);
    else if (p->neighbours) rotary_kernel<T, false, true><<<grid, RO_THREADS, 0, s>>>(a);
    else rotary_kernel<T, false, false><<<grid, RO_THREADS, 0, s>>>(a);
  });
  KCH_LAUNCH_OK();
  return KCH_OK;
}
