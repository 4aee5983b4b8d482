// What the kernels of the paged key / value cache share: where a token of a ragged batch lies, and how the attention over the
// pages is divided over the CTAs.
//
// Division.  An item is a block of at most R rows (consecutive (token, head of the group) pairs of one sequence, so that the
// heads which share a key head also share its tiles) against the key tiles that any of them sees.  The steps of all items
// form one line: sequence, key head, row block, step.  CTA i of C takes the steps [i, i + 1) * ceil(U / C), whatever items
// they belong to: a single long sequence is split along its keys, a batch of many short ones gives several items to a CTA, a
// causal chunk is balanced to one step, and the host needs no length (they stay on the device, so a captured graph replays
// with other ones).  An item that one CTA has whole is stored by it; the parts of the others go to the workspace (at most two
// a CTA: the item that its range ends in, and the one that it starts in the middle of) and are joined by a second kernel, in
// the order of the CTAs, so that the result does not depend on when they ran.
#pragma once
#include "kch_common.cuh"

#define PG_MAX_B 4096                  // sequences of a call: their table of steps is kept in shared memory
#define PG_LOG2E 1.4426950408889634f
#define PG_EXTRA 2                     // places of the line before an item's steps (see above) on tcgen05
#define PG_EXTRA_MOST 4                // of any form: what the host counts (pa_steps)
#define PG_ROWS 16                     // kind of keys and values that are packed rows like the queries, and not in pages (beside the KCH_ types)

unsigned int* kch_status_device_ptr();

struct PgBatch {
  const int32_t* table; int64_t ld_table;      // (of pages)
  const int32_t *t0, *cu;              // (t0: of pages)
  int B, N;                            // sequences; rows of the packed tensors
  int cap;                             // positions that a row of the table covers (below 2^31)
  int64_t num_pages;
  int shift;                           // log2(page_size)
  unsigned int* status;                // [0]: of expired waits, which ends the others; [1]: of tables, which ends none
  int n_kv, G, window;                 // key heads, query heads of one, window (attention only)
  uint32_t g_mul; int g_shift;         // n / G = n * g_mul >> 32 + g_shift for n < 2^31; g_mul 0: n >> g_shift
  // of an item, where the kernel leaves that open (ahead of the group's numbers, which it put on an odd word, it made ptxas spill 160 bytes in
  // steps of 16 and 32 rows over e4m3 pages, and fp32 chunks took 102.3 us for 100.5)
  int rows;
};
// With s = floor(log2 G) and M = floor(2^(32 + s) / G) + 1, M G exceeds 2^(32 + s) by at most G < 2^(s + 1): exact below 2^31.
static inline void pg_set_group(PgBatch& a, int G) {
  a.G = G;
  a.g_shift = 0;
  while ((2LL << a.g_shift) <= G) ++a.g_shift;
  a.g_mul = (G & (G - 1)) == 0 ? 0u : (uint32_t)((1ULL << (32 + a.g_shift)) / (uint32_t)G + 1);
}
__device__ __forceinline__ int pg_token(const PgBatch& a, int row) {          // row / G
  return a.g_mul ? (int)(__umulhi((uint32_t)row, a.g_mul) >> a.g_shift) : row >> a.g_shift;
}

struct PgSeq { int row0, len, t0, kv; };      // first packed row, new tokens, tokens before them, keys in all

// (Whatever cu_seqlens and t0 hold, rows stay inside the packed tensors and keys inside the table.)
// PACKED: keys and values are packed rows, and no sequence has earlier tokens.
template <bool PACKED = false>
__device__ __forceinline__ PgSeq pg_seq(const PgBatch& a, int b) {
  PgSeq s;
  s.row0 = min(max(__ldg(a.cu + b), 0), a.N);
  s.len = min(max(__ldg(a.cu + b + 1), s.row0), a.N) - s.row0;
  const int t0 = PACKED ? 0 : __ldg(a.t0 + b);
  s.t0 = max(t0, 0);
  s.kv = t0 < 0 ? 0 : (int)min((int64_t)t0 + s.len, (int64_t)a.cap);       // (positions before 0: no keys)
  return s;
}
__device__ __forceinline__ void pg_bad(const PgBatch& a) { atomicCAS(a.status + 1, 0u, (unsigned)KCH_STATUS_PAGED_TABLE); }
// page of `index` pages into sequence b, or -1 (and the status word) where the table holds none
__device__ __forceinline__ int pg_page(const PgBatch& a, int b, int index) {
  const int p = __ldg(a.table + b * a.ld_table + index);
  if (p >= 0 && p < a.num_pages) return p;
  pg_bad(a);
  return -1;
}

// One block of rows of a sequence: which keys its rows see together.
// tiles of KT keys from first_key (a multiple of KT) on; the keys before `lo` no row sees: their pages need not be there any more
struct PgSpan { int rows, lo, first_key, tiles, steps; };
// R rows a block (0: a.rows), KT keys a tile.  TWO: blocks of at most TWO rows (R 0: of half of them) take two tiles a step.
template <int R, int KT, int TWO>
__device__ __forceinline__ PgSpan pg_span(const PgBatch& a, const PgSeq& s, int block) {
  PgSpan x;
  const int all = R ? R : a.rows, two = R ? TWO : a.rows / 2;
  const int r0 = block * all, r1 = min(r0 + all, s.len * a.G);
  x.rows = r1 - r0;
  const int64_t first = (int64_t)s.t0 + pg_token(a, r0), last = (int64_t)s.t0 + pg_token(a, r1 - 1);      // positions of the first and the last query
  const int hi = (int)min(last + 1, (int64_t)s.kv);
  x.lo = a.window > 0 ? (int)min(max(first - a.window + 1, (int64_t)0), (int64_t)s.kv) : 0;
  x.first_key = x.lo / KT * KT;
  x.tiles = hi > x.first_key ? (hi - x.first_key + KT - 1) / KT : 0;
  x.steps = max(x.rows <= two ? (x.tiles + 1) / 2 : x.tiles, 1);            // (a row without keys is stored all the same)
  return x;
}
template <int R>
__device__ __forceinline__ int pg_blocks(const PgBatch& a, const PgSeq& s) {
  return R ? (s.len * a.G + R - 1) / (R ? R : 1) : (int)((unsigned)(s.len * a.G + a.rows - 1) / (unsigned)a.rows);
}
// the keys [x, y) that row `row` (token * G + head of the group) of a sequence sees
__device__ __forceinline__ int2 pg_sees(const PgBatch& a, const PgSeq& s, int row) {
  const int64_t pos = (int64_t)s.t0 + pg_token(a, row);
  return make_int2(a.window > 0 ? (int)min(max(pos - a.window + 1, (int64_t)0), (int64_t)s.kv) : 0, (int)min(pos + 1, (int64_t)s.kv));
}

// Where a CTA's range of steps begins.  (Steps are counted in 32 bits: the host refuses a call that could have 2^31 - 1.)
struct PgPlace {
  int per, left;                       // places of the line of a CTA; of this one
  int b, h, block, step;               // step: place in the item (its steps come behind EXTRA others)
  PgSeq s;                             // of b
  PgSpan x;                            // of the block
};

// steps of sequence b (0 behind the last) for each key head: by the lane where it is one block, as in a batch of single tokens, else
// by the warp over its blocks
template <int R, int KT, int TWO, int EXTRA>
__device__ __forceinline__ int pg_steps(const PgBatch& a, const PgSeq& s) {
  const int lane = threadIdx.x & 31, blocks = pg_blocks<R>(a, s);
  int mine = blocks == 1 ? pg_span<R, KT, TWO>(a, s, 0).steps + EXTRA : 0;
  for (unsigned many = __ballot_sync(0xffffffffu, blocks > 1); many; many &= many - 1) {
    const int from = __ffs(many) - 1;
    PgSeq t;
    t.row0 = 0;
    t.len = __shfl_sync(0xffffffffu, s.len, from);
    t.t0 = __shfl_sync(0xffffffffu, s.t0, from);
    t.kv = __shfl_sync(0xffffffffu, s.kv, from);
    const int nb = pg_blocks<R>(a, t);
    int sum = 0;
#pragma unroll 1
    for (int i = lane; i < nb; i += 32) sum += pg_span<R, KT, TWO>(a, t, i).steps + EXTRA;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == from) mine = sum;
  }
  return mine * a.n_kv;
}
template <bool PACKED>
__device__ __forceinline__ PgSeq pg_seq_or_none(const PgBatch& a, int b) {
  PgSeq s = {0, 0, 0, 0};
  if (b < a.B) {
    s = pg_seq<PACKED>(a, b);
    if (s.len > 0 && s.kv - s.t0 < s.len) pg_bad(a);        // it begins before position 0, or the table ends before it does (without new tokens it needs no page)
  }
  return s;
}
#define PG_MOST 0x7FFFFFFF
__device__ __forceinline__ int pg_sum(int x, int y) { return (int)min((unsigned)x + (unsigned)y, (unsigned)PG_MOST); }      // (of what is not negative)
__device__ __forceinline__ int pg_scan(int x) {             // sums over the lanes up to this one
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if ((threadIdx.x & 31) >= o) x = pg_sum(x, y);
  }
  return x;
}

// The whole block calls it; `mem`: PG_PLAN_BYTES(B) of shared memory, free again after the next __syncthreads().
#define PG_PLAN_BYTES(B) (32 + 4 * ((B) + 1))
template <int R, int KT, int TWO, int EXTRA = 0, bool PACKED = false>
__device__ __forceinline__ PgPlace pg_plan(const PgBatch& a, void* mem, int cta, int ctas) {
  static_assert(EXTRA <= PG_EXTRA_MOST, "the host's bound on the places of a call counts fewer");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  PgPlace p = {};
  int total, before = 0, mine = 0;                          // steps: of all, before sequence p.b, of it
  auto range = [&] {
    // The host has counted a row once.  Where cu_seqlens falls and rises again a row is of several sequences, and there may be more
    // steps than are counted: such a call does nothing.
    if (total == PG_MOST) {
      pg_bad(a);
      total = 0;
    }
    p.per = max((int)(((unsigned)total + (unsigned)ctas - 1u) / (unsigned)ctas), 1);
    const int64_t start = (int64_t)p.per * cta;
    p.left = (int)max(min((int64_t)p.per, total - start), (int64_t)0);
    return p.left > 0 ? (int)start : 0x7FFFFFFF;
  };
  int start;
  const bool one = (int64_t)a.N * a.G <= (int64_t)(R ? R : a.rows) * a.B;       // a block a sequence, on average
  // Few sequences: every warp by itself, without memory and barriers.  This / through memory, us, chunks over bf16 pages, prompts, chunks over e4m3 pages, 16 heads of
  // 128 on 4, about 6000 tokens in all: 2 sequences 154.0 / 154.5, 77.2 / 77.0, 214.7 / 216.1;  4: 119.4 / 119.6, 51.0 / 50.4, 157.6 / 158.0;  8: 104.7 / 104.1,
  // 42.6 / 40.5, 138.4 / 137.6;  16: 101.2 / 98.8, 39.1 / 34.9, 129.9 / 127.0;  32: 107.3 / 101.4, 37.8 / 28.9, 135.7 / 128.5.
  if (a.B <= 4 || (a.B <= 32 && one)) {
    const PgSeq s = pg_seq_or_none<PACKED>(a, lane);
    const int x = pg_steps<R, KT, TWO, EXTRA>(a, s), upto = pg_scan(x);
    total = __shfl_sync(0xffffffffu, upto, 31);
    start = range();
    if (p.left > 0) {
      p.b = __ffs(__ballot_sync(0xffffffffu, upto > start)) - 1;
      mine = __shfl_sync(0xffffffffu, x, p.b);
      before = __shfl_sync(0xffffffffu, upto, p.b) - mine;
      p.s.row0 = __shfl_sync(0xffffffffu, s.row0, p.b);
      p.s.len = __shfl_sync(0xffffffffu, s.len, p.b);
      p.s.t0 = __shfl_sync(0xffffffffu, s.t0, p.b);
      p.s.kv = __shfl_sync(0xffffffffu, s.kv, p.b);
    }
  } else {
    int* base = reinterpret_cast<int*>(mem);                // [B + 1] steps before sequence b
    int* found = base + a.B + 1;
    // (Sequences of several blocks are dealt out over the warps: one that has 32 of them takes 10 000 clocks.  Of a block each, a lane has one, and few
    // warps are sooner done: steps of 64 sequences 37.2 us, dealt out 37.8; 8-bit pages, 16 heads of 128 on 1.)
    const int deal = one ? 32 : min((a.B + warps - 1) / warps, 32);
#pragma unroll 1
    for (int b0 = warp * deal; b0 < a.B; b0 += warps * deal) {
      const int x = pg_steps<R, KT, TWO, EXTRA>(a, pg_seq_or_none<PACKED>(a, lane < deal ? b0 + lane : a.B));
      if (lane < deal && b0 + lane < a.B) base[b0 + lane + 1] = x;
    }
    if (tid == 0) base[0] = 0;
    __syncthreads();
    if (warp == 0) {
      int run = 0;
#pragma unroll 1
      for (int b0 = 0; b0 < a.B; b0 += 32) {
        const int x = pg_sum(run, pg_scan(b0 + lane < a.B ? base[b0 + lane + 1] : 0));
        if (b0 + lane < a.B) base[b0 + lane + 1] = x;
        run = __shfl_sync(0xffffffffu, x, 31);
      }
    }
    __syncthreads();
    total = base[a.B];
    start = range();
    if (p.left > 0)
      for (int b = tid; b < a.B; b += blockDim.x)
        if (base[b] <= start && start < base[b + 1]) found[0] = b;
    __syncthreads();
    if (p.left > 0) {
      p.b = found[0];
      before = base[p.b];
      mine = base[p.b + 1] - before;
      p.s = pg_seq<PACKED>(a, p.b);
    }
  }
  if (p.left > 0) {                    // the key head, then the block, by every warp
    const int blocks = pg_blocks<R>(a, p.s);
    int rest = start - before;
    if (a.n_kv > 1) {
      const unsigned head = (unsigned)mine / (unsigned)a.n_kv;
      p.h = (int)((unsigned)rest / head);
      rest -= p.h * (int)head;
    }
    if (blocks > 1) {
#pragma unroll 1
      for (int i0 = 0; i0 < blocks; i0 += 32) {
        const int i = i0 + lane, n = i < blocks ? pg_span<R, KT, TWO>(a, p.s, i).steps + EXTRA : 0, x = pg_scan(n);
        const unsigned hit = __ballot_sync(0xffffffffu, i < blocks && x > rest);
        if (hit) {
          const int at = __ffs(hit) - 1;
          p.block = i0 + at;
          rest -= __shfl_sync(0xffffffffu, x - n, at);
          break;
        }
        rest -= __shfl_sync(0xffffffffu, x, 31);
      }
    }
    p.step = rest;
    p.x = pg_span<R, KT, TWO>(a, p.s, p.block);
  }
  return p;
}

// The items of a CTA, one after the other; every role of a kernel walks them by itself.
template <int R, int KT, int TWO, int EXTRA = 0, bool PACKED = false>
struct PgWalk {
  const PgBatch& a;
  int b, h, block;                     // the item
  int first, count;                    // its steps that belong to this CTA
  PgSeq s;
  PgSpan x;
  int left;                            // places of the CTA's range behind them
  int from, taken;                     // places of the item that are in it
  __device__ __forceinline__ PgWalk(const PgBatch& a_, const PgPlace& p)
      : a(a_), b(p.b), h(p.h), block(p.block), first(p.step), count(0), s(p.s), x(p.x), left(p.left), from(p.step), taken(0) {
    if (left > 0) take();
  }
  __device__ __forceinline__ bool valid() const { return count > 0; }      // (a range that ends before an item's first step has no more of it)
  __device__ __forceinline__ bool starts() const { return first == 0; }
  __device__ __forceinline__ bool ends() const { return first + count == x.steps; }
  // the CTA that has the end of an item which starts in this one's range and is its last
  __device__ __forceinline__ int last(const PgPlace& p, int cta) const {
    return (int)(((int64_t)p.per * cta + (p.left - (EXTRA ? taken : count)) - (EXTRA ? from : 0) + EXTRA + x.steps - 1) / p.per);
  }
  __device__ __forceinline__ void next() {
    if (EXTRA) from = 0; else first = 0;
    count = 0;
    if (left <= 0) return;
    if (++block == pg_blocks<R>(a, s)) {
      block = 0;
      if (++h == a.n_kv) {
        h = 0;
        do { s = pg_seq<PACKED>(a, ++b); } while (s.len == 0);       // (places are left, so a sequence with rows follows)
      }
    }
    x = pg_span<R, KT, TWO>(a, s, block);
    take();
  }

 private:
  __device__ __forceinline__ void take() {
    if constexpr (EXTRA == 0) {
      count = min(x.steps - first, left);
      left -= count;
    } else {
      taken = min(x.steps + EXTRA - from, left);
      left -= taken;
      first = max(from - EXTRA, 0);
      count = max(from + taken - EXTRA, 0) - first;
    }
  }
};

// Parts of items in the workspace: one record a CTA (the item that starts in its range and ends in another's), then two slots
// a CTA of R rows (or what rows the call has, where these are fewer): c sums a row, the rows' maxima (base 2), their sums.
struct PgRecord { int valid, b, h, block, last, rows, row0; };       // last: the CTA that has the item's end
__host__ __device__ __forceinline__ int64_t pg_slot_floats(int R, int c) { return (int64_t)R * (c + 2); }
__host__ __device__ __forceinline__ int64_t pg_records_bytes(int ctas) { return ((int64_t)ctas * (int64_t)sizeof(PgRecord) + 255) / 256 * 256; }
static inline int64_t pg_workspace_bytes(int ctas, int R, int c) { return pg_records_bytes(ctas) + 2 * ctas * pg_slot_floats(R, c) * 4; }

struct PgJoinArgs {
  void* out; int dtype;                // [N, nh, c]
  int nh, G, c, R, slot_rows;          // R: rows of an item
  const void* sink; int sink_dtype;
  const PgRecord* records; const float* slots;
};
int kch_paged_join(const PgJoinArgs& a, int ctas, cudaStream_t s);

struct PgAttend {                      // what both attention kernels get
  PgBatch bt;
  const void *q, *k, *v, *ks, *vs;      // (ks, vs: scales; float, in 4 bits bf16)
  void* out;
  int64_t ld_q, ld_k, ld_v;             // (ld_k, ld_v: of packed rows)
  int c, page, zero_rest, slot_rows, q_map;      // q_map: queries are fetched by a tensor map
  float scale;                         // times log2(e)
  const void* sink; int sink_dtype;
  PgRecord* records; float* slots;
};

// rows behind the last sequence (and before the first), where the caller wants zeros there
__device__ __forceinline__ void pg_zero_rest(const PgAttend& a, int es, int cta, int ctas) {
  if (!a.zero_rest) return;
  const int64_t lo = min(max(__ldg(a.bt.cu), 0), a.bt.N), hi = min(max(__ldg(a.bt.cu + a.bt.B), (int)lo), a.bt.N);
  if (lo == 0 && hi == a.bt.N) return;
  const int64_t row = (int64_t)a.bt.n_kv * a.bt.G * a.c * es / 16, words = (lo + a.bt.N - hi) * row;      // 16-byte words of a token
  for (int64_t i = (int64_t)cta * blockDim.x + threadIdx.x; i < words; i += (int64_t)ctas * blockDim.x) {
    const int64_t t = i / row, at = (t < lo ? t : hi + t - lo) * row + i % row;
    reinterpret_cast<uint4*>(a.out)[at] = make_uint4(0u, 0u, 0u, 0u);
  }
}
