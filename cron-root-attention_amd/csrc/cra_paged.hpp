// The paged key/value cache as the kernels see it, and the geometry of a
// sequence's present length. Host-compilable: the index arithmetic is tested
// on the CPU.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/cra.h"

namespace cra {

// Row (page, head, offset) of a cache whose pages are [H_kv, page_size] rows:
// the index of the row in k, v, and of its norm and scales. 32 bits hold it
// (the ABI refuses caches of 2^31 rows); byte offsets take 64.
__host__ __device__ inline uint32_t cache_row(int page, int H_kv, int log_page, int h, int off) {
  return (((uint32_t)page * (uint32_t)H_kv + (uint32_t)h) << log_page) + (uint32_t)off;
}

constexpr uint32_t kNoRow = 0xffffffffu;  // of a page outside the cache

struct PagedView {
  const char* k;
  const char* v;
  const float* k_norm;
  const float* k_scale;
  const float* v_scale;
  const int32_t* table;  // [n_seqs, pages_per_seq], rows table_stride apart
  const int32_t* lens;   // [n_seqs]
  const int32_t* cu;     // [n_seqs + 1] first token of each sequence, or null
  int64_t table_stride;
  int num_pages, H_kv, log_page, n_seqs, pages_per_seq;
  int tokens, query_len;  // cu: rows of the packed tensors; else tokens per sequence
};

// Length of a sequence, within what its row of the table can hold (lengths
// live on the device and are not known when the launch is checked).
__host__ __device__ inline int seq_length(int len, int pages_per_seq, int log_page) {
  const int64_t most = (int64_t)pages_per_seq << log_page;
  const int cap = most < 0x7fffffff ? (int)most : 0x7fffffff;
  return len < 0 ? 0 : len < cap ? len : cap;
}

// Row that new token `t` of a sequence's `count` new ones is written to, or -1: before
// the first row (more new tokens than the length), or behind what the table's row
// holds. Counted back from the length as it is given: from one held within the table a
// sequence that outgrew it would overwrite its last rows.
__host__ __device__ inline int write_row(int len, int count, int t, int pages_per_seq, int log_page) {
  const int64_t row = (int64_t)len - count + t;
  return row >= 0 && row < seq_length(len, pages_per_seq, log_page) ? (int)row : -1;
}

// Tokens [first, last) of sequence b in the packed tensors; within them
// whatever cu holds.
struct TokenRange {
  int first, last;
};
__host__ __device__ inline TokenRange token_range(const int32_t* cu, int b, int tokens) {
  const int a = cu[b] < 0 ? 0 : cu[b] < tokens ? cu[b] : tokens;
  const int e = cu[b + 1] < a ? a : cu[b + 1] < tokens ? cu[b + 1] : tokens;
  return TokenRange{a, e};
}

// Sequence of packed token t: the last b with cu[b] <= t, or -1 for a token
// before the first or behind the last sequence. `lanes` offsets are looked at at
// a time: upto(first, step, n) counts those of cu[first + i step] <= t, i < lanes,
// i step < n (at least the first, whatever it answers).
template <typename F>
__host__ __device__ inline int seq_of_token(const int32_t* cu, int n_seqs, int t, int lanes, F upto) {
  int lo = 0, n = n_seqs;
  while (n > 1) {
    const int step = (n + lanes - 1) / lanes, c = upto(lo, step, n), skip = (c > 1 ? c - 1 : 0) * step;
    lo += skip;
    n = step < n - skip ? step : n - skip;
  }
  return t < cu[0] || t >= cu[n_seqs] ? -1 : lo;
}

// ceil(sqrt(n)), n >= 0: the float root is within one of it, squares of up to
// 46342 fit 32 bits.
__host__ __device__ inline int ceil_sqrt(int n) {
  if (n <= 0) return 0;
  uint32_t r = (uint32_t)sqrtf((float)n);
  r = r > 0 ? r - 1 : 0;
#pragma unroll
  for (int i = 0; i < 3; ++i) r += r * r < (uint32_t)n ? 1 : 0;
  return (int)r;
}

// The plan of a sequence of n tokens: window W (the rule, or the caller's,
// within the length), rows per block of the global rows.
struct SeqPlan {
  int n, W, rpb;
};
__host__ __device__ inline SeqPlan seq_plan(int n, int window, int relay, int top_k) {
  SeqPlan p;
  p.n = n;
  p.W = window > 0 ? (window < n ? window : n) : ceil_sqrt(n);
  if (p.W < 1) p.W = 1;
  p.rpb = (relay < 0 ? n > 2048 : relay != 0) ? 1 + top_k : 1;
  return p;
}

// Global rows that the query at position i sees: a prefix of this length.
__host__ __device__ inline int seq_prefix(int i, const SeqPlan& p) {
  const int ls = i - p.W + 1 > 0 ? i - p.W + 1 : 0;
  const int f = ls / p.W;
  return p.rpb * f + (ls != f * p.W ? 1 : 0);
}

// 32-key tiles of a sequence of n tokens, the last m of them new, that a row of
// few_kernel meets; key tiles of BN rows that a row tile of the chunk kernels,
// `span` new tokens wide, meets at most.
__host__ __device__ inline int few_tile_count(int n, int m, const SeqPlan& p) {
  const int pos0 = n - m > 0 ? n - m : 0, lo = pos0 - p.W + 1 > 0 ? pos0 - p.W + 1 : 0;
  return ((n > 0 ? seq_prefix(n - 1, p) : 0) + 31) / 32 + (n - lo + 31) / 32;
}
__host__ __device__ inline int chunk_tile_count(int n, int span, int BN, const SeqPlan& p) {
  const int64_t local = (int64_t)p.W + span;
  return ((n > 0 ? seq_prefix(n - 1, p) : 0) + BN - 1) / BN + (int)(((local < n ? local : n) + BN - 1) / BN) + 1;
}

// The most of these over all lengths up to max_len: windows and the numbers of
// blocks grow with the length.
struct PlanMost {
  int64_t globals;  // global rows
  int W, max_len, rpb;
};
inline PlanMost plan_most(int max_len, int window, int relay, int top_k) {
  const SeqPlan p = seq_plan(max_len, window, relay, top_k);
  const int64_t below = max_len > p.W ? max_len - p.W : 0;
  return PlanMost{(below + p.W - 1) / p.W * p.rpb, p.W, max_len, p.rpb};
}
inline int64_t few_tile_most(const PlanMost& m, int max_m) {
  const int64_t local = (int64_t)m.W + max_m - 1;
  return (m.globals + 31) / 32 + ((local < m.max_len ? local : m.max_len) + 31) / 32;
}
inline int64_t chunk_tile_most(const PlanMost& m, int span, int BN) {
  const int64_t local = (int64_t)m.W + span;
  return (m.globals + BN - 1) / BN + ((local < m.max_len ? local : m.max_len) + BN - 1) / BN + 1;
}

// Cache row of logical row `row` of a sequence whose table row is `pages`, or
// kNoRow if its page lies outside the cache.
__host__ __device__ inline uint32_t seq_row(const int32_t* pages, int row, int num_pages, int H_kv,
                                            int log_page, int h) {
  const int page = pages[row >> log_page];
  if ((uint32_t)page >= (uint32_t)num_pages) return kNoRow;
  return cache_row(page, H_kv, log_page, h, row & ((1 << log_page) - 1));
}

// Checks of the C ABI shared by its calls over a cache (CRA_OK or an error with
// its text set), and the view the kernels take.
int check_cache(const cra_cache* c);
int check_batch(const cra_cache* c, const cra_batch* b);
PagedView paged_view(const cra_cache* c, const cra_batch* b);

}  // namespace cra
