// Attention of new tokens over a paged key/value cache (serving), with the C
// ABI front end. The new tokens of a sequence are its last m; query i of a
// sequence of n tokens sees what it sees in the attention of the whole
// sequence: its window of W tokens, the first row of every earlier W-block and
// (relay) the top_k rows of largest norm of every W-block that ends before the
// window, all under one softmax:
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i.k_j - max_j)
// over the multiset of rows j; W = ceil(sqrt(n)), or the caller's (W >= n: plain
// causal attention). Lengths, page tables and the plan's window are read and
// formed on the device, so a captured call serves growing sequences.
//
// Launches: select_kernel ranks the stored norms and lists the cache rows of
// the global rows (sequences with relay only); few_kernel takes the sequences
// whose rows (new tokens x query heads of a kv head) fit one 16-row MFMA block,
// their keys cut into pieces of equal length, joined by combine_kernel;
// chunk_kernel takes the others in tiles of 128 rows, the rows of a kv head's
// query heads side by side so that a K/V tile serves them all. fp32 runs
// f32_kernel for both.
//
// A row that a query does not see never reaches its result, whatever it holds
// (NaN and infinity included): masked scores are replaced, and where a tile that
// not every query sees holds such values P.V is formed apart from them
// (pv_not_finite). What a seen row of V holds reaches the query however small its
// weight: an infinity times a weight that is 0 is found in the result, and the tiles
// are gone through once more. A query that sees no row gives zeros.
#include <stdio.h>

#include <algorithm>
#include <type_traits>

#include "cra_common.hpp"
#include "cra_internal.hpp"
#include "cra_paged_dev.hpp"
#include "cra_paged_few.hpp"

namespace cra {

int set_error(int code, const char* msg);

namespace {

// ---------------------------------------------------------------------------
// The global rows of sequences with relay, as cache rows: of each W-block its
// first row, and behind it (blocks that end before the last query's window) the
// top_k rows of largest norm, of equals the earlier; a slot without a row left
// is the block's first row, as in the packed rows of whole sequences. NaN norms
// are never chosen.
//
// A lane loads the norms of eight rows with one page lookup; a block of up to 121,
// 249 or 505 rows (at any alignment) takes 16, 32 or 64 lanes, so a wave picks in
// four, two or one blocks at a time: the largest norm of a lane, then of its group, by
// exchanges in the VALU; the lane that holds a pick stores its cache row. Bound by
// that VALU work (and below a few thousand blocks by the latency of page table and
// norm loads, the next blocks' of which are on their way). Wider blocks go to
// select_wide_kernel, which carries rows along with norms, 64 rows at a time.
// Measured, 8 heads: 16 sequences of 700-131072 tokens 14.5 us (select_wide_kernel
// 23.4; a block a wave, picks found by the whole wave, 16.6), 64 of up to 32768 tokens
// 7.1 us (15.5; 11.4); 34000 blocks of 31 rows 12.5 us (a block a wave 34).
// ---------------------------------------------------------------------------
constexpr int kSelWaves = 4, kSelLoads = 8;
constexpr int kSelMost = 64 * 8 - 7;   // rows of a block in select_kernel, at any alignment

// The blocks of a wave: [first, end) of sequence b's, head h.
struct SelWork {
  SeqPlan p;
  int b, h, full, first, end;
  uint32_t* out;
  const int32_t* pages;
};
// A wave takes a multiple of `at_once(W)` blocks.
template <typename F>
__device__ __forceinline__ SelWork sel_work(const PagedArgs& a, int steps, F at_once) {
  SelWork k{};
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t bh = div_by(blockIdx.x, a.d_steps);  // workgroups a (sequence, head)
  const uint32_t own = (uint32_t)a.c.n_seqs * a.c.H_kv;
  int step = (int)(blockIdx.x - bh * steps);
  if (bh >= own) {  // the shared prefix has steps of its own
    const int i = (int)(blockIdx.x - own * steps);
    steps = (int)(gridDim.x - own * steps) / a.c.H_kv;
    bh = own + i / steps;
    step = i % steps;
  }
  const int nw = steps * kSelWaves, w = step * kSelWaves + wave;
  k.b = (int)div_by(bh, a.d_hkv);
  k.h = (int)(bh - (uint32_t)k.b * a.c.H_kv);
  int ls, skip = 0;  // blocks of rows below ls, but for the first ones
  if (k.b < a.c.n_seqs) {
    const Seq s = wave_seq(a, k.b);
    k.p = get_plan(a, s.n);
    if (k.p.rpb == 1 || s.m < 1) return k;
    ls = s.n - k.p.W > 0 ? s.n - k.p.W : 0;  // window start of the last query
    k.out = a.list + (int64_t)bh * a.list_cap;
    k.pages = a.c.table + k.b * a.c.table_stride;
    if (a.plen) skip = share_of(a, prefix_plan(a), s, k.p).P / k.p.W;
  } else {  // the shared prefix
    k.p = prefix_plan(a);
    if (k.p.rpb == 1 || k.p.n < 1) return k;
    ls = k.p.n;
    k.out = a.plist + (int64_t)k.h * a.plist_cap;
    k.pages = a.ptable;
  }
  k.full = ls / k.p.W;
  const int blocks = k.full + (ls != k.full * k.p.W ? 1 : 0), n = at_once(k.p.W);
  const int per = ((max(blocks - skip, 0) + nw - 1) / nw + n - 1) / n * n;
  k.first = skip + w * per;
  k.end = min(blocks, k.first + per);
  return k;
}

// Maximum over the lane's group of G lanes, in all of them.
template <int G>
__device__ __forceinline__ int lanes_max(int x) {
  auto with = [&](uint32_t o) { x = max(x, (int)o); };
  if constexpr (G == 64) {
    const auto r = __builtin_amdgcn_permlane32_swap((uint32_t)x, (uint32_t)x, false, false);
    x = max((int)r[0], (int)r[1]);
  }
  if constexpr (G >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap((uint32_t)x, (uint32_t)x, false, false);
    x = max((int)r[0], (int)r[1]);
  }
  with(from_lane_xor<8>((uint32_t)x));
  with(from_lane_xor<4>((uint32_t)x));
  with(from_lane_xor<2>((uint32_t)x));
  with(from_lane_xor<1>((uint32_t)x));
  return x;
}

// The wave's blocks, 64 / G at a time.
template <int G>
__device__ __forceinline__ void select_blocks(const PagedArgs& a, const SelWork& w) {
  constexpr int P = 64 / G;
  const int lane = threadIdx.x & 63, l = lane & (G - 1), grp = lane / G;
  const uint64_t mine = (G == 64 ? ~0ull : (1ull << (G & 63)) - 1) << (lane & ~(G - 1));  // the group's lanes
  const uint64_t below = mine & ((1ull << lane) - 1);
  const int W = w.p.W;
  const int32_t* pages = w.pages;
  // cache row of logical row 8 (first row / 8 + l): eight rows of one page; lanes
  // behind the last eight (of the block, or of the sequence) repeat it
  auto load_row = [&](int blk) -> uint32_t {
    if (blk >= w.end) return 0u;
    const int last = min(blk * W + W - 1, w.p.n - 1);
    return seq_row(pages, min((blk * W & ~7) + 8 * l, last & ~7), a.c.num_pages, a.c.H_kv,
                   a.c.log_page, w.h);
  };
  struct Eight {
    float4 lo, hi;
  };
  auto load_norms = [&](int blk, uint32_t at) -> Eight {
    if (blk >= w.end) return Eight{};
    const float4* p = reinterpret_cast<const float4*>(a.c.k_norm + (at == kNoRow ? 0u : at));
    return Eight{p[0], p[1]};
  };
  int blk = w.first + grp;
  uint32_t at = load_row(blk), at1 = load_row(blk + P);
  Eight x = load_norms(blk, at);
  for (int base = w.first; base < w.end; base += P, blk += P) {
    const Eight x1 = load_norms(blk + P, at1);
    const uint32_t at2 = load_row(blk + 2 * P);
    const int lead = blk * W & 7;
    const bool full = blk < w.full;
    uint32_t* out = w.out + (int64_t)w.p.rpb * blk;
    const uint32_t head = at == kNoRow ? kNoRow : at + lead;  // lane 0 of the group: the block's first row
    if (blk < w.end && l == 0) out[0] = head;
    const bool bad = (__ballot(at == kNoRow) & mine) != 0;
    // a norm's bits, which order as the norms do; negative: not a row of a whole
    // block, or NaN
    int key[8], top = -1;
    const float f[8] = {x.lo.x, x.lo.y, x.lo.z, x.lo.w, x.hi.x, x.hi.y, x.hi.z, x.hi.w};
    const uint32_t rows = full ? W : 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool in = (uint32_t)(8 * l + j - lead) < rows;
      key[j] = in ? __float_as_int(fmaxf(f[j], -1.f)) : -1;
      top = max(top, key[j]);
    }
    for (int j = 0; j < a.top_k; ++j) {
      const int m = lanes_max<G>(top);
      const bool has = m >= 0 && top == m;
      const bool pick = has && (__ballot(has) & below) == 0;  // lanes rise with their rows
      if (pick) {
        int e = 7;
#pragma unroll
        for (int i = 6; i >= 0; --i) e = key[i] == m ? i : e;
        out[1 + j] = bad ? kNoRow : at + e;
        top = -1;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          key[i] = i == e ? -1 : key[i];
          top = max(top, key[i]);
        }
      }
      if (full && m < 0 && l == 0) out[1 + j] = bad ? kNoRow : head;  // no row is left
    }
    at = at1, at1 = at2, x = x1;
  }
}

__global__ __launch_bounds__(64 * kSelWaves) void select_kernel(int steps, PagedArgs a) {
  const SelWork w = sel_work(a, steps, [](int W) { return W <= 121 ? 4 : W <= 249 ? 2 : 1; });
  if (w.first >= w.end) return;
  if (w.p.W <= 121)
    select_blocks<16>(a, w);
  else if (w.p.W <= 249)
    select_blocks<32>(a, w);
  else
    select_blocks<64>(a, w);
}

template <int KEEP>
__global__ __launch_bounds__(64 * kSelWaves) void select_wide_kernel(int steps, PagedArgs a) {
  const int lane = threadIdx.x & 63;
  const SelWork w = sel_work(a, steps, [](int) { return 1; });
  if (w.first >= w.end) return;
  const SeqPlan p = w.p;
  const int full = w.full, first = w.first, end = w.end;
  const int32_t* pages = w.pages;
  auto row_at = [&](int row) {
    return seq_row(pages, row, a.c.num_pages, a.c.H_kv, a.c.log_page, w.h);
  };
  constexpr int kPiece = 64 * kSelLoads;
  auto load_rows = [&](int blk, int base, uint32_t (&at)[kSelLoads]) {
#pragma unroll
    for (int u = 0; u < kSelLoads; ++u)
      at[u] = blk < min(end, full) && base + 64 * u < p.W  // whole wave
                  ? row_at(blk * p.W + min(base + 64 * u + lane, p.W - 1))
                  : 0u;
  };
  auto load_norms = [&](int blk, int base, const uint32_t (&at)[kSelLoads], float (&x)[kSelLoads]) {
#pragma unroll
    for (int u = 0; u < kSelLoads; ++u)
      x[u] = blk < min(end, full) && base + 64 * u < p.W && at[u] != kNoRow ? a.c.k_norm[at[u]] : -1.f;
  };
  auto advance = [&](int& blk, int& base) {
    base += kPiece;
    if (base >= p.W || blk >= full) ++blk, base = 0;
  };
  uint32_t at[kSelLoads], at2[kSelLoads];
  float x[kSelLoads];
  int blk = first, base = 0, blk1 = first, base1 = 0;
  load_rows(blk, base, at);
  load_norms(blk, base, at, x);
  advance(blk1, base1);
  load_rows(blk1, base1, at2);
  uint32_t key[KEEP];  // norm's bits + 1, falling; 0: none
  int row[KEEP];
  bool bad = false;
#pragma unroll
  for (int j = 0; j < KEEP; ++j) key[j] = 0, row[j] = 0;
  while (blk < end) {
    float xn[kSelLoads];
    uint32_t atn[kSelLoads];
    int blk2 = blk1, base2 = base1;
    load_norms(blk1, base1, at2, xn);
    advance(blk2, base2);
    load_rows(blk2, base2, atn);
#pragma unroll
    for (int u = 0; u < kSelLoads; ++u) {
      if (base + 64 * u >= p.W) break;  // whole wave
      const int i = base + 64 * u + lane;
      bad |= at[u] == kNoRow;
      uint32_t k = i < p.W && x[u] >= 0.f ? __float_as_uint(x[u]) + 1 : 0u;
      int ri = i;
#pragma unroll
      for (int j = 0; j < KEEP; ++j) {  // rows rise: of equals the earlier stays
        const bool up = k > key[j];
        const uint32_t ok = key[j];
        const int orow = row[j];
        key[j] = up ? k : ok;
        row[j] = up ? ri : orow;
        k = up ? ok : k;
        ri = up ? orow : ri;
      }
    }
    if (base + kPiece >= p.W || blk >= full) {  // the block is complete
      const bool any_bad = __any(bad);
      int mine = 0;  // lane e: entry e of the block
      for (int j = 0; j < a.top_k; ++j) {
        const uint32_t m = wave_max(key[0]);
        int pick = 0;
        if (m) {
          uint64_t eq = __ballot(key[0] == m);
          int l = __builtin_ctzll(eq);
          pick = __builtin_amdgcn_readlane(row[0], l);
          for (eq &= eq - 1; eq; eq &= eq - 1) {  // equal norms: the earliest row
            const int l2 = __builtin_ctzll(eq);
            const int other = __builtin_amdgcn_readlane(row[0], l2);
            if (other < pick) pick = other, l = l2;
          }
          if (lane == l) {
#pragma unroll
            for (int i = 0; i + 1 < KEEP; ++i) key[i] = key[i + 1], row[i] = row[i + 1];
            key[KEEP - 1] = 0;
          }
        }
        if (lane == 1 + j) mine = any_bad ? -1 : pick;
      }
      if (lane < (blk < full ? p.rpb : 1))
        w.out[(int64_t)p.rpb * blk + lane] = mine < 0 ? kNoRow : row_at(blk * p.W + mine);
      bad = false;
#pragma unroll
      for (int j = 0; j < KEEP; ++j) key[j] = 0, row[j] = 0;
    }
#pragma unroll
    for (int u = 0; u < kSelLoads; ++u) at[u] = at2[u], at2[u] = atn[u], x[u] = xn[u];
    blk = blk1, base = base1;
    blk1 = blk2, base1 = base2;
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
int err(int code, const char* msg) { return set_error(code, msg); }

int hip_err(hipError_t e, const char* where) {
  if (e == hipSuccess) return CRA_OK;
  char msg[256];
  snprintf(msg, sizeof(msg), "%s: %s", where, hipGetErrorString(e));
  return err(CRA_E_HIP, msg);
}

// What a call launches, from sizes the host knows; the lengths themselves are
// on the device.
struct Launch {
  int grp, max_len, Dp;
  bool few, chunk;
  bool list, wide;        // relay rows are listed; blocks too wide for select_kernel
  int64_t list_cap;
  int sel_steps;          // select workgroups a (sequence, head)
  int64_t prefix_steps;   // and of a head of the shared prefix
  int part_rows, few_grid;
  bool join;              // a sequence's keys may be cut into pieces
  int64_t items, joins;   // chunk pieces and row tiles of cut sequences, over all kv heads, at most
  int64_t parts;          // pieces of cut sequences that the workspace holds
  size_t list_bytes, part_bytes, ml_bytes, piece_bytes;
  bool shared;            // a prefix is given, and sequences may share it
  int64_t plist_cap;
  int prefix_grid, prefix_rows, prefix_most;
  size_t plist_bytes, ppart_bytes, pml_bytes, pinfo_bytes;
  size_t own_bytes() const { return list_bytes + part_bytes + ml_bytes + piece_bytes; }
  size_t bytes() const { return own_bytes() + plist_bytes + ppart_bytes + pml_bytes + pinfo_bytes; }
};

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

int check_paged(const cra_cache* c, const cra_batch* b, const cra_paged_plan* p) {
  if (int e = check_cache(c)) return e;
  if (int e = check_batch(c, b)) return e;
  if (!p) return err(CRA_E_INVALID, "plan is NULL");
  if (p->H_q < 1 || p->H_q % c->H_kv) return err(CRA_E_INVALID, "H_q must be a multiple of H_kv");
  if (p->D < 8 || p->D > c->D || p->D % 8)
    return err(CRA_E_INVALID, "D must be a multiple of 8 up to the cache's row width");
  if (p->window < 0) return err(CRA_E_INVALID, "window must be >= 0 (0: the rule)");
  if (p->relay < -1 || p->relay > 1) return err(CRA_E_INVALID, "relay must be -1 (the rule), 0 or 1");
  if (p->relay != 0 && (p->top_k < 1 || p->top_k > 4)) return err(CRA_E_INVALID, "top_k outside [1, 4]");
  if (!(p->scale > 0.f)) return err(CRA_E_INVALID, "scale must be > 0");
  if (p->max_seqlen < 1) return err(CRA_E_INVALID, "max_seqlen must be >= 1");
  if (b->cu_seqlens && p->max_query_len < 1) return err(CRA_E_INVALID, "max_query_len must be >= 1");
  const int64_t tokens = b->cu_seqlens ? b->tokens : (int64_t)b->n_seqs * b->query_len;
  if (tokens * (p->H_q / c->H_kv) >= (int64_t)1 << 30)
    return err(CRA_E_INVALID, "2^30 query rows of a kv head or more");
  // sums of 64 sequences' tiles take 32 bits
  const int64_t held = (int64_t)b->pages_per_seq * c->page_size;
  const int most = (int)std::min<int64_t>(p->max_seqlen, std::min<int64_t>(held, 0x7fffffff));
  if (most > 0x7fff0000)  // row numbers behind the last tile stay within 32 bits
    return err(CRA_E_INVALID, "sequences of 2^31 - 2^16 tokens or more");
  const PlanMost pm = plan_most(most, p->window, p->relay, p->top_k);
  if (pm.globals + pm.W >= (int64_t)1 << 30)
    return err(CRA_E_INVALID, "2^30 keys of a query or more");
  return CRA_OK;
}

int check_prefix(const cra_cache* c, const cra_paged_plan* p, const cra_prefix* x) {
  if (!x) return CRA_OK;
  if (!x->page_table || !x->length) return err(CRA_E_INVALID, "prefix: page_table or length is NULL");
  if (reinterpret_cast<uintptr_t>(x->page_table) % 4 || reinterpret_cast<uintptr_t>(x->length) % 4)
    return err(CRA_E_LAYOUT, "prefix: misaligned pointer");
  if (x->pages < 1) return err(CRA_E_INVALID, "prefix: pages must be >= 1");
  if ((int64_t)x->pages * c->page_size > 0x7fff0000) return err(CRA_E_INVALID, "prefix: 2^31 - 2^16 rows or more");
  if (p->window < 1) return err(CRA_E_INVALID, "a shared prefix needs a window (each length has its own by the rule)");
  const int64_t held = (int64_t)x->pages * c->page_size, rpb = p->relay != 0 ? 1 + p->top_k : 1;
  if ((held / p->window + 1) * rpb + std::min<int64_t>(p->window, held) >= (int64_t)1 << 30)
    return err(CRA_E_INVALID, "prefix: 2^30 keys of a query or more");
  return CRA_OK;
}

Launch plan_launch(const cra_cache* c, const cra_batch* b, const cra_paged_plan* p, const cra_prefix* x) {
  Launch l{};
  const bool f32 = c->dtype == CRA_F32;
  l.grp = p->H_q / c->H_kv;
  l.Dp = c->D <= 32 ? 32 : c->D <= 64 ? 64 : c->D <= 128 ? 128 : 256;
  const int64_t held = (int64_t)b->pages_per_seq * c->page_size;
  l.max_len = (int)std::min<int64_t>(p->max_seqlen, std::min<int64_t>(held, 0x7fffffff));
  const int64_t most_rows = (int64_t)(b->cu_seqlens ? p->max_query_len : b->query_len) * l.grp;
  l.chunk = most_rows > kFewRows;
  l.few = b->cu_seqlens || !l.chunk;
  const PlanMost pm = plan_most(l.max_len, p->window, p->relay, p->top_k);
  const int64_t cap = pm.globals / pm.rpb;  // blocks
  l.list = pm.rpb > 1 && cap > 0;
  l.list_cap = l.list ? pm.globals : 0;
  l.shared = x && (b->cu_seqlens || !l.chunk);  // sequences of at most kFewRows rows
  if (l.shared) {
    const int64_t held_x = (int64_t)x->pages * c->page_size;
    const int rpb = p->relay != 0 ? 1 + p->top_k : 1;
    // (a window of the longest length: nobody sees global rows)
    if (rpb > 1 && (p->relay > 0 || held_x > 2048) && p->window < l.max_len) {
      l.list = true;
      l.plist_cap = (held_x / p->window + 1) * rpb;
    }
    l.plist_bytes = up256(c->H_kv * l.plist_cap * 4);
  }
  l.wide = pm.W > kSelMost || (l.plist_cap && p->window > kSelMost);  // no shorter sequence has wider blocks
  const int64_t bh = (int64_t)b->n_seqs * c->H_kv;
  // a wave a block while that is at most 4096 workgroups: sixteen a CU hide the
  // loads' latency, more of them cost their launch (the 16 and the 64 sequences of
  // select_kernel's figures with 2048, 4096, 8192: 13.2, 14.5, 19.1 and 12.9, 7.1, 9.6 us)
  auto steps = [](int64_t blocks, int64_t of) {
    return std::max<int64_t>(1, std::min<int64_t>((blocks + kSelWaves - 1) / kSelWaves, 4096 / of));
  };
  l.sel_steps = (int)steps(cap, bh);
  if (l.plist_cap) {
    // sequences that share leave the prefix's blocks (all that its pages hold, most
    // likely) to it
    const int64_t held_x = (int64_t)x->pages * c->page_size;
    l.prefix_steps = steps(held_x / p->window, c->H_kv);
    l.sel_steps = (int)steps(std::max<int64_t>(l.max_len - held_x, 0) / p->window + 1, bh);
  }
  l.list_bytes = up256(bh * l.list_cap * 4);
  l.part_rows = (int)std::min<int64_t>(kFewRows, most_rows);
  if (l.few) {
    // the workgroups that are resident at once (LDS and registers allow two to
    // four a CU), but no more than there can be pieces of four tiles
    const int64_t pieces = (few_tile_most(pm, kFewRows) + kFewWaves - 1) / kFewWaves;
    const int lds = kFewWaves * 64 * l.Dp * (f32 ? 2 : c->store == CRA_STORE_SAME ? 2 : 1);
    const int per_cu = lds > 80 * 1024 ? 1 : l.Dp >= 128 ? 2 : 4;
    l.few_grid = (int)std::min<int64_t>(256 * per_cu, bh * pieces);
    l.join = pieces > 1 || l.shared;
    const int64_t most_pieces = bh + 2 * (int64_t)l.few_grid;  // few_pieces()
    if (l.join) {
      l.part_bytes = up256(most_pieces * l.part_rows * (int64_t)l.Dp * 4);
      l.ml_bytes = up256(most_pieces * l.part_rows * 2 * 4);
    }
    l.piece_bytes = up256(((int64_t)b->n_seqs + 1) * 4);
  }
  if (l.shared) {
    const PrefixTiles t = prefix_tiles(c->dtype, l.Dp);
    const int64_t tokens = b->cu_seqlens ? b->tokens : (int64_t)b->n_seqs * b->query_len;
    const int64_t rows = std::min<int64_t>(tokens * l.grp, (int64_t)b->n_seqs * l.part_rows);
    const int64_t items = (rows + t.rows - 1) / t.rows * c->H_kv;  // before their keys are cut
    l.prefix_rows = t.rows;
    l.prefix_most = (int)rows;
    l.prefix_grid = (int)std::max<int64_t>(256, std::min<int64_t>(items, 1024));
    const int64_t parts = std::max<int64_t>(items, l.prefix_grid) * t.rows;  // rows of all pieces
    l.ppart_bytes = up256(parts * l.Dp * 4);
    l.pml_bytes = up256(parts * 2 * 4);
    l.pinfo_bytes = up256(((int64_t)b->n_seqs + 2) * 4);
  }
  if (l.chunk) {
    const int BM = f32 ? kF32Rows : l.Dp > 128 ? 64 : 128, BN = f32 || l.Dp > 128 ? 32 : 64;
    const int64_t tiles = b->cu_seqlens ? (int64_t)b->tokens * l.grp / BM + b->n_seqs
                                        : (most_rows + BM - 1) / BM * b->n_seqs;
    // a sequence is cut only from 16 key tiles on, and the pieces of cut ones are
    // at most kChunkItems (chunk_find)
    const int64_t nk = chunk_tile_most(pm, BM / l.grp + 2, BN);
    const bool cut = nk >= 16;
    l.items = tiles * c->H_kv + (cut ? kChunkItems : 0);
    l.joins = cut ? std::min<int64_t>(tiles * c->H_kv, kChunkItems / 2) : 0;
    if (cut) {
      l.parts = std::min<int64_t>(kChunkItems, tiles * c->H_kv * (nk / 8));
      l.part_bytes = std::max(l.part_bytes, up256(l.parts * BM * (int64_t)l.Dp * 4));
      l.ml_bytes = std::max(l.ml_bytes, up256(l.parts * BM * 2 * 4));
    }
  }
  return l;
}

template <typename F>
hipError_t with_dim(int Dp, F f) {
  switch (Dp) {
    case 32: return f(std::integral_constant<int, 32>());
    case 64: return f(std::integral_constant<int, 64>());
    case 128: return f(std::integral_constant<int, 128>());
    default: return f(std::integral_constant<int, 256>());
  }
}
template <typename F>
hipError_t with_store(int store, F f) {
  return store == CRA_STORE_SAME ? f(std::integral_constant<int, kSame>())
         : store == CRA_STORE_E4M3 ? f(std::integral_constant<int, kE4M3>())
                                   : f(std::integral_constant<int, kInt8>());
}

template <typename T, int STORE, int D>
hipError_t launch_rows(const PagedArgs& a, const Launch& l, int64_t bh, hipStream_t st) {
  if (l.shared) {
    const hipError_t e =
        launch_prefix(std::is_same<T, f16>::value ? CRA_F16 : std::is_same<T, bf16>::value ? CRA_BF16 : CRA_F32,
                      STORE, D, a, (uint32_t)(bh * l.part_rows), (uint32_t)l.few_grid, st);
    if (e) return e;
  } else if (l.few) {
    if constexpr (std::is_same<T, float>::value)
      f32_kernel<STORE, D, true, false><<<(uint32_t)l.few_grid, 256, 0, st>>>(a);
    else
      few_kernel<T, STORE, D, false><<<(uint32_t)l.few_grid, 64 * kFewWaves, 0, st>>>(a);
    if (hipError_t e = hipGetLastError()) return e;
    if (l.join) {
      combine_kernel<T, false><<<(uint32_t)(bh * l.part_rows), 256, 0, st>>>(D, a);
      if (hipError_t e = hipGetLastError()) return e;
    }
  }
  if (l.chunk) {
    if constexpr (std::is_same<T, float>::value) {
      f32_kernel<STORE, D, false, false><<<(uint32_t)l.items, 256, 0, st>>>(a);
      if (hipError_t e = hipGetLastError()) return e;
      const uint32_t items = (uint32_t)l.joins * (kF32Rows / join_rows<D>());
      if (items) f32_join_kernel<D><<<std::min<uint32_t>(items, kJoinGrid), 256, 0, st>>>(items, a);
      return hipGetLastError();
    } else {
      return launch_chunk(std::is_same<T, f16>::value ? CRA_F16 : CRA_BF16, STORE, D, a,
                          (uint32_t)l.items, (uint32_t)l.joins, st);
    }
  }
  return hipSuccess;
}

size_t workspace_of(const cra_cache* c, const cra_batch* b, const cra_paged_plan* p, const cra_prefix* x) {
  return check_paged(c, b, p) || check_prefix(c, p, x) ? 0 : plan_launch(c, b, p, x).bytes();
}

int attend(const cra_cache* c, const cra_batch* b, const cra_paged_plan* p, const cra_prefix* x, cra_tensor q,
           cra_tensor o, void* workspace, size_t workspace_bytes, void* stream) {
  if (int e = check_paged(c, b, p)) return e;
  if (int e = check_prefix(c, p, x)) return e;
  const int vec = c->dtype == CRA_F32 ? 4 : 8;
  for (const cra_tensor* t : {&q, &o}) {
    if (!t->ptr) return err(CRA_E_INVALID, "q or o is NULL");
    if (reinterpret_cast<uintptr_t>(t->ptr) % 16 || t->sb % vec || t->sh % vec || t->ss % vec)
      return err(CRA_E_LAYOUT, "rows of q and o must be 16-byte aligned");
  }
  const Launch l = plan_launch(c, b, p, x);
  const size_t need = l.bytes();
  if (need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16))
    return err(CRA_E_INVALID, "workspace: NULL or misaligned pointer");
  if (workspace_bytes < need) {
    char msg[96];
    snprintf(msg, sizeof(msg), "workspace holds %zu bytes, %zu needed", workspace_bytes, need);
    return err(CRA_E_WORKSPACE, msg);
  }
  const int64_t bh = (int64_t)b->n_seqs * c->H_kv;
  const int64_t most = std::max({bh * l.sel_steps + c->H_kv * l.prefix_steps, bh * l.part_rows, l.items,
                                 (int64_t)l.ppart_bytes / (4 * l.Dp) / std::max(1, l.prefix_rows)});
  if (most >= (int64_t)1 << 24) return err(CRA_E_INVALID, "too many sequences or rows for one launch");
  PagedArgs a{};
  a.c = paged_view(c, b);
  a.q = q.ptr, a.qsb = q.sb, a.qsh = q.sh, a.qss = q.ss;
  a.o = o.ptr, a.osb = o.sb, a.osh = o.sh, a.oss = o.ss;
  a.Hq = p->H_q, a.grp = l.grp, a.D = p->D, a.Ds = c->D;
  a.window = p->window, a.relay = p->relay, a.top_k = p->top_k, a.max_len = l.max_len;
  a.scale = p->scale;
  a.d_grp = fast_div(l.grp);
  a.d_hkv = fast_div(c->H_kv);
  a.list_cap = (int)l.list_cap;
  char* ws = static_cast<char*>(workspace);
  a.list = reinterpret_cast<uint32_t*>(ws);
  a.part = reinterpret_cast<float*>(ws + l.list_bytes);
  a.part_ml = reinterpret_cast<float*>(ws + l.list_bytes + l.part_bytes);
  a.pieces = reinterpret_cast<int32_t*>(ws + l.list_bytes + l.part_bytes + l.ml_bytes);
  a.part_rows = l.part_rows;
  a.parts = (int)l.parts;
  a.few_grid = std::max(1, l.few_grid);
  a.zero_outside = p->zero_outside != 0;
  a.few_only = !l.chunk;
  if (l.shared) {
    a.ptable = x->page_table;
    a.plen = x->length;
    a.pcap = x->pages * c->page_size;
    a.plist_cap = (int)l.plist_cap;
    ws += l.own_bytes();
    a.plist = reinterpret_cast<uint32_t*>(ws);
    a.ppart = reinterpret_cast<float*>(ws + l.plist_bytes);
    a.ppart_ml = reinterpret_cast<float*>(ws + l.plist_bytes + l.ppart_bytes);
    a.pinfo = reinterpret_cast<int32_t*>(ws + l.plist_bytes + l.ppart_bytes + l.pml_bytes);
    a.prefix_grid = l.prefix_grid;
    a.prefix_rows = l.prefix_rows;
    a.prefix_most = l.prefix_most;
  }
  hipStream_t st = (hipStream_t)stream;
  if (l.list) {
    a.d_steps = fast_div(l.sel_steps);
    const uint32_t grid = (uint32_t)(bh * l.sel_steps + c->H_kv * l.prefix_steps);
    auto kernel = l.wide ? (p->top_k <= 2 ? select_wide_kernel<2> : select_wide_kernel<4>)
                         : select_kernel;
    kernel<<<grid, 64 * kSelWaves, 0, st>>>(l.sel_steps, a);
    if (int e = hip_err(hipGetLastError(), "cra_fwd_paged (relay rows)")) return e;
  }
  return hip_err(with_dim(l.Dp, [&](auto d) {
    return with_store(c->store, [&](auto s) {
      constexpr int D = decltype(d)::value, S = decltype(s)::value;
      if (c->dtype == CRA_F16) return launch_rows<f16, S, D>(a, l, bh, st);
      if (c->dtype == CRA_BF16) return launch_rows<bf16, S, D>(a, l, bh, st);
      return launch_rows<float, S, D>(a, l, bh, st);
    });
  }), "cra_fwd_paged");
}

}  // namespace
}  // namespace cra

using namespace cra;

extern "C" {

size_t cra_fwd_paged_workspace_bytes(const cra_cache* c, const cra_batch* b, const cra_paged_plan* p) {
  return workspace_of(c, b, p, nullptr);
}

int cra_fwd_paged(const cra_cache* c, const cra_batch* b, const cra_paged_plan* p, cra_tensor q,
                  cra_tensor o, void* workspace, size_t workspace_bytes, void* stream) {
  return attend(c, b, p, nullptr, q, o, workspace, workspace_bytes, stream);
}

size_t cra_fwd_paged_shared_workspace_bytes(const cra_cache* c, const cra_batch* b, const cra_paged_plan* p,
                                            const cra_prefix* x) {
  return x ? workspace_of(c, b, p, x) : 0;
}

int cra_fwd_paged_shared(const cra_cache* c, const cra_batch* b, const cra_paged_plan* p, const cra_prefix* x,
                         cra_tensor q, cra_tensor o, void* workspace, size_t workspace_bytes, void* stream) {
  if (!x) return err(CRA_E_INVALID, "prefix is NULL");
  return attend(c, b, p, x, q, o, workspace, workspace_bytes, stream);
}

}  // extern "C"
