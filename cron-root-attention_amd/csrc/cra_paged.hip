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
};
// A wave takes a multiple of `at_once(W)` blocks.
template <typename F>
__device__ __forceinline__ SelWork sel_work(const PagedArgs& a, int steps, F at_once) {
  SelWork k{};
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t bh = div_by(blockIdx.x, a.d_steps);  // workgroups a (sequence, head)
  const int nw = steps * kSelWaves, w = (int)(blockIdx.x - bh * steps) * kSelWaves + wave;
  k.b = (int)div_by(bh, a.d_hkv);
  k.h = (int)(bh - (uint32_t)k.b * a.c.H_kv);
  const Seq s = wave_seq(a, k.b);
  k.p = get_plan(a, s.n);
  if (k.p.rpb == 1 || s.m < 1) return k;
  const int ls = s.n - k.p.W > 0 ? s.n - k.p.W : 0;  // window start of the last query
  k.full = ls / k.p.W;
  const int blocks = k.full + (ls != k.full * k.p.W ? 1 : 0), n = at_once(k.p.W);
  const int per = ((blocks + nw - 1) / nw + n - 1) / n * n;
  k.first = w * per;
  k.end = min(blocks, k.first + per);
  k.out = a.list + (int64_t)bh * a.list_cap;
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
  const int32_t* pages = a.c.table + w.b * a.c.table_stride;
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

__global__ __launch_bounds__(64 * kSelWaves) void select_kernel(PagedArgs a, int steps) {
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
__global__ __launch_bounds__(64 * kSelWaves) void select_wide_kernel(PagedArgs a, int steps) {
  const int lane = threadIdx.x & 63;
  const SelWork w = sel_work(a, steps, [](int) { return 1; });
  if (w.first >= w.end) return;
  const SeqPlan p = w.p;
  const int full = w.full, first = w.first, end = w.end;
  const int32_t* pages = a.c.table + w.b * a.c.table_stride;
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
    if (base >= p.W) ++blk, base = 0;
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
// Few rows: at most 16 rows a (sequence, kv head). The keys of all sequences are
// cut into pieces of equal length, as many as keep the resident workgroups busy
// about twice over; each workgroup takes pieces from the grid's stride, each
// wave of it whole 32-key tiles, filled with per-lane addresses straight into
// its part of LDS (a row of a page is contiguous, rows lie anywhere), with no
// barrier until the piece's end; the 16-column operand Q^T holds the rows.
// Bound by memory latency and bandwidth: the rows seen, once per kv head. The
// waves' results, and those of a sequence's pieces, are joined by their maxima.
// Measured (D = 128, with combine_kernel's 4-5 us behind it): one token of 131072, 16
// heads fp16 9 us; 64 of 1-32768, 32/8 heads bf16 17 us; 16 of 700-131072 over an
// e4m3 store 16 us; 14 sequences of 1-20000, dense, 16/4 heads, int8 23 us + 6 us.
// Up to D = 64 the registers are held to three waves a SIMD (D = 64: 168; left to
// itself the compiler takes 170, and two waves).
// ---------------------------------------------------------------------------
constexpr int kFewWaves = 4;

// 32-key tiles of a sequence that few rows attend (0: it has no new tokens, or
// more rows than the kernel takes), found out from the device's lengths.
struct FewTiles {
  int tiles;
  bool mine;  // takes at least one piece
};
__device__ __forceinline__ FewTiles few_tiles(const PagedArgs& a, int b) {
  const Seq s = get_seq(a, b);
  const int64_t rows = (int64_t)s.m * a.grp;
  // more rows than the caller's bound: one piece, which answers NaN
  if (rows == 0 || (rows > a.part_rows && !a.few_only)) return FewTiles{0, false};
  if (rows > a.part_rows) return FewTiles{0, true};
  return FewTiles{few_tile_count(s.n, s.m, get_plan(a, s.n)), true};
}
// The pieces of the call: tiles a piece, and pieces a kv head. Every wave adds
// the sequences up, 64 at a time; the first 64 stay in registers (lane b).
struct FewPieces {
  int per, total;
  int n, upto;  // of sequence `lane`: pieces, and pieces up to its last
};
__device__ __forceinline__ int few_count(const FewTiles& t, int per) {
  return t.mine ? max(1, (t.tiles + per - 1) / per) : 0;
}
__device__ __forceinline__ FewPieces few_pieces(const PagedArgs& a) {
  const int lane = threadIdx.x & 63;
  FewTiles t0{0, false};
  int64_t tiles = 0;
  for (int base = 0; base < a.c.n_seqs; base += 64) {
    FewTiles t{0, false};
    if (base + lane < a.c.n_seqs) t = few_tiles(a, base + lane);
    if (base == 0) t0 = t;
    tiles += (uint32_t)__builtin_amdgcn_readlane((int)wave_upto(t.tiles), 63);
  }
  // at most 2 few_grid pieces of whole length, and one short one a sequence
  const int64_t per = (tiles * a.c.H_kv + 2 * a.few_grid - 1) / (2 * a.few_grid);
  FewPieces f{};
  f.per = (int)min(max(per, (int64_t)1) + kFewWaves - 1, (int64_t)1 << 28) / kFewWaves * kFewWaves;
  for (int base = 0; base < a.c.n_seqs; base += 64) {
    FewTiles t = t0;
    if (base > 0) {
      t = FewTiles{0, false};
      if (base + lane < a.c.n_seqs) t = few_tiles(a, base + lane);
    }
    const int n = few_count(t, f.per), upto = f.total + (int)wave_upto(n);
    if (base == 0) f.n = n, f.upto = upto;
    if (blockIdx.x == 0 && threadIdx.x < 64 && base + lane < a.c.n_seqs) a.pieces[base + lane] = upto - n;
    f.total = __builtin_amdgcn_readlane(upto, 63);
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.pieces[a.c.n_seqs] = f.total;
  return f;
}
// Sequence of piece `idx` of a kv head, which of its pieces it is, and whether
// it is its only one.
struct FewPiece {
  int b, piece;
  bool only;
};
__device__ __forceinline__ FewPiece few_piece(const PagedArgs& a, const FewPieces& f, int idx) {
  const int lane = threadIdx.x & 63;
  int n = f.n, upto = f.upto;
  for (int base = 0;;) {
    const uint64_t hit = __ballot(upto > idx);
    if (hit) {
      const int l = __builtin_ctzll(hit), mine = __builtin_amdgcn_readlane(n, l);
      return FewPiece{base + l, idx - (__builtin_amdgcn_readlane(upto, l) - mine), mine == 1};
    }
    base += 64;
    if (base >= a.c.n_seqs) return FewPiece{-1, 0, false};
    const int before = __builtin_amdgcn_readlane(upto, 63);
    FewTiles t{0, false};
    if (base + lane < a.c.n_seqs) t = few_tiles(a, base + lane);
    n = few_count(t, f.per);
    upto = before + (int)wave_upto(n);
  }
}

// Rows of tokens before the first and behind the last sequence: zeros, shared by
// the grid's workgroups (a fresh output; the caller's own is left as it is).
template <typename T>
__device__ __forceinline__ void zero_outside(const PagedArgs& a, int threads) {
  if (!a.zero_outside || !a.c.cu) return;
  const int first = token_range(a.c.cu, 0, a.c.tokens).first;
  const int last = token_range(a.c.cu, a.c.n_seqs - 1, a.c.tokens).last;
  const int64_t outside = (int64_t)first + a.c.tokens - last, quads = a.D / 4;
  const int64_t all = outside * a.Hq * quads;
  for (int64_t i = (int64_t)blockIdx.x * threads + threadIdx.x; i < all; i += (int64_t)gridDim.x * threads) {
    const int64_t row = i / quads;
    const int64_t tok = row / a.Hq, t = tok < first ? tok : last + (tok - first);
    T* p = static_cast<T*>(a.o) + (row - tok * a.Hq) * a.osh + t * a.oss + (i - row * quads) * 4;
    typedef T t4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<t4*>(p) = t4{(T)0.f, (T)0.f, (T)0.f, (T)0.f};
  }
}

// ROWS rows of RB bytes, 16-byte chunks XOR-swizzled as in SwzTile.
template <int RB, int ROWS>
struct ByteTile {
  static constexpr int kCPR = RB / 16;
  static constexpr int kRPL = RB < 256 ? 256 / RB : 1;
  static constexpr int kSwz = kCPR < 16 ? kCPR : 16;
  static constexpr int kBytes = RB * ROWS;
  static constexpr int kInstr = kBytes / 1024;  // 64 lanes x 16 bytes
  __device__ __forceinline__ static int swz(int row) { return (row / kRPL) % kSwz; }
  __device__ __forceinline__ static int off(int row, int chunk) {
    return row * RB + ((chunk ^ swz(row)) << 4);
  }
};

template <typename T, int STORE, int D>
__global__ __launch_bounds__(64 * kFewWaves) __attribute__((amdgpu_waves_per_eu(D > 128 ? 1 : D > 64 ? 2 : 3)))
void few_kernel(PagedArgs a) {
  constexpr int NW = kFewWaves;
  constexpr int ES = STORE == kSame ? 2 : 1;
  using Tile = ByteTile<D * ES, 32>;
  __shared__ __attribute__((aligned(1024))) char stage[NW][2][Tile::kBytes];
  __shared__ float scales[NW][64];
  __shared__ float join_ml[NW][kFewRows][2];

  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row_bytes = a.Ds * ES;
  zero_outside<T>(a, 64 * NW);
  const FewPieces fp = few_pieces(a);
  for (int64_t item = blockIdx.x; item < (int64_t)fp.total * a.c.H_kv; item += gridDim.x) {
  const uint32_t idx = div_by((uint32_t)item, a.d_hkv);
  const int hk = (int)((uint32_t)item - idx * a.c.H_kv);
  const FewPiece fi = few_piece(a, fp, (int)idx);
  const int b = fi.b;
  if (b < 0) break;
  const Seq s = wave_seq(a, b);
  const int64_t rows64 = (int64_t)s.m * a.grp;
  if (rows64 > a.part_rows) {  // more new tokens than the caller's bound
    for (int64_t i = tid; i < rows64 * a.D; i += 64 * NW) {
      const int r = (int)(i / a.D);
      o_row<T>(a, s, hk, r)[i - (int64_t)r * a.D] = from_f32<T>(__builtin_nanf(""));
    }
    continue;
  }
  const int rows = (int)rows64;
  const SeqPlan p = get_plan(a, s.n);
  const int pos0 = s.n - s.m;  // of the first new token
  const int G = s.n > 0 ? seq_prefix(s.n - 1, p) : 0;
  const int lo = max(0, max(pos0, 0) - p.W + 1);
  const int nG = (G + 31) >> 5, nAll = nG + ((s.n - lo + 31) >> 5);
  const int nT = min(nAll, (fi.piece + 1) * fp.per);  // the piece's tiles end here
  const int32_t* pages = a.c.table + b * a.c.table_stride;
  const uint32_t* list = a.list + ((int64_t)b * a.c.H_kv + hk) * a.list_cap;
  bool bad = s.over;
  const int step = NW;
  int it = fi.piece * fp.per + wave;

  // cache row of the tile's row lane % 32
  auto slot_of = [&](int it) -> uint32_t {
    const int ko = lane & 31;
    if (it < nG) {
      const int i = min(it * 32 + ko, G - 1);
      if (p.rpb > 1) return list[i];
      return seq_row(pages, i * p.W, a.c.num_pages, a.c.H_kv, a.c.log_page, hk);
    }
    const int i = min(lo + (it - nG) * 32 + ko, s.n - 1);
    return seq_row(pages, i, a.c.num_pages, a.c.H_kv, a.c.log_page, hk);
  };
  auto fill = [&](char (&dst)[2][Tile::kBytes], uint32_t slot) {
#pragma unroll
    for (int i = 0; i < Tile::kInstr; ++i) {
      const int row = (i * 64 + lane) / Tile::kCPR;
      const int chunk = (lane % Tile::kCPR) ^ Tile::swz(row);
      const int64_t at = (int64_t)(uint32_t)__shfl((int)slot, row) * row_bytes + chunk * 16;
      if (chunk * 16 < row_bytes) {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(a.c.k + at),
                                         CRA_LDS(dst[0] + i * 1024), 16, 0, 0);
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(a.c.v + at),
                                         CRA_LDS(dst[1] + i * 1024), 16, 0, 0);
      }
    }
  };
  // scales of the tile's rows: k in lanes 0..31, v in lanes 32..63
  auto load_scale = [&](uint32_t slot) -> float {
    if constexpr (STORE == kSame) return 0.f;
    return (lane < 32 ? a.c.k_scale : a.c.v_scale)[slot];
  };
  auto checked = [&](uint32_t slot) -> uint32_t {
    bad |= slot == kNoRow;
    return slot == kNoRow ? 0u : slot;
  };

  if (D * ES > row_bytes) {  // columns that no load fills
    for (int i = lane; i < 2 * Tile::kBytes / 16; i += 64)
      reinterpret_cast<uint4*>(stage[wave])[i] = make_uint4(0, 0, 0, 0);
    wait_all();  // before loads to the same memory
  }
  float sc = 0.f;
  uint32_t next = 0;
  auto start = [&]() {
    if (it >= nT) return;
    const uint32_t first = checked(slot_of(it));
    fill(stage[wave], first);
    sc = load_scale(first);
    if (it + step < nT) next = slot_of(it + step);
  };
  start();

  Frag<T> qf[D / 32];
  const bool have = l16 < rows;
  const T* qp = q_row<T>(a, s, hk, have ? l16 : 0);
#pragma unroll
  for (int c = 0; c < D / 32; ++c)
    qf[c] = have && 32 * c + 8 * g < a.D ? lds_frag_row<T>(qp + 32 * c + 8 * g) : zero_frag<T>();
  const int pos = have ? pos0 + row_token(a, l16) : -1;
  const int glen = pos >= 0 ? seq_prefix(pos, p) : 0;
  const int glen0 = pos0 >= 0 ? seq_prefix(pos0, p) : 0;
  const float c2 = a.scale * kLog2e;
  float m_run = -kInf, l_run = 0.f;
  f32x4 acc[D / 16][1];
#pragma unroll
  for (int db = 0; db < D / 16; ++db) acc[db][0] = f32x4{0.f, 0.f, 0.f, 0.f};
  bool careful = false;  // look for elements of V that are not finite in every tile

  auto attend = [&](const char (&cur)[2][Tile::kBytes], int it, float sc_now) __attribute__((always_inline)) {
    const char *tK = cur[0], *tV = cur[1];
    f32x4 sK[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        Frag<T> kf;
        if constexpr (STORE == kSame) {
          kf.w[0] = *reinterpret_cast<const uint4*>(tK + Tile::off(16 * kb + l16, 4 * c + g));
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(
              tK + Tile::off(16 * kb + l16, 2 * c + (g >> 1)) + 8 * (g & 1));
          const uint2 x = widen4<T, STORE>(w.x), y = widen4<T, STORE>(w.y);
          kf.w[0] = make_uint4(x.x, x.y, y.x, y.y);
        }
        sK[kb] = mma(sK[kb], kf, qf[c]);
      }
    float ks[8], vs[8];
    if constexpr (STORE != kSame) {
      scales[wave][lane] = sc_now;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          ks[4 * kb + r] = scales[wave][16 * kb + 4 * g + r];
          vs[4 * kb + r] = scales[wave][32 + 16 * kb + 4 * g + r];
        }
    }
    const bool loc = it >= nG;
    const int ts = loc ? lo + (it - nG) * 32 : it * 32;
    const int hi = loc ? pos - ts : glen - 1 - ts;
    const unsigned span = loc ? (unsigned)(p.W - 1) : 0x7fffffffu;
    float x[8], mx = -kInf;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = sK[i >> 2][i & 3] * c2;
      if constexpr (STORE != kSame) v *= ks[i];
      const int ko = 16 * (i >> 2) + 4 * g + (i & 3);
      x[i] = (unsigned)(hi - ko) <= span ? v : -kInf;
      mx = fmaxf(mx, x[i]);
    }
    // rows behind the end of a range repeat its last row (slot_of): not seen either
    const float m_new = fmaxf(m_run, group_max(mx));
    const float mu = m_new == -kInf ? 0.f : m_new;
    if (__any(m_new > m_run)) {
      const float alpha = __builtin_amdgcn_exp2f(m_run - mu);
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < D / 16; ++db) acc[db][0] *= alpha;
      m_run = m_new;
    }
    float pv[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      pv[i] = __builtin_amdgcn_exp2f(x[i] - mu);
      l_run += pv[i];
    }
    float vref = 1.f;
    if constexpr (STORE != kSame) {
#pragma unroll
      for (int i = 0; i < 8; ++i) pv[i] = x[i] == -kInf ? 0.f : pv[i] * vs[i];
      if constexpr (std::is_same<T, f16>::value) {
        // p times a row's scale would leave fp16's range: it is taken relative to the
        // query's largest in the tile, which multiplies the product in fp32
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) most = fmaxf(most, pv[i]);
        most = group_max(most);
        vref = most > 0x1p-100f ? most : 1.f;
        const float inv = 1.f / vref;
#pragma unroll
        for (int i = 0; i < 8; ++i) pv[i] *= inv;
      }
    }
    const Frag<T> pf[1] = {pack8<T>(pv)};
    auto v_frag = [&](int db) __attribute__((always_inline)) {
      Frag<T> vt;
      if constexpr (STORE == kSame) {
        const int row = 4 * g + (l16 >> 2), chunk = 2 * db + ((l16 & 3) >> 1), in = 8 * (l16 & 1);
        vt = SwzTile<D, 32>::template tr_frag_at<T>(tV + Tile::off(row, chunk) + in,
                                                    tV + Tile::off(row + 16, chunk) + in);
      } else {
        typedef int i32x2 __attribute__((ext_vector_type(2)));
        const int j = l16 >> 1, row = (j < 4 ? 0 : 12) + 4 * g + j;
        const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (__attribute__((address_space(3))) i32x2*)(tV + Tile::off(row, db) + 8 * (l16 & 1)));
        const uint2 x0 = widen4<T, STORE>((uint32_t)w[0]), x1 = widen4<T, STORE>((uint32_t)w[1]);
        vt.w[0] = make_uint4(x0.x, x0.y, x1.x, x1.y);
      }
      return vt;
    };
    // one new token: every row of the tile, a repeated last one too, is a row that its
    // query sees, and what is not finite in it shows in the result
    const bool full = s.m == 1 || (loc ? ts >= s.n - p.W && ts + 31 <= pos0 : ts + 32 <= glen0);
    if (!full || careful) {
      f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
      const Frag<T> one = ones_frag<T>();
#pragma unroll
      for (int db = 0; db < D / 16; ++db) sum = mma(sum, v_frag(db), one);
      if (any_not_finite(sum)) {
        TileMask<1> mk;
        mk.hi[0] = hi;
        mk.span[0] = span;
        pv_not_finite<T, D / 16, 1>(v_frag, pf, acc, mk, 0, g, vref);
        return;
      }
    }
#pragma unroll
    for (int db = 0; db < D / 16; ++db) {
      if constexpr (STORE != kSame && std::is_same<T, f16>::value)
        acc[db][0] += mma(f32x4{0.f, 0.f, 0.f, 0.f}, v_frag(db), pf[0]) * vref;
      else
        acc[db][0] = mma(acc[db][0], v_frag(db), pf[0]);
    }
  };
  for (;;) {
    for (; it < nT; it += step) {
      wait_all();
      attend(stage[wave], it, sc);
      wait_all();  // LDS reads are done before the loads that overwrite
      if (it + step < nT) {
        const uint32_t slot = checked(next);
        fill(stage[wave], slot);
        sc = load_scale(slot);
        if (it + 2 * step < nT) next = slot_of(it + 2 * step);
      }
    }
    if (STORE != kSame || careful) break;  // (8-bit codes are finite: P holds a scale that is not)
    // An infinity in V times a weight of 0 (of a repeated last row, or rounded to 0 in
    // fp16) has made a NaN where the row's query gets the infinity: the wave's tiles
    // once more.
    float z = 0.f;
#pragma unroll
    for (int db = 0; db < D / 16; ++db)
#pragma unroll
      for (int r = 0; r < 4; ++r) z += acc[db][0][r] - acc[db][0][r];
    if (!__any(have && !(z == 0.f))) break;
    careful = true;
    m_run = -kInf;
    l_run = 0.f;
#pragma unroll
    for (int db = 0; db < D / 16; ++db) acc[db][0] = f32x4{0.f, 0.f, 0.f, 0.f};
    it = fi.piece * fp.per + wave;
    start();
  }

  // join the waves
  l_run = group_sum(l_run);
  if (__any(bad)) l_run = __builtin_nanf("");
  __syncthreads();
  // the tiles' memory holds the waves' O now: [wave][row][D], quads swizzled by row
  static_assert(sizeof(float) * NW * kFewRows * D <= sizeof(stage), "join area");
  f32x4* join_o = reinterpret_cast<f32x4*>(&stage[0][0][0]);
  auto join_at = [](int w, int r, int quad) {
    return (w * kFewRows + r) * (D / 4) + (quad ^ (r & (D / 4 - 1)));
  };
#pragma unroll
  for (int db = 0; db < D / 16; ++db) join_o[join_at(wave, l16, 4 * db + g)] = acc[db][0];
  if (g == 0) {
    join_ml[wave][l16][0] = m_run;
    join_ml[wave][l16][1] = l_run;
  }
  __syncthreads();
  for (int i = tid; i < rows * (D / 4); i += 64 * NW) {
    const int r = i / (D / 4), c = i % (D / 4) * 4;
    float M = -kInf;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, join_ml[w][r][0]);
    float L = 0.f;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = join_ml[w][r][0];
      const float e = mw == -kInf ? 0.f : __builtin_amdgcn_exp2f(mw - M);
      L += e * join_ml[w][r][1];
      o += join_o[join_at(w, r, c / 4)] * e;
    }
    if (fi.only) {
      if (c >= a.D) continue;
      const float inv = L == 0.f ? 0.f : 1.f / L;
      T e[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) e[j] = from_f32<T>(o[j] * inv);
      *reinterpret_cast<uint2*>(o_row<T>(a, s, hk, r) + c) = *reinterpret_cast<const uint2*>(e);
    } else {
      const int64_t at = item * a.part_rows + r;
      *reinterpret_cast<f32x4*>(a.part + at * D + c) = o;
      if (c == 0) {
        a.part_ml[2 * at] = M;
        a.part_ml[2 * at + 1] = L;
      }
    }
  }
  __syncthreads();  // the join area is the next piece's tiles
  }
}

// Joins the pieces of sequences that have more than one: one workgroup a
// (sequence, kv head, row), its threads 4 columns each of some of the pieces.
template <typename T>
__global__ __launch_bounds__(256) void combine_kernel(PagedArgs a, int Dp) {
  __shared__ float red[256][4];
  __shared__ float red_l[64];
  const int tid = threadIdx.x;
  const int r = blockIdx.x % a.part_rows;
  const uint32_t bh = blockIdx.x / a.part_rows;
  const int b = (int)div_by(bh, a.d_hkv), hk = (int)(bh - (uint32_t)b * a.c.H_kv);
  const int first = a.pieces[b], n = a.pieces[b + 1] - first;
  if (n < 2) return;
  const Seq s = wave_seq(a, b);
  if (r >= (int64_t)s.m * a.grp) return;
  const int quads = Dp / 4, lanes = 256 / quads;  // groups of pieces
  const int quad = tid % quads, sg = tid / quads;
  auto at = [&](int i) { return ((int64_t)(first + i) * a.c.H_kv + hk) * a.part_rows + r; };
  float M = -kInf;  // a lane a piece, each wave for itself
  for (int i = tid & 63; i < n; i += 64) M = fmaxf(M, a.part_ml[2 * at(i)]);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor(M, d));
  float L = 0.f;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = sg; i < n; i += lanes) {
    const float mi = a.part_ml[2 * at(i)];
    const float e = mi == -kInf ? 0.f : __builtin_amdgcn_exp2f(mi - M);
    L += e * a.part_ml[2 * at(i) + 1];
    o += *reinterpret_cast<const f32x4*>(a.part + at(i) * Dp + quad * 4) * e;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) red[tid][j] = o[j];
  if (quad == 0) red_l[sg] = L;
  __syncthreads();
  if (sg != 0 || quad * 4 >= a.D) return;
  L = 0.f;
  for (int i = 0; i < lanes; ++i) L += red_l[i];
  const float inv = L == 0.f ? 0.f : 1.f / L;
  T* op = o_row<T>(a, s, hk, r) + quad * 4;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float x = 0.f;
    for (int i = 0; i < lanes; ++i) x += red[i * quads + quad][j];
    op[j] = from_f32<T>(x * inv);
  }
}

// ---------------------------------------------------------------------------
// fp32: tiles of 64 rows, 32 keys at a time as fp32 in LDS (8-bit codes times
// their scale), v_mfma_f32_16x16x4_f32. FEW: at most 16 rows (one of the four waves
// has rows, all of them load) and a piece of the key tiles, else a chunk tile.
// ---------------------------------------------------------------------------
__device__ __forceinline__ f32x4 mma4(f32x4 c, float x, float y) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(x, y, c, 0, 0, 0);
}

constexpr int kF32Rows = 64, kF32Keys = 32;

// One work item: rows r0.. of a (sequence, kv head) over its key tiles from
// t_first up to t_end; the result goes to o, or (part_at >= 0) to the partial rows.
template <int STORE, int D>
__device__ void f32_item(const PagedArgs& a, const Seq& s, int b, int hk, int r0, int t_first, int t_end,
                         int64_t part_at) {
  constexpr int BN = kF32Keys, kStride = D + 4;
  __shared__ __attribute__((aligned(16))) float tK[BN][kStride];
  __shared__ __attribute__((aligned(16))) float tV[BN][kStride];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, g = lane >> 4;
  const int rows = s.m * a.grp, q0 = r0 + 16 * wave;
  const SeqPlan p = get_plan(a, s.n);
  const int pos0 = s.n - s.m;
  auto pos_of = [&](int r) { return pos0 + row_token(a, r); };
  const int wg_first = pos_of(r0), wg_last = pos_of(min(r0 + kF32Rows, rows) - 1);
  const int lo_k = max(0, wg_first - p.W + 1), hi = max(0, wg_last + 1);
  const int gmax = seq_prefix(wg_last, p);
  const int nglob = (gmax + BN - 1) / BN, ntot = nglob + (hi > lo_k ? (hi - lo_k + BN - 1) / BN : 0);
  const int32_t* pages = a.c.table + b * a.c.table_stride;
  const uint32_t* list = a.list + ((int64_t)b * a.c.H_kv + hk) * a.list_cap;
  bool bad = s.over;

  // eight threads a row, D / 8 columns each: quads of them, 32 columns apart
  constexpr int kCols = D / 8;
  const int frow = tid >> 3, fcol = (tid & 7) * 4;
  f32x4 rk[kCols / 4], rv[kCols / 4];
  auto load = [&](int it) {
    const int ts = it >= nglob ? lo_k + (it - nglob) * BN : it * BN;
    uint32_t sl;
    if (it < nglob) {
      const int i = min(ts + frow, gmax - 1);
      sl = p.rpb > 1 ? list[i] : seq_row(pages, i * p.W, a.c.num_pages, a.c.H_kv, a.c.log_page, hk);
    } else {
      sl = seq_row(pages, min(ts + frow, hi - 1), a.c.num_pages, a.c.H_kv, a.c.log_page, hk);
    }
    bad |= sl == kNoRow;
    if (sl == kNoRow) sl = 0;
    const int64_t at = (int64_t)sl * a.Ds;
    float ks = 1.f, vs = 1.f;
    if (STORE != kSame) ks = a.c.k_scale[sl], vs = a.c.v_scale[sl];
#pragma unroll
    for (int j = 0; j < kCols / 4; ++j) {
      const int col = fcol + 32 * j;
      rk[j] = rv[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (col >= a.Ds) continue;
      if constexpr (STORE == kSame) {
        rk[j] = *reinterpret_cast<const f32x4*>(a.c.k + (at + col) * 4);
        rv[j] = *reinterpret_cast<const f32x4*>(a.c.v + (at + col) * 4);
      } else {
        const uint32_t wk = *reinterpret_cast<const uint32_t*>(a.c.k + at + col);
        const uint32_t wv = *reinterpret_cast<const uint32_t*>(a.c.v + at + col);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          rk[j][i] = code_value<STORE>(wk, i) * ks;
          rv[j][i] = code_value<STORE>(wv, i) * vs;
        }
      }
    }
  };
  auto store = [&]() {
#pragma unroll
    for (int j = 0; j < kCols / 4; ++j) {
      *reinterpret_cast<f32x4*>(&tK[frow][fcol + 32 * j]) = rk[j];
      *reinterpret_cast<f32x4*>(&tV[frow][fcol + 32 * j]) = rv[j];
    }
  };
  const int t_last = min(t_end, ntot);
  if (t_first < t_last) load(t_first);

  const int r = q0 + l16;
  const bool have = r < rows, active = q0 < rows;
  const int pos = have ? pos_of(r) : -1;
  const int glen = pos >= 0 ? seq_prefix(pos, p) : 0;
  const int first = active ? pos_of(q0) : 0, last = active ? pos_of(min(q0 + 16, rows) - 1) : -1;
  const int w_lo = max(0, first - p.W + 1);
  const int g_all = active ? seq_prefix(first, p) : 0, g_any = active ? seq_prefix(last, p) : 0;
  // Q^T operand: MFMA 4 c + i of a 16-column step takes column 16 c + 4 g + i
  f32x4 qf[D / 16];
  const float* qp = q_row<float>(a, s, hk, have ? r : 0);
#pragma unroll
  for (int c = 0; c < D / 16; ++c)
    qf[c] = have && 16 * c + 4 * g < a.D ? *reinterpret_cast<const f32x4*>(qp + 16 * c + 4 * g)
                                         : f32x4{0.f, 0.f, 0.f, 0.f};
  const float c2 = a.scale * kLog2e;
  float m_run = -kInf, l_run = 0.f;
  f32x4 acc[D / 16];
#pragma unroll
  for (int db = 0; db < D / 16; ++db) acc[db] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int it = t_first; it < t_last; ++it) {
    __syncthreads();  // every wave is done with the previous tile
    store();
    __syncthreads();
    if (it + 1 < t_last) load(it + 1);
    const bool loc = it >= nglob;
    const int ts = loc ? lo_k + (it - nglob) * BN : it * BN;
    if (!(active && (loc ? ts <= last && ts + BN - 1 >= w_lo : ts < g_any))) continue;
    const bool full = loc ? ts >= last - p.W + 1 && ts + BN - 1 <= first : ts + BN <= g_all;
    const int vis = loc ? pos - ts : glen - 1 - ts;
    const unsigned span = loc ? (unsigned)(p.W - 1) : 0x7fffffffu;
    f32x4 sc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const f32x4 k = *reinterpret_cast<const f32x4*>(&tK[16 * kb + l16][16 * c + 4 * g]);
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[kb] = mma4(sc[kb], k[i], qf[c][i]);
      }
    float x[8], mx = -kInf;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int ko = 16 * (i >> 2) + 4 * g + (i & 3);
      x[i] = (unsigned)(vis - ko) <= span ? sc[i >> 2][i & 3] * c2 : -kInf;
      mx = fmaxf(mx, x[i]);
    }
    const float m_new = fmaxf(m_run, group_max(mx));
    const float mu = m_new == -kInf ? 0.f : m_new;
    if (__any(m_new > m_run)) {
      const float alpha = __builtin_amdgcn_exp2f(m_run - mu);
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < D / 16; ++db) acc[db] *= alpha;
      m_run = m_new;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = __builtin_amdgcn_exp2f(x[i] - mu);
      l_run += x[i];
    }
#pragma unroll
    for (int db = 0; db < D / 16; ++db) {
      // P^T register i is key 16 (i / 4) + 4 g + i % 4 of the lane's query
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = tV[16 * (i >> 2) + 4 * g + (i & 3)][16 * db + l16];
      if (full) {
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[db] = mma4(acc[db], v[i], x[i]);
        continue;
      }
      f32x4 t = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 8; ++i) t = mma4(t, v[i], x[i]);
      const float z = (t[0] - t[0]) + (t[1] - t[1]) + (t[2] - t[2]) + (t[3] - t[3]);
      if (__any(have && !(z == 0.f))) {  // a query at a time, over the rows it sees
#pragma unroll 1
        for (int qi = 0; qi < 16; ++qi) {
          const int h = __shfl(vis, qi);
          f32x4 c = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int ko = 16 * (i >> 2) + 4 * g + (i & 3);
            c = mma4(c, (unsigned)(h - ko) <= span ? v[i] : 0.f, l16 == qi ? x[i] : 0.f);
          }
          if (l16 == qi) t = c;
        }
      }
      acc[db] += t;
    }
  }

  bad = __syncthreads_or(bad);
  l_run = group_sum(l_run);
  if (bad) l_run = __builtin_nanf("");
  if (!have) return;
  if (part_at < 0) {
    const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
    float* op = o_row<float>(a, s, hk, r);
#pragma unroll
    for (int db = 0; db < D / 16; ++db)
      if (16 * db + 4 * g < a.D) *reinterpret_cast<f32x4*>(op + 16 * db + 4 * g) = acc[db] * inv;
  } else {
    const int64_t at = part_at + (r - r0);
#pragma unroll
    for (int db = 0; db < D / 16; ++db)
      *reinterpret_cast<f32x4*>(a.part + at * D + 16 * db + 4 * g) = acc[db];
    if (g == 0) {
      a.part_ml[2 * at] = m_run;
      a.part_ml[2 * at + 1] = l_run;
    }
  }
}

template <int STORE, int D, bool FEW>
__global__ __launch_bounds__(256) void f32_kernel(PagedArgs a) {
  if constexpr (FEW) {
    zero_outside<float>(a, 256);
    const FewPieces fp = few_pieces(a);
    for (int64_t item = blockIdx.x; item < (int64_t)fp.total * a.c.H_kv; item += gridDim.x) {
      const uint32_t idx = div_by((uint32_t)item, a.d_hkv);
      const int hk = (int)((uint32_t)item - idx * a.c.H_kv);
      const FewPiece fi = few_piece(a, fp, (int)idx);
      if (fi.b < 0) break;
      const Seq s = wave_seq(a, fi.b);
      const int64_t rows = (int64_t)s.m * a.grp;
      if (rows > a.part_rows) {  // more new tokens than the caller's bound
        for (int64_t i = threadIdx.x; i < rows * a.D; i += 256) {
          const int r = (int)(i / a.D);
          o_row<float>(a, s, hk, r)[i - (int64_t)r * a.D] = __builtin_nanf("");
        }
        continue;
      }
      f32_item<STORE, D>(a, s, fi.b, hk, 0, fi.piece * fp.per, (fi.piece + 1) * fp.per,
                         fi.only ? -1 : item * a.part_rows);
    }
  } else {
    const ChunkWork w = chunk_work<kF32Rows, kF32Keys>(a);
    if (w.b < 0) return;
    f32_item<STORE, D>(a, wave_seq(a, w.b), w.b, w.hk, w.tile * kF32Rows, w.t_first, w.t_end, w.part);
  }
}

template <int D>
__global__ __launch_bounds__(256) void f32_join_kernel(PagedArgs a, uint32_t items) {
  join_chunk<float, kF32Rows, kF32Keys, D>(a, items);
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
  int part_rows, few_grid;
  bool join;              // a sequence's keys may be cut into pieces
  int64_t items, joins;   // chunk pieces and row tiles of cut sequences, over all kv heads, at most
  int64_t parts;          // pieces of cut sequences that the workspace holds
  size_t list_bytes, part_bytes, ml_bytes, piece_bytes;
  size_t bytes() const { return list_bytes + part_bytes + ml_bytes + piece_bytes; }
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

Launch plan_launch(const cra_cache* c, const cra_batch* b, const cra_paged_plan* p) {
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
  l.wide = pm.W > kSelMost;  // no shorter sequence has wider blocks
  const int64_t bh = (int64_t)b->n_seqs * c->H_kv;
  // a wave a block while that is at most 4096 workgroups: sixteen a CU hide the
  // loads' latency, more of them cost their launch (the 16 and the 64 sequences of
  // select_kernel's figures with 2048, 4096, 8192: 13.2, 14.5, 19.1 and 12.9, 7.1, 9.6 us)
  l.sel_steps = (int)std::max<int64_t>(1, std::min<int64_t>((cap + kSelWaves - 1) / kSelWaves, 4096 / bh));
  l.list_bytes = up256(bh * l.list_cap * 4);
  l.part_rows = (int)std::min<int64_t>(kFewRows, most_rows);
  if (l.few) {
    // the workgroups that are resident at once (LDS and registers allow two to
    // four a CU), but no more than there can be pieces of four tiles
    const int64_t pieces = (few_tile_most(pm, kFewRows) + kFewWaves - 1) / kFewWaves;
    const int lds = kFewWaves * 64 * l.Dp * (f32 ? 2 : c->store == CRA_STORE_SAME ? 2 : 1);
    const int per_cu = lds > 80 * 1024 ? 1 : l.Dp >= 128 ? 2 : 4;
    l.few_grid = (int)std::min<int64_t>(256 * per_cu, bh * pieces);
    l.join = pieces > 1;
    const int64_t most_pieces = bh + 2 * (int64_t)l.few_grid;  // few_pieces()
    if (l.join) {
      l.part_bytes = up256(most_pieces * l.part_rows * (int64_t)l.Dp * 4);
      l.ml_bytes = up256(most_pieces * l.part_rows * 2 * 4);
    }
    l.piece_bytes = up256(((int64_t)b->n_seqs + 1) * 4);
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
  if (l.few) {
    if constexpr (std::is_same<T, float>::value)
      f32_kernel<STORE, D, true><<<(uint32_t)l.few_grid, 256, 0, st>>>(a);
    else
      few_kernel<T, STORE, D><<<(uint32_t)l.few_grid, 64 * kFewWaves, 0, st>>>(a);
    if (hipError_t e = hipGetLastError()) return e;
    if (l.join) {
      combine_kernel<T><<<(uint32_t)(bh * l.part_rows), 256, 0, st>>>(a, D);
      if (hipError_t e = hipGetLastError()) return e;
    }
  }
  if (l.chunk) {
    if constexpr (std::is_same<T, float>::value) {
      f32_kernel<STORE, D, false><<<(uint32_t)l.items, 256, 0, st>>>(a);
      if (hipError_t e = hipGetLastError()) return e;
      const uint32_t items = (uint32_t)l.joins * (kF32Rows / join_rows<D>());
      if (items) f32_join_kernel<D><<<std::min<uint32_t>(items, kJoinGrid), 256, 0, st>>>(a, items);
      return hipGetLastError();
    } else {
      return launch_chunk(std::is_same<T, f16>::value ? CRA_F16 : CRA_BF16, STORE, D, a,
                          (uint32_t)l.items, (uint32_t)l.joins, st);
    }
  }
  return hipSuccess;
}

}  // namespace
}  // namespace cra

using namespace cra;

extern "C" {

size_t cra_fwd_paged_workspace_bytes(const cra_cache* c, const cra_batch* b, const cra_paged_plan* p) {
  if (check_paged(c, b, p)) return 0;
  return plan_launch(c, b, p).bytes();
}

int cra_fwd_paged(const cra_cache* c, const cra_batch* b, const cra_paged_plan* p, cra_tensor q,
                  cra_tensor o, void* workspace, size_t workspace_bytes, void* stream) {
  if (int e = check_paged(c, b, p)) return e;
  const int vec = c->dtype == CRA_F32 ? 4 : 8;
  for (const cra_tensor* t : {&q, &o}) {
    if (!t->ptr) return err(CRA_E_INVALID, "q or o is NULL");
    if (reinterpret_cast<uintptr_t>(t->ptr) % 16 || t->sb % vec || t->sh % vec || t->ss % vec)
      return err(CRA_E_LAYOUT, "rows of q and o must be 16-byte aligned");
  }
  const Launch l = plan_launch(c, b, p);
  const size_t need = l.bytes();
  if (need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16))
    return err(CRA_E_INVALID, "workspace: NULL or misaligned pointer");
  if (workspace_bytes < need) {
    char msg[96];
    snprintf(msg, sizeof(msg), "workspace holds %zu bytes, %zu needed", workspace_bytes, need);
    return err(CRA_E_WORKSPACE, msg);
  }
  const int64_t bh = (int64_t)b->n_seqs * c->H_kv;
  const int64_t most = std::max({bh * l.sel_steps, bh * l.part_rows, l.items});
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
  hipStream_t st = (hipStream_t)stream;
  if (l.list) {
    a.d_steps = fast_div(l.sel_steps);
    const uint32_t grid = (uint32_t)(bh * l.sel_steps);
    auto kernel = l.wide ? (p->top_k <= 2 ? select_wide_kernel<2> : select_wide_kernel<4>)
                         : select_kernel;
    kernel<<<grid, 64 * kSelWaves, 0, st>>>(a, l.sel_steps);
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

}  // extern "C"
