// Device-side pieces shared by the kernels over a paged cache: a call's arguments,
// its sequences, wave-wide scans, 8-bit operands, and products with rows that a
// query does not see.
#pragma once

#include <type_traits>

#include "cra_common.hpp"
#include "cra_internal.hpp"
#include "cra_paged.hpp"
#include "cra_tile.hpp"

namespace cra {

constexpr float kInf = __builtin_huge_valf();
constexpr int kFewRows = 16;  // rows of few_kernel's MFMA block
constexpr int kChunkItems = 1024;  // pieces that chunk_kernel aims at: two rounds of resident workgroups
enum { kSame = CRA_STORE_SAME, kE4M3 = CRA_STORE_E4M3, kInt8 = CRA_STORE_INT8 };

struct PagedArgs {
  PagedView c;
  const void* q;
  void* o;
  int64_t qsb, qsh, qss, osb, osh, oss;
  int Hq, grp, D, Ds;  // query heads, per kv head; columns of q and o; of a cache row
  int window, relay, top_k, max_len;
  float scale;
  FastDiv d_grp, d_hkv, d_steps;
  uint32_t* list;  // [n_seqs, H_kv, list_cap] cache rows of the global rows (relay)
  int list_cap;
  float* part;     // few rows: O of shared sequences' pieces, [piece, part_rows, Dp], and (m, l)
  float* part_ml;
  int32_t* pieces;  // [n_seqs + 1] first piece of each sequence (a kv head), for combine_kernel
  int part_rows, few_grid;
  int parts;       // pieces of cut sequences (all kv heads) that the workspace holds
  int few_only;    // no chunk_kernel follows: longer sequences are refused (NaN)
  int zero_outside;  // rows of tokens outside every sequence are set to zero
};

// A sequence of the call: length, new tokens, and where they lie in q and o.
struct Seq {
  int n, m, qb, q0;
  bool over;  // longer than the caller's bound, or than its table: nothing is read
};
__device__ __forceinline__ Seq get_seq(const PagedArgs& a, int b) {
  Seq s;
  const int len = a.c.lens[b];
  s.over = len > a.max_len;
  s.n = s.over || len < 0 ? 0 : len;
  if (a.c.cu) {
    const TokenRange t = token_range(a.c.cu, b, a.c.tokens);
    s.m = t.last - t.first;
    s.qb = 0;
    s.q0 = t.first;
  } else {
    s.m = a.c.query_len;
    s.qb = b;
    s.q0 = 0;
  }
  return s;
}

// The sequence of a whole wave: its numbers in scalar registers (they are loaded
// with vector loads, and what is formed of them would stay in vector registers).
__device__ __forceinline__ Seq wave_seq(const PagedArgs& a, int b) {
  Seq s = get_seq(a, __builtin_amdgcn_readfirstlane(b));
  s.n = __builtin_amdgcn_readfirstlane(s.n);
  s.m = __builtin_amdgcn_readfirstlane(s.m);
  s.q0 = __builtin_amdgcn_readfirstlane(s.q0);
  s.qb = __builtin_amdgcn_readfirstlane(s.qb);
  s.over = __builtin_amdgcn_readfirstlane(s.over);
  return s;
}

__device__ __forceinline__ SeqPlan get_plan(const PagedArgs& a, int n) {
  return seq_plan(n, a.window, a.relay, a.top_k);
}

// Row r of a kv head's rows is query head r % grp of the kv head, new token r / grp.
__device__ __forceinline__ int row_token(const PagedArgs& a, int r) { return (int)div_by(r, a.d_grp); }

template <typename T>
__device__ __forceinline__ const T* q_row(const PagedArgs& a, const Seq& s, int hk, int r) {
  const int t = row_token(a, r);
  return static_cast<const T*>(a.q) + s.qb * a.qsb + (int64_t)(hk * a.grp + r - t * a.grp) * a.qsh +
         (int64_t)(s.q0 + t) * a.qss;
}
template <typename T>
__device__ __forceinline__ T* o_row(const PagedArgs& a, const Seq& s, int hk, int r) {
  const int t = row_token(a, r);
  return static_cast<T*>(a.o) + s.qb * a.osb + (int64_t)(hk * a.grp + r - t * a.grp) * a.osh +
         (int64_t)(s.q0 + t) * a.oss;
}

// Maximum over the wave, and sums up to each lane, by row shifts and broadcasts in
// the VALU (lanes without a source take 0).
#define CRA_DPP(x, ctrl, rows) (uint32_t) __builtin_amdgcn_update_dpp(0, (int)(x), ctrl, rows, 0xf, false)
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  x = max(x, CRA_DPP(x, 0x111, 0xf));  // row_shr:1, 2, 4, 8: the row's last lane has its maximum
  x = max(x, CRA_DPP(x, 0x112, 0xf));
  x = max(x, CRA_DPP(x, 0x114, 0xf));
  x = max(x, CRA_DPP(x, 0x118, 0xf));
  x = max(x, CRA_DPP(x, 0x142, 0xf));  // row_bcast:15, row_bcast:31
  x = max(x, CRA_DPP(x, 0x143, 0xf));
  return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}
__device__ __forceinline__ uint32_t wave_upto(uint32_t x) {
  x += CRA_DPP(x, 0x111, 0xf);
  x += CRA_DPP(x, 0x112, 0xf);
  x += CRA_DPP(x, 0x114, 0xf);
  x += CRA_DPP(x, 0x118, 0xf);
  x += CRA_DPP(x, 0x142, 0xa);  // the row before, into rows 1 and 3
  x += CRA_DPP(x, 0x143, 0xc);  // the half before, into rows 2 and 3
  return x;
}

// ---------------------------------------------------------------------------
// 8-bit codes to operands of a 2-byte type (exact for both stores).
// ---------------------------------------------------------------------------
template <typename T, int STORE>
__device__ __forceinline__ uint2 widen4(uint32_t w) {  // four codes -> four elements
  uint2 r;
  if constexpr (STORE == kE4M3) {
    if constexpr (std::is_same<T, bf16>::value) {
      r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.f, false));
      r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.f, true));
    } else {
      r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.f, false));
      r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.f, true));
    }
  } else {
    typedef T t2 __attribute__((ext_vector_type(2)));
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (float)(int8_t)(w >> (8 * i) & 0xffu);
    r.x = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{f[0], f[1]}, t2));
    r.y = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{f[2], f[3]}, t2));
  }
  return r;
}
template <int STORE>
__device__ __forceinline__ float code_value(uint32_t w, int i) {  // code i of four, i constant
  if constexpr (STORE == kE4M3) {
    switch (i) {
      case 0: return __builtin_amdgcn_cvt_f32_fp8((int)w, 0);
      case 1: return __builtin_amdgcn_cvt_f32_fp8((int)w, 1);
      case 2: return __builtin_amdgcn_cvt_f32_fp8((int)w, 2);
      default: return __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
    }
  } else {
    return (float)(int8_t)(w >> (8 * i) & 0xffu);
  }
}

template <typename T>
__device__ __forceinline__ Frag<T> zero_frag() {
  Frag<T> f;
  f.w[0] = make_uint4(0, 0, 0, 0);
  return f;
}

// Whether a lane of the wave holds an operand element that is not finite (or
// elements whose sum leaves fp32), from their sum over the tile's rows and columns.
__device__ __forceinline__ bool any_not_finite(f32x4 sum) {
  const float z = (sum[0] - sum[0]) + (sum[1] - sum[1]) + (sum[2] - sum[2]) + (sum[3] - sum[3]);
  return __any(!(z == 0.f));
}

// O^T += scale V^T . P^T where rows that not every query sees hold elements that
// are not finite (0 times them would be NaN). The product takes V with those
// elements set to zero; which queries see one is counted by products of
// indicators (of +inf, -inf and NaN in V, and of the rows that a query sees),
// and their sums become what such a row makes of them. v(db): the V operand of
// 16-column block db; row of slot s of lane group g: k0 + 4g + s (s < 4),
// k0 + 16 + 4g + s - 4.
template <typename T, int NDB, int QB, typename V>
__device__ __forceinline__ void pv_not_finite(V v, const Frag<T> (&pf)[QB], f32x4 (&acc)[NDB][QB],
                                              const TileMask<QB>& mk, int k0, int g, float scale) {
  constexpr uint32_t kExp = std::is_same<T, bf16>::value ? 0x7f80u : 0x7c00u;
  constexpr uint32_t kOne = std::is_same<T, bf16>::value ? 0x3f80u : 0x3c00u;
  const f32x4 zero = f32x4{0.f, 0.f, 0.f, 0.f};
  Frag<T> sees[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = k0 + (i < 2 ? 0 : 16) + 4 * g + 2 * (i & 1);
      reinterpret_cast<uint32_t*>(sees[qb].w)[i] = (mk.ok(row, qb) ? kOne : 0u) |
                                                   (mk.ok(row + 1, qb) ? kOne << 16 : 0u);
    }
#pragma unroll
  for (int db = 0; db < NDB; ++db) {
    Frag<T> f[4];  // V without them; +inf, -inf, NaN
    f[0] = v(db);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = reinterpret_cast<const uint32_t*>(f[0].w)[i];
      uint32_t o[4] = {0, 0, 0, 0};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t x = w >> (16 * h) & 0xffffu, mag = x & 0x7fffu;
        o[0] |= (mag < kExp ? x : 0u) << (16 * h);
        o[1] |= (x == kExp ? kOne : 0u) << (16 * h);
        o[2] |= (x == (kExp | 0x8000u) ? kOne : 0u) << (16 * h);
        o[3] |= (mag > kExp ? kOne : 0u) << (16 * h);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) reinterpret_cast<uint32_t*>(f[j].w)[i] = o[j];
    }
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const f32x4 o = mma(zero, f[0], pf[qb]) * scale;
      const f32x4 pos = mma(zero, f[1], sees[qb]), neg = mma(zero, f[2], sees[qb]);
      const f32x4 nan = mma(zero, f[3], sees[qb]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float x = o[r];
        if (pos[r] > 0.f) x += kInf;
        if (neg[r] > 0.f) x -= kInf;
        if (nan[r] > 0.f) x = __builtin_nanf("");
        acc[db][qb][r] += x;
      }
    }
  }
}

// All of the wave's loads have landed (in LDS too) and its LDS reads are done; no
// memory access moves across.
__device__ __forceinline__ void wait_all() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }

// ---------------------------------------------------------------------------
// Work of the chunk kernels: tiles of BM rows of a (sequence, kv head), each over
// its BN-key tiles. Where a sequence's key range is at least twice its share (the
// call's key tiles over kChunkItems) it is cut into pieces of equal length, whose
// results join_chunk adds up: a short chunk behind a long context under a wide
// window would otherwise leave most of the chip idle. The scan is every wave's
// own, 64 sequences at a time.
// ---------------------------------------------------------------------------
struct ChunkSeq {
  int tiles, nk;  // row tiles; key tiles of any of them, at most
};
template <int BM, int BN>
__device__ __forceinline__ ChunkSeq chunk_seq(const PagedArgs& a, int b) {
  const Seq s = get_seq(a, b);
  const int64_t rows = (int64_t)s.m * a.grp;
  if (rows <= kFewRows) return ChunkSeq{0, 0};
  return ChunkSeq{(int)((rows + BM - 1) / BM), chunk_tile_count(s.n, BM / a.grp + 2, BN, get_plan(a, s.n))};
}

struct ChunkFind {
  int b, j;             // sequence (-1: none), and the index within its items
  int tiles, pieces, len;  // its row tiles, pieces of each, key tiles a piece
  int split0;           // items of cut sequences before it
};
// Item `idx` of all items (JOIN: of the cut sequences' row tiles).
template <int BM, int BN, bool JOIN>
__device__ __forceinline__ ChunkFind chunk_find(const PagedArgs& a, int idx) {
  const int lane = threadIdx.x & 63;
  auto load = [&](int base) {
    return base + lane < a.c.n_seqs ? chunk_seq<BM, BN>(a, base + lane) : ChunkSeq{0, 0};
  };
  const ChunkSeq c0 = load(0);
  uint64_t total = 0;
  for (int base = 0; base < a.c.n_seqs; base += 64) {
    const ChunkSeq c = base == 0 ? c0 : load(base);
    const uint64_t all = (uint64_t)c.tiles * c.nk;  // below 2^50: summed in halves of 25 bits
    total += (uint32_t)__builtin_amdgcn_readlane((int)wave_upto((uint32_t)(all & 0x1ffffffu)), 63);
    total += (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)wave_upto((uint32_t)(all >> 25)), 63) << 25;
  }
  const uint64_t share = (total * a.c.H_kv + kChunkItems - 1) / kChunkItems;
  const int per = (int)(share < 8 ? 8 : share < (1u << 30) ? share : 1u << 30);
  int before = 0, split0 = 0;
  for (int base = 0; base < a.c.n_seqs; base += 64) {
    const ChunkSeq c = base == 0 ? c0 : load(base);
    const int pieces = max(1, c.nk / per), cut = pieces > 1 ? c.tiles * pieces : 0;
    const int n = JOIN ? (pieces > 1 ? c.tiles : 0) : c.tiles * pieces;
    const int upto = before + (int)wave_upto(n), cuts = split0 + (int)wave_upto(cut);
    const uint64_t hit = __ballot(upto > idx);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
      ChunkFind f;
      f.b = base + l;
      f.j = idx - (of(upto) - of(n));
      f.tiles = of(c.tiles);
      f.pieces = of(pieces);
      f.len = (of(c.nk) + f.pieces - 1) / f.pieces;
      f.split0 = of(cuts) - of(cut);
      return f;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
    split0 = __builtin_amdgcn_readlane(cuts, 63);
  }
  return ChunkFind{-1, 0, 0, 0, 0, 0};
}

struct ChunkWork {
  int b, hk, tile;     // sequence (-1: none), kv head, row tile
  int t_first, t_end;  // key tiles
  int64_t part;        // partial row of the tile's first row, or -1: the result is whole
};
// Tiles of a sequence's last tokens (the longest ranges) come first;
// neighbouring workgroups take other heads, and so other XCDs.
template <int BM, int BN>
__device__ __forceinline__ ChunkWork chunk_work(const PagedArgs& a) {
  const uint32_t item = div_by(blockIdx.x, a.d_hkv);
  ChunkWork w{};
  w.hk = (int)(blockIdx.x - item * a.c.H_kv);
  const ChunkFind f = chunk_find<BM, BN, false>(a, (int)item);
  w.b = f.b;
  if (f.b < 0) return w;
  // offsets of tokens that run backwards may give more pieces than the call's
  // tokens can have
  if (f.pieces > 1 && (int64_t)(f.split0 + f.j + 1) * a.c.H_kv > a.parts) w.b = -1;
  const int t = f.j / f.pieces, piece = f.j - t * f.pieces;
  w.tile = f.tiles - 1 - t;
  w.t_first = f.pieces > 1 ? piece * f.len : 0;
  w.t_end = f.pieces > 1 ? w.t_first + f.len : 0x7fffffff;
  w.part = f.pieces > 1 ? ((int64_t)(f.split0 + f.j) * a.c.H_kv + w.hk) * BM : -1;
  return w;
}

// Adds the pieces of cut sequences' row tiles up: `items` of join_rows(D) rows each
// over the grid's stride, a thread four columns of a row. One pass over the pieces
// with a running maximum, eight pieces' loads on their way: a chunk of 32 rows behind
// 26000 dense keys has 51 pieces 20 us (32 rows a workgroup, the maximum first:
// 83); where nothing was cut the launch costs 4.7 us.
constexpr int kJoinGrid = 1024;  // workgroups at most: calls without cut sequences pass through quickly
template <int D>
__host__ __device__ constexpr int join_rows() { return 1024 / D; }
template <typename T, int BM, int BN, int D>
__device__ void join_chunk(const PagedArgs& a, uint32_t items) {
  constexpr int R = join_rows<D>(), kParts = BM / R;
  const int r0 = threadIdx.x / (D / 4), c = threadIdx.x % (D / 4) * 4;
  for (uint32_t v = blockIdx.x; v < items; v += gridDim.x) {
    const uint32_t block = v / kParts, item = div_by(block, a.d_hkv);
    const int hk = (int)(block - item * a.c.H_kv);
    const ChunkFind f = chunk_find<BM, BN, true>(a, (int)item);
    if (f.b < 0 || (int64_t)(f.split0 + (f.j + 1) * f.pieces) * a.c.H_kv > a.parts) return;
    const Seq s = wave_seq(a, f.b);
    const int r = (int)(v % kParts) * R + r0, row = (f.tiles - 1 - f.j) * BM + r;
    if (row >= s.m * a.grp || c >= a.D) continue;
    const int64_t first = ((int64_t)(f.split0 + f.j * f.pieces) * a.c.H_kv + hk) * BM + r;
    const int64_t step = (int64_t)a.c.H_kv * BM;  // partial rows from piece to piece
    float M = -kInf, L = 0.f;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < f.pieces; k += 8) {
      float2 ml[8];
      f32x4 x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t at = first + min(k + i, f.pieces - 1) * step;
        ml[i] = *reinterpret_cast<const float2*>(a.part_ml + 2 * at);
        x[i] = *reinterpret_cast<const f32x4*>(a.part + at * D + c);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (k + i >= f.pieces) break;
        const float m = fmaxf(M, ml[i].x), mu = m == -kInf ? 0.f : m;
        const float e = __builtin_amdgcn_exp2f(M - mu), en = __builtin_amdgcn_exp2f(ml[i].x - mu);
        L = L * e + ml[i].y * en;
        o = o * e + x[i] * en;
        M = m;
      }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    T* op = o_row<T>(a, s, hk, row) + c;
#pragma unroll
    for (int j = 0; j < 4; ++j) op[j] = from_f32<T>(o[j] * inv);
  }
}

// chunk_kernel and the joining of its pieces (cra_paged_chunk.hip): grid
// workgroups, at most join_tiles (sequence, tile, kv head)s of several pieces.
hipError_t launch_chunk(int dtype, int store, int Dp, const PagedArgs& a, uint32_t grid,
                        uint32_t join_tiles, hipStream_t st);

}  // namespace cra
