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
// its waves and workgroups splitting the keys, joined by combine_kernel;
// chunk_kernel takes the others in tiles of 128 rows, the rows of a kv head's
// query heads side by side so that a K/V tile serves them all. fp32 runs
// f32_kernel for both.
//
// A row that a query does not see never reaches its result, whatever it holds
// (NaN and infinity included): masked scores are replaced, and where a tile that
// not every query sees holds such values P.V is formed apart from them
// (pv_not_finite). A query that sees no row gives zeros.
#include <stdio.h>

#include <algorithm>
#include <type_traits>

#include "cra_common.hpp"
#include "cra_internal.hpp"
#include "cra_paged.hpp"
#include "cra_tile.hpp"

namespace cra {

int set_error(int code, const char* msg);

namespace {

constexpr float kInf = __builtin_huge_valf();
constexpr int kFewRows = 16;  // rows of few_kernel's MFMA block
enum { kSame = CRA_STORE_SAME, kE4M3 = CRA_STORE_E4M3, kInt8 = CRA_STORE_INT8 };

struct PagedArgs {
  PagedView c;
  const void* q;
  void* o;
  int64_t qsb, qsh, qss, osb, osh, oss;
  int Hq, grp, D, Ds;  // query heads, per kv head; columns of q and o; of a cache row
  int window, relay, top_k, max_len;
  float scale;
  FastDiv d_grp, d_hkv, d_splits;
  uint32_t* list;  // [n_seqs, H_kv, list_cap] cache rows of the global rows (relay)
  int list_cap;
  float* part;     // few_kernel, splits > 1: [n_seqs, H_kv, splits, part_rows, Dp], then (m, l)
  float* part_ml;
  int splits, part_rows;
  int few_only;    // no chunk_kernel follows: longer sequences are refused (NaN)
  int tiles;       // chunk tiles of a sequence (batches without cu)
  FastDiv d_tiles;
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

// ---------------------------------------------------------------------------
// The global rows of sequences with relay, as cache rows. One wave a W-block:
// its strided row, and behind it (blocks that end before the last query's
// window) the top_k rows of largest norm, of equals the earlier; a slot without
// a row left is the block's first row, as in the packed rows of whole
// sequences. NaN norms are never chosen.
// ---------------------------------------------------------------------------
constexpr int kSelWaves = 4;

__device__ __forceinline__ uint64_t wave_max(uint64_t x) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const uint32_t lo = __shfl_xor((uint32_t)x, o), hi = __shfl_xor((uint32_t)(x >> 32), o);
    const uint64_t y = (uint64_t)hi << 32 | lo;
    x = y > x ? y : x;
  }
  return x;
}

__global__ __launch_bounds__(64 * kSelWaves) void select_kernel(PagedArgs a, int steps) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t bh = div_by(blockIdx.x, a.d_splits);  // d_splits: blocks a (sequence, head)
  const int first = (int)(blockIdx.x - bh * steps) * kSelWaves + wave;
  const int b = (int)div_by(bh, a.d_hkv), h = (int)(bh - (uint32_t)b * a.c.H_kv);
  const Seq s = get_seq(a, b);
  const SeqPlan p = get_plan(a, s.n);
  if (p.rpb == 1 || s.m < 1) return;
  const int ls = s.n - p.W > 0 ? s.n - p.W : 0;  // window start of the last query
  const int full = ls / p.W, blocks = full + (ls != full * p.W ? 1 : 0);
  const int32_t* pages = a.c.table + b * a.c.table_stride;
  uint32_t* out = a.list + (int64_t)bh * a.list_cap;
  auto row_at = [&](int row) {
    return seq_row(pages, row, a.c.num_pages, a.c.H_kv, a.c.log_page, h);
  };
  for (int r = first; r < blocks; r += steps * kSelWaves) {
    const int row0 = r * p.W;
    uint32_t mine = kNoRow;  // lane j: list entry j of the block
    if (lane == 0) mine = row_at(row0);
    if (r < full) {
      // each lane keeps the top four of its rows (which rise)
      uint64_t key[4] = {0, 0, 0, 0};
      bool bad = false;
      constexpr int kU = 4;
      for (int base = 0; base < p.W; base += 64 * kU) {
        uint32_t at[kU];
        float x[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u)
          at[u] = row_at(row0 + min(base + 64 * u + lane, p.W - 1));
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          bad |= at[u] == kNoRow;
          x[u] = at[u] == kNoRow ? 0.f : a.c.k_norm[at[u]];
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const int i = base + 64 * u + lane;
          if (i >= p.W || !(x[u] >= 0.f)) continue;
          uint64_t k = (uint64_t)(__float_as_uint(x[u]) | 0x80000000u) << 32 | (uint32_t)~(uint32_t)i;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint64_t old = key[j];
            key[j] = k > old ? k : old;
            k = k > old ? old : k;
          }
        }
      }
      const bool any_bad = __any(bad);
      for (int j = 0; j < a.top_k; ++j) {
        const uint64_t m = wave_max(key[0]);
        const int i = m ? (int)~(uint32_t)m : 0;
        if (m && key[0] == m) {  // keys differ in their rows: one lane has it
          key[0] = key[1];
          key[1] = key[2];
          key[2] = key[3];
          key[3] = 0;
        }
        if (lane == 1 + j) mine = any_bad ? kNoRow : row_at(row0 + i);
      }
    }
    if (lane < (r < full ? p.rpb : 1)) out[(int64_t)p.rpb * r + lane] = mine;
  }
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
    const uint32_t u = w ^ 0x80808080u;
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (float)(u >> (8 * i) & 0xffu) - 128.f;
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

// ---------------------------------------------------------------------------
// Few rows: at most 16 rows a (sequence, kv head). Each wave takes whole 32-key
// tiles of its own, filled with per-lane addresses straight into its part of
// LDS (a row of a page is contiguous, rows lie anywhere), two stages deep, with
// no barrier until the end; the 16-column operand Q^T holds the rows. Bound by
// memory: the rows seen, once per kv head. The waves' results, and those of the
// `splits` workgroups that share a sequence's keys, are joined by their maxima.
// ---------------------------------------------------------------------------
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

constexpr int kFewWaves = 4;
template <int D, int STORE>
constexpr int kFewStages = D * (STORE == kSame ? 2 : 1) > 256 ? 1 : 2;

// All of the wave's loads have landed (in LDS too) and its LDS reads are done; no
// memory access moves across.
__device__ __forceinline__ void wait_all() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }

template <typename T, int STORE, int D>
__global__ __launch_bounds__(64 * kFewWaves) void few_kernel(PagedArgs a) {
  constexpr int NW = kFewWaves, NS = kFewStages<D, STORE>;
  constexpr int ES = STORE == kSame ? 2 : 1;
  using Tile = ByteTile<D * ES, 32>;
  // the stages as objects of their own, so that reads of one do not wait for the fill of the other
  __shared__ __attribute__((aligned(1024))) char stage0[NW][2][Tile::kBytes];
  __shared__ __attribute__((aligned(1024))) char stage1[NS == 2 ? NW : 1][2][NS == 2 ? Tile::kBytes : 16];
  __shared__ float scales[NW][64];
  __shared__ float join_ml[NW][kFewRows][2];

  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t bh = div_by(blockIdx.x, a.d_splits);
  const int split = (int)(blockIdx.x - bh * a.splits);
  const int b = (int)div_by(bh, a.d_hkv), hk = (int)(bh - (uint32_t)b * a.c.H_kv);
  const Seq s = get_seq(a, b);
  const int64_t rows64 = (int64_t)s.m * a.grp;
  if (rows64 == 0) return;
  if (rows64 > a.part_rows) {  // kFewRows, or fewer by the caller's bound
    if (a.few_only && split == 0)  // more new tokens than the caller's bound
      for (int64_t i = tid; i < rows64 * a.D; i += 64 * NW) {
        const int r = (int)(i / a.D);
        o_row<T>(a, s, hk, r)[i - (int64_t)r * a.D] = from_f32<T>(__builtin_nanf(""));
      }
    return;
  }
  const int rows = (int)rows64;
  const SeqPlan p = get_plan(a, s.n);
  const int pos0 = s.n - s.m;  // of the first new token
  const int G = s.n > 0 ? seq_prefix(s.n - 1, p) : 0;
  const int lo = max(0, max(pos0, 0) - p.W + 1);
  const int nG = (G + 31) >> 5, nT = nG + ((s.n - lo + 31) >> 5);
  const int32_t* pages = a.c.table + b * a.c.table_stride;
  const uint32_t* list = a.list + (int64_t)bh * a.list_cap;
  bool bad = s.over;

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
  const int row_bytes = a.Ds * ES;
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

  const int step = a.splits * NW;
  int it = split * NW + wave;
  if (D * ES > row_bytes) {  // columns that no load fills
    for (int i = lane; i < 2 * Tile::kBytes / 16; i += 64) {
      reinterpret_cast<uint4*>(stage0[wave])[i] = make_uint4(0, 0, 0, 0);
      if constexpr (NS == 2) reinterpret_cast<uint4*>(stage1[wave])[i] = make_uint4(0, 0, 0, 0);
    }
    wait_all();  // before loads to the same memory
  }
  float sc = 0.f;
  uint32_t next = 0;
  if (it < nT) {
    const uint32_t first = checked(slot_of(it));
    fill(stage0[wave], first);
    sc = load_scale(first);
    if (it + step < nT) next = slot_of(it + step);
  }

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
    float vref = 1.f;
    if constexpr (STORE != kSame && std::is_same<T, f16>::value) {
      // p times a row's scale would leave fp16's range: it is taken relative to
      // the tile's largest scale, which multiplies the product in fp32
      float most = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) most = fmaxf(most, vs[i]);
      vref = group_max(most);
      vref = vref > 0.f ? vref : 1.f;
    }
    float pv[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      pv[i] = __builtin_amdgcn_exp2f(x[i] - mu);
      l_run += pv[i];
    }
    if constexpr (STORE != kSame) {
      const float inv = std::is_same<T, f16>::value ? 1.f / vref : 1.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) pv[i] = x[i] == -kInf ? 0.f : pv[i] * (vs[i] * inv);
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
    // one new token: every row of the tile, a repeated last one too, is a row that its query sees
    const bool full = s.m == 1 || (loc ? ts >= s.n - p.W && ts + 31 <= pos0 : ts + 32 <= glen0);
    if (!full) {
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
  auto turn = [&](auto second) __attribute__((always_inline)) {
    constexpr bool kSecond = decltype(second)::value && NS == 2;
    wait_all();
    const float sc_now = sc;
    const bool more = it + step < nT;
    auto refill = [&](char (&dst)[2][Tile::kBytes]) {
      const uint32_t slot = checked(next);
      fill(dst, slot);
      sc = load_scale(slot);
      if (it + 2 * step < nT) next = slot_of(it + 2 * step);
    };
    if constexpr (NS == 2) {
      if constexpr (kSecond) {
        if (more) refill(stage0[wave]);
        attend(stage1[wave], it, sc_now);
      } else {
        if (more) refill(stage1[wave]);
        attend(stage0[wave], it, sc_now);
      }
    } else {
      attend(stage0[wave], it, sc_now);
      wait_all();
      if (more) refill(stage0[wave]);
    }
    it += step;
  };
  while (it < nT) {
    turn(std::false_type{});
    if (it < nT) turn(std::true_type{});
  }

  // join the waves
  l_run = group_sum(l_run);
  if (__any(bad)) l_run = __builtin_nanf("");
  __syncthreads();
  // the tiles' memory holds the waves' O now: [wave][row][D], quads swizzled by row
  static_assert(sizeof(float) * NW * kFewRows * D <= sizeof(stage0), "join area");
  f32x4* join_o = reinterpret_cast<f32x4*>(&stage0[0][0][0]);
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
    if (a.splits == 1) {
      if (c >= a.D) continue;
      const float inv = L == 0.f ? 0.f : 1.f / L;
      T e[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) e[j] = from_f32<T>(o[j] * inv);
      *reinterpret_cast<uint2*>(o_row<T>(a, s, hk, r) + c) = *reinterpret_cast<const uint2*>(e);
    } else {
      const int64_t at = ((int64_t)bh * a.splits + split) * a.part_rows + r;
      *reinterpret_cast<f32x4*>(a.part + at * D + c) = o;
      if (c == 0) {
        a.part_ml[2 * at] = M;
        a.part_ml[2 * at + 1] = L;
      }
    }
  }
}

// Joins the splits of few rows: one workgroup a (sequence, kv head, row).
template <typename T>
__global__ __launch_bounds__(256) void combine_kernel(PagedArgs a, int Dp) {
  __shared__ float red[256][4];
  __shared__ float red_l[64];
  const int tid = threadIdx.x;
  const int r = blockIdx.x % a.part_rows;
  const uint32_t bh = blockIdx.x / a.part_rows;
  const int b = (int)div_by(bh, a.d_hkv), hk = (int)(bh - (uint32_t)b * a.c.H_kv);
  const Seq s = get_seq(a, b);
  const int64_t rows = (int64_t)s.m * a.grp;
  if (rows > a.part_rows || r >= rows) return;
  const int quads = Dp / 4, lanes = 256 / quads;  // split groups
  const int quad = tid % quads, sg = tid / quads;
  const float* ml = a.part_ml + 2 * ((int64_t)bh * a.splits * a.part_rows + r);
  const float* po = a.part + ((int64_t)bh * a.splits * a.part_rows + r) * Dp + quad * 4;
  float M = -kInf;
  for (int i = 0; i < a.splits; ++i) M = fmaxf(M, ml[(int64_t)2 * i * a.part_rows]);
  float L = 0.f;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int i = sg; i < a.splits; i += lanes) {
    const float mi = ml[(int64_t)2 * i * a.part_rows];
    const float e = mi == -kInf ? 0.f : __builtin_amdgcn_exp2f(mi - M);
    L += e * ml[(int64_t)2 * i * a.part_rows + 1];
    o += *reinterpret_cast<const f32x4*>(po + (int64_t)i * a.part_rows * Dp) * e;
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
// Chunks: tiles of 128 (D = 256: 64) rows of a (sequence, kv head), four waves.
// ---------------------------------------------------------------------------
// The work item of a workgroup: sequence and tile, tiles of a sequence's last
// tokens (the longest ranges) first; -1: none. With cu every wave adds up the
// sequences' tiles, 64 at a time.
template <int BM>
__device__ __forceinline__ void find_tile(const PagedArgs& a, int item, int& b, int& tile) {
  if (!a.c.cu) {
    b = (int)div_by(item, a.d_tiles);
    tile = a.tiles - 1 - (item - b * a.tiles);
    return;
  }
  const int lane = threadIdx.x & 63;
  int before = 0;
  b = -1;
  for (int base = 0; base < a.c.n_seqs; base += 64) {
    int count = 0;
    if (base + lane < a.c.n_seqs) {
      const TokenRange t = token_range(a.c.cu, base + lane, a.c.tokens);
      const int64_t rows = (int64_t)(t.last - t.first) * a.grp;
      count = rows > kFewRows ? (int)((rows + BM - 1) / BM) : 0;
    }
    int upto = count;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(upto, o);
      if (lane >= o) upto += x;
    }
    const uint64_t hit = __ballot(before + upto > item);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      const int end = before + __shfl(upto, l);
      b = base + l;
      tile = end - 1 - item;
      return;
    }
    before += __shfl(upto, 63);
  }
}

// P.V of a 32-row half that not all of the wave's queries see.
template <typename T, int D, int BN, int QB>
__device__ __forceinline__ void pv_half_masked(const char* tV, int kh, const LaneOffs<D>& lo,
                                               const Frag<T> (&pf)[QB], f32x4 (&acc)[D / 16][QB],
                                               const TileMask<QB>& mk, const Frag<T>& one, int g) {
  using Tile = SwzTile<D, BN>;
  auto v_frag = [&](int db) __attribute__((always_inline)) {
    const char* pa = tV + 2 * kh * Tile::kBlk16 + lo.tr_at(db);
    return Tile::template tr_frag_at<T>(pa, pa + Tile::kBlk16);
  };
  f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int db = 0; db < D / 16; ++db) sum = mma(sum, v_frag(db), one);
  if (any_not_finite(sum))
    pv_not_finite<T, D / 16, QB>(v_frag, pf, acc, mk, 32 * kh, g, 1.f);
  else
    pv_half<T, D, BN, QB>(tV, kh, lo, pf, acc);
}

// Scores of 8-bit keys: the rows' scales (LDS) come in here, exactly as fp32.
template <int QB>
__device__ __forceinline__ void scale_scores(f32x4 (&s)[2][QB], const float* ks, int kc, int g) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f32x4 k = *reinterpret_cast<const f32x4*>(ks + 32 * kc + 16 * h + 4 * g);
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) s[h][qb] *= k;
  }
}

template <typename T, int STORE, int D, int BN, int QB, bool MASK>
__device__ __forceinline__ void attend_chunk(const char* tK, const char* tV, const float* ks,
                                             const LaneOffs<D>& lo, const Frag<T> (&qf)[QB][D / 32],
                                             f32x4 (&acc)[D / 16][QB], float (&m_run)[QB],
                                             float (&l_run)[QB], float c2, int g,
                                             const TileMask<QB>& mk, const Frag<T>& one,
                                             int kc0, int kc1) {
#pragma unroll
  for (int kc = 0; kc < BN / 32; ++kc) {
    if (MASK && (kc < kc0 || kc > kc1)) continue;  // no row of this half is seen
    f32x4 s[2][QB];
    tile_scores<T, D, BN, QB>(tK, lo, qf, kc, s);
    if constexpr (STORE != kSame) scale_scores<QB>(s, ks, kc, g);
    Frag<T> pf[QB];
    float ps[QB];
    bool high = false;
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      half_exp<T, MASK, QB>(s, kc, qb, c2, m_run[qb], g, mk, one, pf[qb], ps[qb]);
      high |= !(ps[qb] <= kSumMax);
    }
    if (__any(high)) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
        if (__any(!(ps[qb] <= kSumMax)))
          half_rescale<T, D, QB>(s, qb, c2, acc, m_run, l_run, one, pf[qb], ps[qb]);
    }
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) l_run[qb] += ps[qb];
    if constexpr (MASK)
      pv_half_masked<T, D, BN, QB>(tV, kc, lo, pf, acc, mk, one, g);
    else
      pv_half<T, D, BN, QB>(tV, kc, lo, pf, acc);
  }
}

template <int D>
constexpr int kChunkQB = D > 128 ? 1 : 2;
template <int D>
constexpr int kChunkBN = D > 128 ? 32 : 64;
constexpr int kChunkWaves = 4;

template <typename T, int STORE, int D>
__global__ __launch_bounds__(64 * kChunkWaves) __attribute__((amdgpu_waves_per_eu(2)))
void chunk_kernel(PagedArgs a) {
  constexpr int NW = kChunkWaves, QB = kChunkQB<D>, BN = kChunkBN<D>, kQW = 16 * QB, BM = NW * kQW;
  using Tile = SwzTile<D, BN>;
  __shared__ __attribute__((aligned(1024))) char stage0[2][Tile::kBytes];
  __shared__ __attribute__((aligned(1024))) char stage1[2][Tile::kBytes];
  __shared__ __attribute__((aligned(16))) float kscale[2][BN];

  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) & (NW - 1);
  const uint32_t item = div_by(blockIdx.x, a.d_hkv);
  const int hk = (int)(blockIdx.x - item * a.c.H_kv);  // neighbouring workgroups: another head, another XCD
  int b, tile;
  find_tile<BM>(a, (int)item, b, tile);
  if (b < 0) return;
  const Seq s = get_seq(a, b);
  const int rows = s.m * a.grp;
  if (rows <= kFewRows || tile * BM >= rows) return;
  const SeqPlan p = get_plan(a, s.n);
  const int pos0 = s.n - s.m;
  const int r0 = tile * BM, q0 = r0 + wave * kQW;
  auto pos_of = [&](int r) { return pos0 + row_token(a, r); };
  const int wg_first = pos_of(r0), wg_last = pos_of(min(r0 + BM, rows) - 1);
  const int lo_k = max(0, wg_first - p.W + 1), hi = max(0, wg_last + 1);
  const int gmax = seq_prefix(wg_last, p);
  const int nglob = (gmax + BN - 1) / BN, nloc = (hi - lo_k + BN - 1) / BN;
  const int ntot = nglob + (hi > lo_k ? nloc : 0);
  const int32_t* pages = a.c.table + b * a.c.table_stride;
  const uint32_t* list = a.list + ((int64_t)b * a.c.H_kv + hk) * a.list_cap;
  bool bad = s.over;

  // global tiles first, then the window from its highest tile down
  auto tile_start = [&](int it) {
    return it >= nglob ? lo_k + (nloc - 1 - (it - nglob)) * BN : it * BN;
  };
  auto slot_of = [&](int it, int row) -> uint32_t {
    const int ts = tile_start(it);
    if (it < nglob) {
      const int i = min(ts + row, gmax - 1);
      if (p.rpb > 1) return list[i];
      return seq_row(pages, i * p.W, a.c.num_pages, a.c.H_kv, a.c.log_page, hk);
    }
    return seq_row(pages, min(ts + row, hi - 1), a.c.num_pages, a.c.H_kv, a.c.log_page, hk);
  };

  // Rows of a tile that this thread fills. 16-bit: the wave's instruction t
  // moves 1 KB, each lane one 16-byte chunk from its own address straight into
  // LDS. 8-bit: pieces of 16 codes through registers, widened on the way (V
  // times its scale: one more rounding; K's scales go to the scores).
  constexpr int kPiecesRow = STORE == kSame ? Tile::kCPR : D / 16;
  constexpr int kAll = BN * kPiecesRow, kPer = (kAll + 64 * NW - 1) / (64 * NW);
  const int row_bytes = a.Ds * (STORE == kSame ? 2 : 1);
  auto piece_of = [&](int i) { return STORE == kSame ? (i * NW + wave) * 64 + lane : i * 64 * NW + tid; };
  uint32_t slot[kPer];
  auto load_slots = [&](int it) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) slot[i] = slot_of(it, min(piece_of(i), kAll - 1) / kPiecesRow);
  };
  uint4 rk[STORE == kSame ? 1 : kPer], rv[STORE == kSame ? 1 : kPer];
  float rks[STORE == kSame ? 1 : kPer], rvs[STORE == kSame ? 1 : kPer];
  auto issue = [&](char (&dst)[2][Tile::kBytes]) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int piece = piece_of(i), row = piece / kPiecesRow;
      if (kAll % (64 * NW) != 0 && piece >= kAll) break;
      bad |= slot[i] == kNoRow;
      const uint32_t sl = slot[i] == kNoRow ? 0u : slot[i];
      const int col = piece % kPiecesRow;
      if constexpr (STORE == kSame) {
        const int chunk = col ^ Tile::swz(row);
        const int64_t at = (int64_t)sl * row_bytes + chunk * 16;
        if (D * 2 == row_bytes || chunk * 16 < row_bytes) {
          const int lds = (i * NW + wave) * 1024;
          __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(a.c.k + at),
                                           CRA_LDS(dst[0] + lds), 16, 0, 0);
          __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(a.c.v + at),
                                           CRA_LDS(dst[1] + lds), 16, 0, 0);
        }
      } else {
        const int64_t at = (int64_t)sl * row_bytes + col * 16;
        const bool in = col * 16 < row_bytes;
        rk[i] = in ? *reinterpret_cast<const uint4*>(a.c.k + at) : make_uint4(0, 0, 0, 0);
        rv[i] = in ? *reinterpret_cast<const uint4*>(a.c.v + at) : make_uint4(0, 0, 0, 0);
        rks[i] = a.c.k_scale[sl];
        rvs[i] = a.c.v_scale[sl];
      }
    }
  };
  auto store = [&](char (&dst)[2][Tile::kBytes], float (&ks)[BN]) {
    if constexpr (STORE != kSame) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int piece = piece_of(i), row = piece / kPiecesRow, col = piece % kPiecesRow;
        if (kAll % (64 * NW) != 0 && piece >= kAll) break;
        const uint32_t* wk = reinterpret_cast<const uint32_t*>(&rk[i]);
        const uint32_t* wv = reinterpret_cast<const uint32_t*>(&rv[i]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint2 x = widen4<T, STORE>(wk[2 * h]), y = widen4<T, STORE>(wk[2 * h + 1]);
          *reinterpret_cast<uint4*>(dst[0] + Tile::off(row, 2 * col + h)) = make_uint4(x.x, x.y, y.x, y.y);
          float f[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = code_value<STORE>(wv[2 * h + j / 4], j % 4) * rvs[i];
          *reinterpret_cast<uint4*>(dst[1] + Tile::off(row, 2 * col + h)) = pack8<T>(f).w[0];
        }
        if (col == 0) ks[row] = rks[i];
      }
    }
  };
  if (STORE == kSame && D * 2 > row_bytes) {  // columns that no load fills
    for (int i = tid; i < 2 * Tile::kBytes / 16; i += 64 * NW) {
      reinterpret_cast<uint4*>(stage0)[i] = make_uint4(0, 0, 0, 0);
      reinterpret_cast<uint4*>(stage1)[i] = make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
  }
  if (ntot > 0) {
    load_slots(0);
    issue(stage0);
    store(stage0, kscale[0]);
    if (ntot > 1) load_slots(1);
  }

  LaneOffs<D> lo;
  lo.init(lane);
  Frag<T> qf[QB][D / 32];
  int pos[QB], glen[QB];
  bool counts[QB];
  float m_run[QB], l_run[QB];
  f32x4 acc[D / 16][QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int r = q0 + 16 * qb + l16;
    counts[qb] = r < rows;
    pos[qb] = counts[qb] ? pos_of(r) : -1;
    glen[qb] = pos[qb] >= 0 ? seq_prefix(pos[qb], p) : 0;
    const T* qp = q_row<T>(a, s, hk, counts[qb] ? r : 0);
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
      qf[qb][c] = counts[qb] && 32 * c + 8 * g < a.D ? lds_frag_row<T>(qp + 32 * c + 8 * g) : zero_frag<T>();
    m_run[qb] = -kInf;
    l_run[qb] = 0.f;
#pragma unroll
    for (int db = 0; db < D / 16; ++db) acc[db][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float c2 = a.scale * kLog2e;
  const bool active = q0 < rows;
  const int first = active ? pos_of(q0) : 0;  // positions of the wave's rows: [first, last]
  const int last = active ? pos_of(min(q0 + kQW, rows) - 1) : -1;
  const int w_lo = max(0, first - p.W + 1);
  const int g_all = active ? seq_prefix(first, p) : 0, g_any = active ? seq_prefix(last, p) : 0;
  const Frag<T> one = ones_frag<T>();

  auto turn = [&](auto second, int it) __attribute__((always_inline)) {
    constexpr int kS = decltype(second)::value;
    char(&cur)[2][Tile::kBytes] = kS ? stage1 : stage0;
    char(&nxt)[2][Tile::kBytes] = kS ? stage0 : stage1;
    if (STORE == kSame) wait_vmem();
    __syncthreads();
    if (it + 1 < ntot) {
      issue(nxt);
      if (it + 2 < ntot) load_slots(it + 2);
    }
    const bool loc = it >= nglob;
    const int ts = tile_start(it);
    const bool work = active && (loc ? ts <= last && ts + BN - 1 >= w_lo : ts < g_any);
    if (work) {
      const bool full = loc ? ts >= last - p.W + 1 && ts + BN - 1 <= first : ts + BN <= g_all;
      TileMask<QB> mk;
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        mk.hi[qb] = loc ? pos[qb] - ts : glen[qb] - 1 - ts;
        mk.span[qb] = loc ? (unsigned)(p.W - 1) : 0x7fffffffu;
      }
      if (full) {
        attend_chunk<T, STORE, D, BN, QB, false>(cur[0], cur[1], kscale[kS], lo, qf, acc, m_run, l_run,
                                                 c2, g, mk, one, 0, 0);
      } else {
        const int vis_lo = loc ? max(0, w_lo - ts) : 0, vis_hi = loc ? last - ts : g_any - 1 - ts;
        attend_chunk<T, STORE, D, BN, QB, true>(cur[0], cur[1], kscale[kS], lo, qf, acc, m_run, l_run,
                                                c2, g, mk, one, vis_lo >> 5, vis_hi >> 5);
      }
    }
    if (it + 1 < ntot) store(nxt, kscale[1 - kS]);
  };
  for (int it = 0; it < ntot; it += 2) {
    turn(std::integral_constant<int, 0>{}, it);
    if (it + 1 < ntot) turn(std::integral_constant<int, 1>{}, it + 1);
  }

  bad = __syncthreads_or(bad);
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    if (!counts[qb]) continue;
    const float l = l_run[qb];
    const float inv = bad ? __builtin_nanf("") : l == 0.f ? 0.f : 1.f / l;
    T* op = o_row<T>(a, s, hk, q0 + 16 * qb + l16);
#pragma unroll
    for (int db = 0; db < D / 16; ++db) {
      if (16 * db + 4 * g >= a.D) continue;
      T e[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) e[r] = from_f32<T>(acc[db][qb][r] * inv);
      *reinterpret_cast<uint2*>(op + 16 * db + 4 * g) = *reinterpret_cast<const uint2*>(e);
    }
  }
}

// ---------------------------------------------------------------------------
// fp32: tiles of 64 rows, 32 keys at a time as fp32 in LDS (8-bit codes times
// their scale), v_mfma_f32_16x16x4_f32. FEW: at most 16 rows and a share of
// the key tiles (splits), else a chunk tile.
// ---------------------------------------------------------------------------
__device__ __forceinline__ f32x4 mma4(f32x4 c, float x, float y) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(x, y, c, 0, 0, 0);
}

constexpr int kF32Rows = 64, kF32Keys = 32;

template <int STORE, int D, bool FEW>
__global__ __launch_bounds__(256) void f32_kernel(PagedArgs a) {
  constexpr int BN = kF32Keys, kStride = D + 4;
  __shared__ __attribute__((aligned(16))) float tK[BN][kStride];
  __shared__ __attribute__((aligned(16))) float tV[BN][kStride];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, g = lane >> 4;
  int b, tile = 0, hk, split = 0, nsplit = 1;
  if constexpr (FEW) {
    const uint32_t bh = div_by(blockIdx.x, a.d_splits);
    split = (int)(blockIdx.x - bh * a.splits);
    nsplit = a.splits;
    b = (int)div_by(bh, a.d_hkv);
    hk = (int)(bh - (uint32_t)b * a.c.H_kv);
  } else {
    const uint32_t item = div_by(blockIdx.x, a.d_hkv);
    hk = (int)(blockIdx.x - item * a.c.H_kv);
    find_tile<kF32Rows>(a, (int)item, b, tile);
    if (b < 0) return;
  }
  const Seq s = get_seq(a, b);
  const int64_t rows64 = (int64_t)s.m * a.grp;
  if (rows64 == 0) return;
  if (FEW && rows64 > a.part_rows) {
    if (a.few_only && split == 0)
      for (int64_t i = tid; i < rows64 * a.D; i += 256) {
        const int r = (int)(i / a.D);
        o_row<float>(a, s, hk, r)[i - (int64_t)r * a.D] = __builtin_nanf("");
      }
    return;
  }
  const int rows = (int)rows64;
  if (!FEW && (rows <= kFewRows || tile * kF32Rows >= rows)) return;
  const SeqPlan p = get_plan(a, s.n);
  const int pos0 = s.n - s.m, r0 = tile * kF32Rows, q0 = r0 + 16 * wave;
  auto pos_of = [&](int r) { return pos0 + row_token(a, r); };
  const int wg_first = pos_of(r0), wg_last = pos_of(min(r0 + kF32Rows, rows) - 1);
  const int lo_k = max(0, wg_first - p.W + 1), hi = max(0, wg_last + 1);
  const int gmax = seq_prefix(wg_last, p);
  const int nglob = (gmax + BN - 1) / BN, ntot = nglob + (hi > lo_k ? (hi - lo_k + BN - 1) / BN : 0);
  const int32_t* pages = a.c.table + b * a.c.table_stride;
  const uint32_t* list = a.list + ((int64_t)b * a.c.H_kv + hk) * a.list_cap;
  bool bad = s.over;

  // 16 threads a row pair: thread's row tid / 8, D / 8 columns each
  constexpr int kCols = D / 8;  // columns of a thread, 4 at a time
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
  if (split < ntot) load(split);

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

  for (int it = split; it < ntot; it += nsplit) {
    __syncthreads();  // every wave is done with the previous tile
    store();
    __syncthreads();
    if (it + nsplit < ntot) load(it + nsplit);
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
  if (!FEW || nsplit == 1) {
    const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
    float* op = o_row<float>(a, s, hk, r);
#pragma unroll
    for (int db = 0; db < D / 16; ++db)
      if (16 * db + 4 * g < a.D) *reinterpret_cast<f32x4*>(op + 16 * db + 4 * g) = acc[db] * inv;
  } else {
    const int64_t at = (((int64_t)b * a.c.H_kv + hk) * a.splits + split) * a.part_rows + r;
#pragma unroll
    for (int db = 0; db < D / 16; ++db)
      *reinterpret_cast<f32x4*>(a.part + at * D + 16 * db + 4 * g) = acc[db];
    if (g == 0) {
      a.part_ml[2 * at] = m_run;
      a.part_ml[2 * at + 1] = l_run;
    }
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
  bool list;
  int64_t list_cap;
  int sel_steps;          // select workgroups a (sequence, head)
  int splits, part_rows;
  int64_t tiles;          // chunk workgroups a kv head
  int tiles_seq;          // of a sequence (batches without cu)
  size_t list_bytes, part_bytes, ml_bytes;
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
  const SeqPlan sp = seq_plan(l.max_len, p->window, p->relay, p->top_k);
  const int64_t blocks = (std::max(0, l.max_len - sp.W) + (int64_t)sp.W - 1) / sp.W;
  // shorter sequences have no more blocks under a fixed window, and at most
  // ceil(sqrt(max_len)) under the rule
  const int64_t cap = p->window > 0 ? blocks : ceil_sqrt(l.max_len);
  l.list = sp.rpb > 1 && cap > 0;
  l.list_cap = l.list ? cap * sp.rpb : 0;
  l.sel_steps = (int)std::min<int64_t>((cap + kSelWaves - 1) / kSelWaves, 4096);
  const int64_t bh = (int64_t)b->n_seqs * c->H_kv;
  l.list_bytes = up256(bh * l.list_cap * 4);
  // few rows: about two workgroups a CU, each wave with at least one tile
  const int64_t keys = blocks * sp.rpb + std::min<int64_t>((int64_t)sp.W + kFewRows, l.max_len);
  const int64_t tiles = (keys + 31) / 32 + 1;
  const int64_t share = f32 ? tiles : (tiles + 3) / 4;
  l.splits = (int)std::max<int64_t>(1, std::min<int64_t>((2 * 256 + bh - 1) / bh, share));
  if (!l.few) l.splits = 1;
  l.part_rows = (int)std::min<int64_t>(kFewRows, most_rows);
  if (l.splits > 1) {
    l.part_bytes = up256(bh * l.splits * l.part_rows * (int64_t)l.Dp * 4);
    l.ml_bytes = up256(bh * l.splits * l.part_rows * 2 * 4);
  }
  const int BM = f32 ? kF32Rows : l.Dp > 128 ? 64 : 128;
  if (b->cu_seqlens) {
    l.tiles = (int64_t)b->tokens * l.grp / BM + b->n_seqs;
  } else {
    l.tiles_seq = (int)((most_rows + BM - 1) / BM);
    l.tiles = (int64_t)l.tiles_seq * b->n_seqs;
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
      f32_kernel<STORE, D, true><<<(uint32_t)(bh * l.splits), 256, 0, st>>>(a);
    else
      few_kernel<T, STORE, D><<<(uint32_t)(bh * l.splits), 64 * kFewWaves, 0, st>>>(a);
    if (hipError_t e = hipGetLastError()) return e;
    if (l.splits > 1) {
      combine_kernel<T><<<(uint32_t)(bh * l.part_rows), 256, 0, st>>>(a, D);
      if (hipError_t e = hipGetLastError()) return e;
    }
  }
  if (l.chunk) {
    const uint32_t grid = (uint32_t)(l.tiles * a.c.H_kv);
    if constexpr (std::is_same<T, float>::value)
      f32_kernel<STORE, D, false><<<grid, 256, 0, st>>>(a);
    else
      chunk_kernel<T, STORE, D><<<grid, 64 * kChunkWaves, 0, st>>>(a);
    return hipGetLastError();
  }
  return hipSuccess;
}

}  // namespace
}  // namespace cra

using namespace cra;

extern "C" {

size_t cra_fwd_paged_workspace_bytes(const cra_cache* c, const cra_batch* b, const cra_paged_plan* p) {
  if (check_paged(c, b, p)) return 0;
  const Launch l = plan_launch(c, b, p);
  return l.list_bytes + l.part_bytes + l.ml_bytes;
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
  const size_t need = l.list_bytes + l.part_bytes + l.ml_bytes;
  if (need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16))
    return err(CRA_E_INVALID, "workspace: NULL or misaligned pointer");
  if (workspace_bytes < need) {
    char msg[96];
    snprintf(msg, sizeof(msg), "workspace holds %zu bytes, %zu needed", workspace_bytes, need);
    return err(CRA_E_WORKSPACE, msg);
  }
  const int64_t bh = (int64_t)b->n_seqs * c->H_kv;
  const int64_t most = std::max({bh * l.sel_steps, bh * l.splits, bh * l.part_rows, l.tiles * c->H_kv});
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
  a.splits = l.splits;
  a.part_rows = l.part_rows;
  a.few_only = !l.chunk;
  a.tiles = l.tiles_seq;
  a.d_tiles = fast_div(std::max(1, l.tiles_seq));
  hipStream_t st = (hipStream_t)stream;
  if (l.list) {
    a.d_splits = fast_div(l.sel_steps);
    select_kernel<<<(uint32_t)(bh * l.sel_steps), 64 * kSelWaves, 0, st>>>(a, l.sel_steps);
    if (int e = hip_err(hipGetLastError(), "cra_fwd_paged (relay rows)")) return e;
  }
  a.d_splits = fast_div(l.splits);
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
