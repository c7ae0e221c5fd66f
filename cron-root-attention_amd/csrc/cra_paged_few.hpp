// Kernels of the paged attention for few rows a (sequence, kv head), with the joining of
// their pieces, and those of fp32. SHARED: the rows of a prefix that the sequences have in
// common are left to prefix kernels (cra_paged_prefix.hip), whose results combine_kernel
// adds.
#pragma once

#include <type_traits>

#include "cra_common.hpp"
#include "cra_internal.hpp"
#include "cra_paged_dev.hpp"

namespace cra {
namespace {

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
template <bool SHARED>
__device__ __forceinline__ FewTiles few_tiles(const PagedArgs& a, int b) {
  const Seq s = get_seq(a, b);
  const int64_t rows = (int64_t)s.m * a.grp;
  // more rows than the caller's bound: one piece, which answers NaN
  if (rows == 0 || (rows > a.part_rows && !a.few_only)) return FewTiles{0, false};
  if (rows > a.part_rows) return FewTiles{0, true};
  const SeqPlan p = get_plan(a, s.n);
  if constexpr (SHARED) {
    const Share sh = share_of(a, prefix_plan(a), s, p);
    return FewTiles{few_tile_count(s.n, s.m, p, sh.P, sh.G0), true};
  }
  return FewTiles{few_tile_count(s.n, s.m, p), true};
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
template <bool SHARED>
__device__ __forceinline__ FewPieces few_pieces(const PagedArgs& a) {
  const int lane = threadIdx.x & 63;
  FewTiles t0{0, false};
  int64_t tiles = 0;
  for (int base = 0; base < a.c.n_seqs; base += 64) {
    FewTiles t{0, false};
    if (base + lane < a.c.n_seqs) t = few_tiles<SHARED>(a, base + lane);
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
      if (base + lane < a.c.n_seqs) t = few_tiles<SHARED>(a, base + lane);
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
template <bool SHARED>
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
    if (base + lane < a.c.n_seqs) t = few_tiles<SHARED>(a, base + lane);
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

template <typename T, int STORE, int D, bool SHARED>
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
  const FewPieces fp = few_pieces<SHARED>(a);
  for (int64_t item = blockIdx.x; item < (int64_t)fp.total * a.c.H_kv; item += gridDim.x) {
  const uint32_t idx = div_by((uint32_t)item, a.d_hkv);
  const int hk = (int)((uint32_t)item - idx * a.c.H_kv);
  const FewPiece fi = few_piece<SHARED>(a, fp, (int)idx);
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
  const Share sh = SHARED ? share_of(a, prefix_plan(a), s, p) : Share{0, 0};
  const int G = s.n > 0 ? seq_prefix(s.n - 1, p) : 0, g0 = min(sh.G0, G);  // global rows g0 .. G - 1
  const int lo = max(sh.P, max(pos0, 0) - p.W + 1);
  const int nG = (G - g0 + 31) >> 5, nAll = nG + ((s.n - lo + 31) >> 5);
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
      const int i = min(g0 + it * 32 + ko, G - 1);
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
    const int ts = loc ? lo + (it - nG) * 32 : g0 + it * 32;
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
    if (fi.only && sh.P == 0) {
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
template <typename T, bool SHARED>
__global__ __launch_bounds__(256) void combine_kernel(int Dp, PagedArgs a) {
  __shared__ float red[256][4];
  __shared__ float red_l[64];
  const int tid = threadIdx.x;
  const int r = blockIdx.x % a.part_rows;
  const uint32_t bh = blockIdx.x / a.part_rows;
  const int b = (int)div_by(bh, a.d_hkv), hk = (int)(bh - (uint32_t)b * a.c.H_kv);
  const int first = a.pieces[b], own = a.pieces[b + 1] - first;
  int n = own, prow = 0, ptiles = 0;  // own pieces, and those of the prefix's rows
  if constexpr (SHARED) {
    prow = a.pinfo[b] + r;
    ptiles = a.pinfo[a.c.n_seqs];
    if (a.pinfo[b] >= 0) n += a.pinfo[a.c.n_seqs + 1];
  }
  if (n < 2) return;
  const Seq s = wave_seq(a, b);
  if (r >= (int64_t)s.m * a.grp) return;
  const int quads = Dp / 4, lanes = 256 / quads;  // groups of pieces
  const int quad = tid % quads, sg = tid / quads;
  auto at = [&](int i) { return ((int64_t)(first + i) * a.c.H_kv + hk) * a.part_rows + r; };
  auto prefix_at = [&](int i) {
    const int tile = prow / a.prefix_rows;
    return ((int64_t)((i - own) * ptiles + tile) * a.c.H_kv + hk) * a.prefix_rows + (prow - tile * a.prefix_rows);
  };
  auto ml_of = [&](int i) {
    return reinterpret_cast<const float2*>(!SHARED || i < own ? a.part_ml + 2 * at(i) : a.ppart_ml + 2 * prefix_at(i));
  };
  auto o_of = [&](int i) {
    return reinterpret_cast<const f32x4*>((!SHARED || i < own ? a.part + at(i) * Dp : a.ppart + prefix_at(i) * Dp) + quad * 4);
  };
  float M = -kInf;  // a lane a piece, each wave for itself
  for (int i = tid & 63; i < n; i += 64) M = fmaxf(M, ml_of(i)->x);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor(M, d));
  float L = 0.f;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = sg; i < n; i += lanes) {
    const float2 ml = *ml_of(i);
    const float e = ml.x == -kInf ? 0.f : __builtin_amdgcn_exp2f(ml.x - M);
    L += e * ml.y;
    o += *o_of(i) * e;
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

// Softmax and P.V of a tile's scores: key ko is seen where (unsigned)(vis - ko) <= span;
// full: all of them by every row.
template <int D>
__device__ __forceinline__ void attend_f32(const f32x4 (&sc)[2], const float (&tV)[kF32Keys][D + 4], int vis,
                                           unsigned span, bool full, bool have, float c2, float& m_run,
                                           float& l_run, f32x4 (&acc)[D / 16]) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
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
          const unsigned sp = (unsigned)__shfl((int)span, qi);
        f32x4 c = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int ko = 16 * (i >> 2) + 4 * g + (i & 3);
          c = mma4(c, (unsigned)(h - ko) <= sp ? v[i] : 0.f, l16 == qi ? x[i] : 0.f);
        }
        if (l16 == qi) t = c;
      }
    }
    acc[db] += t;
  }
}

// One work item: rows r0.. of a (sequence, kv head) over its key tiles from
// t_first up to t_end; the result goes to o, or (part_at >= 0) to the partial rows.
template <int STORE, int D, bool SHARED>
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
  const Share sh = SHARED ? share_of(a, prefix_plan(a), s, p) : Share{0, 0};
  const int lo_k = max(sh.P, wg_first - p.W + 1), hi = max(0, wg_last + 1);
  const int gmax = seq_prefix(wg_last, p), g0 = min(sh.G0, gmax);  // global rows g0 .. gmax - 1
  const int nglob = (gmax - g0 + BN - 1) / BN, ntot = nglob + (hi > lo_k ? (hi - lo_k + BN - 1) / BN : 0);
  const int32_t* pages = a.c.table + b * a.c.table_stride;
  const uint32_t* list = a.list + ((int64_t)b * a.c.H_kv + hk) * a.list_cap;
  bool bad = s.over;

  // eight threads a row, D / 8 columns each: quads of them, 32 columns apart
  constexpr int kCols = D / 8;
  const int frow = tid >> 3, fcol = (tid & 7) * 4;
  f32x4 rk[kCols / 4], rv[kCols / 4];
  auto load = [&](int it) {
    const int ts = it >= nglob ? lo_k + (it - nglob) * BN : g0 + it * BN;
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
    const int ts = loc ? lo_k + (it - nglob) * BN : g0 + it * BN;
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
    attend_f32<D>(sc, tV, vis, span, full, have, c2, m_run, l_run, acc);
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

template <int STORE, int D, bool FEW, bool SHARED>
__global__ __launch_bounds__(256) void f32_kernel(PagedArgs a) {
  if constexpr (FEW) {
    zero_outside<float>(a, 256);
    const FewPieces fp = few_pieces<SHARED>(a);
    for (int64_t item = blockIdx.x; item < (int64_t)fp.total * a.c.H_kv; item += gridDim.x) {
      const uint32_t idx = div_by((uint32_t)item, a.d_hkv);
      const int hk = (int)((uint32_t)item - idx * a.c.H_kv);
      const FewPiece fi = few_piece<SHARED>(a, fp, (int)idx);
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
      const bool whole = !SHARED || share_of(a, prefix_plan(a), s, get_plan(a, s.n)).P == 0;
      f32_item<STORE, D, SHARED>(a, s, fi.b, hk, 0, fi.piece * fp.per, (fi.piece + 1) * fp.per,
                                 fi.only && whole ? -1 : item * a.part_rows);
    }
  } else {
    const ChunkWork w = chunk_work<kF32Rows, kF32Keys>(a);
    if (w.b < 0) return;
    f32_item<STORE, D, false>(a, wave_seq(a, w.b), w.b, w.hk, w.tile * kF32Rows, w.t_first, w.t_end, w.part);
  }
}

template <int D>
__global__ __launch_bounds__(256) void f32_join_kernel(uint32_t items, PagedArgs a) {
  join_chunk<float, kF32Rows, kF32Keys, D>(a, items);
}

}  // namespace
}  // namespace cra
