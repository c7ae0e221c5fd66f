// Steps over one K/V tile in LDS for tiles of many rows over a paged cache (16-bit
// compute): scores, exponentials, P.V, and a row at a time where elements are not finite.
#pragma once

#include <type_traits>

#include "cra_paged_dev.hpp"

namespace cra {
namespace {

// Steps by which operand reads run ahead of their MFMAs: one less for 8-bit stores at
// D = 128, whose scales and widening need the registers (a spilled one would wait
// for the next tile's loads).
template <int D, int STORE>
constexpr int kAhead = D == 128 && STORE != kSame ? 2 : CRA_FWD_PF;

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

// One 32-key half: scores (8-bit: times the rows' scales) and exponentials against
// the running maximum, which is raised where they call for it.
template <typename T, int STORE, int D, int BN, int QB, bool MASK>
__device__ __forceinline__ void chunk_softmax(f32x4 (&s)[2][QB], const float* ks, int kc,
                                              f32x4 (&acc)[D / 16][QB], float (&m_run)[QB],
                                              float (&l_run)[QB], float c2, int g,
                                              const TileMask<QB>& mk, const Frag<T>& one,
                                              Frag<T> (&pf)[QB]) {
  if constexpr (STORE != kSame) scale_scores<QB>(s, ks, kc, g);
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
}

// int8 codes are exact in 16 bits, times their scale they are not, so the scale of V's rows
// goes with P, one rounding for both: all of it (bf16), or (fp16, whose range P would leave)
// its significand, the codes standing in the tile times its power of two.
template <typename T>
__device__ __forceinline__ float scale_of_codes(float s) {
  return std::is_same<T, bf16>::value ? 1.f : __uint_as_float(__float_as_uint(s) & 0x7f800000u);
}
template <typename T>
__device__ __forceinline__ float scale_of_p(float s) {
  return std::is_same<T, bf16>::value ? s : __uint_as_float((__float_as_uint(s) & 0x7fffffu) | 0x3f800000u);
}
template <typename T, int QB>
__device__ __forceinline__ void scale_p(const f32x4 (&s)[2][QB], const float* vs, int kc, int g, float c2,
                                        const float (&m_run)[QB], Frag<T> (&pf)[QB]) {
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const float m = m_run[qb] == -kInf ? 0.f : m_run[qb];
    float pv[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(vs + 32 * kc + 16 * h + 4 * g);
#pragma unroll
      for (int r = 0; r < 4; ++r) pv[4 * h + r] = __builtin_amdgcn_exp2f(fmaf(s[h][qb][r], c2, -m)) * scale_of_p<T>(v[r]);
    }
    pf[qb] = pack8<T>(pv);
  }
}

// A tile's halves kc0 .. kc1. VS: V's scales (vs) come in with P.
template <typename T, int STORE, int D, int BN, int QB, bool MASK, bool VS = false>
__device__ __forceinline__ void attend_chunk(const char* tK, const char* tV, const float* ks,
                                             const LaneOffs<D>& lo, const Frag<T> (&qf)[QB][D / 32],
                                             f32x4 (&acc)[D / 16][QB], float (&m_run)[QB],
                                             float (&l_run)[QB], float c2, int g,
                                             const TileMask<QB>& mk, const Frag<T>& one, int kc0, int kc1,
                                             const float* vs = nullptr) {
  // (a loop over the halves would hold the accumulators twice, for its copies)
#pragma unroll
  for (int kc = 0; kc < BN / 32; ++kc) {
    if (kc < kc0 || kc > kc1) continue;
    f32x4 s[2][QB];
    Frag<T> pf[QB];
    tile_scores<T, D, BN, QB, kAhead<D, STORE>>(tK, lo, qf, kc, s);
    chunk_softmax<T, STORE, D, BN, QB, MASK>(s, ks, kc, acc, m_run, l_run, c2, g, mk, one, pf);
    if constexpr (VS) scale_p<T, QB>(s, vs, kc, g, c2, m_run, pf);
    pv_half<T, D, BN, QB, kAhead<D, STORE>>(tV, kc, lo, pf, acc);
  }
}

// Both halves of a tile that every row sees: the second half's scores stand beside
// the first one's exponentials, the first one's P.V beside the second's.
template <typename T, int STORE, int D, int BN, int QB, bool VS = false>
__device__ __forceinline__ void attend_whole(const char* tK, const char* tV, const float* ks,
                                             const LaneOffs<D>& lo, const Frag<T> (&qf)[QB][D / 32],
                                             f32x4 (&acc)[D / 16][QB], float (&m_run)[QB],
                                             float (&l_run)[QB], float c2, int g,
                                             const TileMask<QB>& mk, const Frag<T>& one,
                                             const float* vs = nullptr) {
  static_assert(BN == 64, "two halves");
  f32x4 s0[2][QB], s1[2][QB];
  Frag<T> p0[QB], p1[QB];
  tile_scores<T, D, BN, QB, kAhead<D, STORE>>(tK, lo, qf, 0, s0);
  if constexpr (STORE != kSame) scale_scores<QB>(s0, ks, 0, g);
  float ps[QB];
  bool high = false;
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    half_exp<T, false, QB>(s0, 0, qb, c2, m_run[qb], g, mk, one, p0[qb], ps[qb]);
    high |= !(ps[qb] <= kSumMax);
  }
  tile_scores<T, D, BN, QB, kAhead<D, STORE>>(tK, lo, qf, 1, s1);
  if (__any(high)) {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
      if (__any(!(ps[qb] <= kSumMax)))
        half_rescale<T, D, QB>(s0, qb, c2, acc, m_run, l_run, one, p0[qb], ps[qb]);
  }
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) l_run[qb] += ps[qb];
  if constexpr (STORE != kSame) scale_scores<QB>(s1, ks, 1, g);
  high = false;
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    half_exp<T, false, QB>(s1, 1, qb, c2, m_run[qb], g, mk, one, p1[qb], ps[qb]);
    high |= !(ps[qb] <= kSumMax);
  }
  if constexpr (VS) scale_p<T, QB>(s0, vs, 0, g, c2, m_run, p0);
  pv_half<T, D, BN, QB, kAhead<D, STORE>>(tV, 0, lo, p0, acc);
  if (__any(high)) {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
      if (__any(!(ps[qb] <= kSumMax)))
        half_rescale<T, D, QB>(s1, qb, c2, acc, m_run, l_run, one, p1[qb], ps[qb]);
  }
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) l_run[qb] += ps[qb];
  if constexpr (VS) scale_p<T, QB>(s1, vs, 1, g, c2, m_run, p1);
  pv_half<T, D, BN, QB, kAhead<D, STORE>>(tV, 1, lo, p1, acc);
}

// Key tiles of a row tile: nglob tiles of global rows (rpb a block of W; by their places
// in `list` where there is more than one), then nloc of the rows from lo on, from the
// highest down.
struct KeyTiles {
  const int32_t* pages;
  const uint32_t* list;
  int hk, W, rpb, nglob, nloc, lo;
};

// One query row over the keys of its piece, in fp32, touching only the rows it
// sees (the first `glen` global rows, and rows `first` to `last`): for rows whose tiles
// hold elements that are not finite. A lane takes a key of the tile for the scores,
// D / 64 columns (or one, below 64) for P.V. The result goes to o, or unfinished to
// part and (m, l).
template <typename T, int STORE, int D, int BN>
__device__ __forceinline__ void careful_row(const PagedArgs& a, const KeyTiles& k, const T* q, int glen,
                                            int first, int last, int t_first, int ntot, bool bad,
                                            float* part, float* part_ml, T* o) {
  constexpr int kCols = D > 64 ? D / 64 : 1;
  const int lane = threadIdx.x & 63;
  const int row_bytes = a.Ds * (STORE == kSame ? 2 : 1);
  auto element = [&](const char* base, uint32_t slot, int col) -> float {
    const int64_t at = (int64_t)slot * row_bytes;
    if constexpr (STORE == kSame)
      return to_f32(reinterpret_cast<const T*>(base + at)[col]);
    else
      return code_value<STORE>((uint32_t)(uint8_t)base[at + col], 0);
  };
  float m = -kInf, l = 0.f, acc[kCols];
#pragma unroll
  for (int c = 0; c < kCols; ++c) acc[c] = 0.f;
#pragma unroll 1
  for (int it = t_first; it < ntot; ++it) {
    const bool loc = it >= k.nglob;
    const int ts = loc ? k.lo + (k.nloc - 1 - (it - k.nglob)) * BN : it * BN;
    const bool sees = lane < BN && (loc ? ts + lane >= first && ts + lane <= last : ts + lane < glen);
    const uint64_t seen = __ballot(sees);
    if (!seen) continue;
    uint32_t slot = 0;
    if (sees) {
      if (!loc && k.rpb > 1)
        slot = k.list[ts + lane];
      else
        slot = seq_row(k.pages, loc ? ts + lane : (ts + lane) * k.W, a.c.num_pages, a.c.H_kv, a.c.log_page, k.hk);
      if (slot == kNoRow) slot = 0;  // the caller's `bad`
    }
    float x = 0.f;
    if (sees) {
#pragma unroll 1
      for (int c = 0; c < a.D; c += 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x += element(a.c.k, slot, c + i) * to_f32(q[c + i]);
      }
    }
    if constexpr (STORE != kSame) x *= sees ? a.c.k_scale[slot] : 0.f;
    x = sees ? x * (a.scale * kLog2e) : -kInf;
    float mx = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const float y = __shfl_xor(mx, o);
      mx = mx > y || mx != mx ? mx : y;  // NaN stays
    }
    const float m_new = m != m || mx != mx ? __builtin_nanf("") : fmaxf(m, mx);
    const float mu = m_new == -kInf ? 0.f : m_new;
    const float alpha = m == -kInf ? 0.f : __builtin_amdgcn_exp2f(m - mu);
    float e = sees ? __builtin_amdgcn_exp2f(x - mu) : 0.f, sum = e;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
    l = l * alpha + sum;
    if constexpr (STORE != kSame) e *= sees ? a.c.v_scale[slot] : 0.f;
    m = m_new;
#pragma unroll
    for (int c = 0; c < kCols; ++c) acc[c] *= alpha;
#pragma unroll 1
    for (int j = 0; j < BN; j += 8) {
      if (!(seen >> j & 0xff)) continue;
      float v[8][kCols];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t sl = (uint32_t)__shfl((int)slot, j + i);  // a valid row where it is not seen
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          const int col = lane * kCols + c;
          v[i][c] = col < a.D ? element(a.c.v, sl, col) : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float ej = __shfl(e, j + i);
        if (seen >> (j + i) & 1) {
#pragma unroll
          for (int c = 0; c < kCols; ++c) acc[c] += ej * v[i][c];
        }
      }
    }
  }
  if (bad) l = __builtin_nanf("");
  if (part) {
#pragma unroll
    for (int c = 0; c < kCols; ++c)
      if (lane * kCols + c < D) part[lane * kCols + c] = acc[c];
    if (lane == 0) {
      part_ml[0] = m;
      part_ml[1] = l;
    }
  } else {
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int c = 0; c < kCols; ++c)
      if (lane * kCols + c < a.D) o[lane * kCols + c] = from_f32<T>(acc[c] * inv);
  }
}

}  // namespace
}  // namespace cra
