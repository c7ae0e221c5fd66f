// Steps of the 16-bit forward over one K/V tile in LDS: scores, exponentials
// against a lazily raised maximum, P.V. Shared by the kernels over whole
// sequences (cra_fwd.hip) and over a paged cache (cra_paged.hip).
#pragma once

#include <type_traits>

#include "cra_common.hpp"

namespace cra {

// MFMA steps by which the forward's LDS operand reads run ahead of their use
// (K row fragments and transposed V fragments). Three measured 0.6% faster
// than two and four no better than two (D = 128: 242, 238 and 246 VGPRs, 2
// waves per SIMD either way; D = 64 stays at 168, 3 waves per SIMD).
#ifndef CRA_FWD_PF
#define CRA_FWD_PF 3
#endif

template <typename T, int D, int BN, int QB, int AHEAD = CRA_FWD_PF>
__device__ __forceinline__ void tile_scores(const char* tK, const LaneOffs<D>& lo,
                                            const Frag<T> (&qf)[QB][D / 32], int kc,
                                            f32x4 (&s)[2][QB]) {
  using Tile = SwzTile<D, BN>;
  constexpr int NC = D / 32, NK = 2 * NC;
  // K fragments are read AHEAD steps ahead of the MFMAs that use them; fences
  // keep the compiler from moving the reads next to their uses. Step t takes
  // key block t % 2 and D-chunk t / 2, so the four accumulators alternate and
  // each MFMA's accumulator was last written four MFMAs earlier (key block
  // major, two apart, measured 0.5% slower).
  auto k_frag = [&](int t) {
    return Tile::template row_frag_at<T>(tK + (2 * kc + t % 2) * Tile::kBlk16 + lo.row_at(t / 2));
  };
  constexpr int PF = AHEAD < NK ? AHEAD : NK;
  Frag<T> kf[PF + 1];
#pragma unroll
  for (int t = 0; t < PF; ++t) kf[t] = k_frag(t);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int t = 0; t < NK; ++t) {
    if (t + PF < NK) kf[(t + PF) % (PF + 1)] = k_frag(t + PF);
    const int h = t % 2, c = t / 2;
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      if (c == 0) s[h][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
      s[h][qb] = mma(s[h][qb], kf[t % (PF + 1)], qf[qb][c]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// O^T += V^T . P^T for 32-key half kh: transposed V fragments read
// AHEAD steps ahead of the MFMAs that use them.
template <typename T, int D, int BN, int QB, int AHEAD = CRA_FWD_PF>
__device__ __forceinline__ void pv_half(const char* tV, int kh, const LaneOffs<D>& lo,
                                        const Frag<T> (&pf)[QB], f32x4 (&acc)[D / 16][QB]) {
  using Tile = SwzTile<D, BN>;
  constexpr int NDB = D / 16;
  auto tr_v = [&](int db) {
    const char* pa = tV + (2 * kh) * Tile::kBlk16 + lo.tr_at(db);
    return Tile::template tr_frag_at<T>(pa, pa + Tile::kBlk16);
  };
  constexpr int PF = AHEAD < NDB ? AHEAD : NDB;
  Frag<T> vt[PF + 1];
#pragma unroll
  for (int db = 0; db < PF; ++db) vt[db] = tr_v(db);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int db = 0; db < NDB; ++db) {
    if (db + PF < NDB) vt[(db + PF) % (PF + 1)] = tr_v(db + PF);
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) acc[db][qb] = mma(acc[db][qb], vt[db % (PF + 1)], pf[qb]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Largest sum of a half's 32 rounded exponentials accepted against the
// running maximum: each term is then at most 2^15 and finite in fp16.
constexpr float kSumMax = 32768.f;

// All-ones A operand: ones . P^T puts the sum over the 32 keys of each query
// (column of P^T) in all four of that query's lanes' result rows.
template <typename T>
__device__ __forceinline__ Frag<T> ones_frag() {
  Frag<T> f;
  const uint32_t w = sizeof(T) == 2 ? (std::is_same<T, bf16>::value ? 0x3f803f80u : 0x3c003c00u)
                                    : 0u;
  f.w[0] = make_uint4(w, w, w, w);
  return f;
}

// Sum of the rounded P of a 32-key half for each query, on the matrix core
// (one MFMA in place of four v_dot2 per lane plus a cross-lane sum).
template <typename T>
__device__ __forceinline__ float half_sum(const Frag<T>& pk, const Frag<T>& one) {
  return mma(f32x4{0.f, 0.f, 0.f, 0.f}, one, pk)[0];
}

// Exponentials of one 32-key half (8 per lane and query block) against the
// running maximum, rounded to the input type, and the sum of the rounded
// values over the half's 32 keys (the P.V operand and its normaliser).
template <typename T, bool MASK, int QB>
__device__ __forceinline__ void half_exp(f32x4 (&s)[2][QB], int kc, int qb, float c2, float m,
                                         int g, const TileMask<QB>& mk, const Frag<T>& one,
                                         Frag<T>& pk, float& ps) {
  float pv[8];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (MASK && !mk.ok(32 * kc + 16 * h + 4 * g + r, qb)) s[h][qb][r] = -__builtin_huge_valf();
      pv[4 * h + r] = __builtin_amdgcn_exp2f(fmaf(s[h][qb][r], c2, -m));
    }
  pk = pack8<T>(pv);
  ps = half_sum(pk, one);
}

// Raise the running maximum of query block qb to this half's maximum,
// rescale its accumulators and redo the half's exponentials. Taken for the
// first visible keys and whenever a score exceeds the running maximum by
// enough to push a sum of 8 rounded terms past kSumMax (inf and NaN sums
// included).
template <typename T, int D, int QB>
__device__ __forceinline__ void half_rescale(f32x4 (&s)[2][QB], int qb, float c2,
                                             f32x4 (&acc)[D / 16][QB], float (&m_run)[QB],
                                             float (&l_run)[QB], const Frag<T>& one, Frag<T>& pk,
                                             float& ps) {
  float mx = -__builtin_huge_valf();
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[h][qb][r]);
  const float m_new = fmaxf(m_run[qb], group_max(mx * c2));
  // Until a query's first visible key its accumulators and l are zero; the
  // whole wave's first rescale (its first tile) has nothing to scale.
  if (!__all(m_run[qb] == -__builtin_huge_valf())) {
    const float alpha =
        m_run[qb] == -__builtin_huge_valf() ? 0.f : __builtin_amdgcn_exp2f(m_run[qb] - m_new);
    l_run[qb] *= alpha;
#pragma unroll
    for (int db = 0; db < D / 16; ++db) acc[db][qb] *= alpha;
  }
  m_run[qb] = m_new;
  const float mu = m_new == -__builtin_huge_valf() ? 0.f : m_new;
  float pv[8];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int r = 0; r < 4; ++r) pv[4 * h + r] = __builtin_amdgcn_exp2f(fmaf(s[h][qb][r], c2, -mu));
  pk = pack8<T>(pv);
  ps = half_sum(pk, one);
}

}  // namespace cra
