// Chunks of new tokens over a paged cache, 16-bit compute: tiles of 128 (D = 256: 64)
// rows of a (sequence, kv head) - the kv head's query heads side by side, so that
// a K/V tile serves them all - against 64-key (32-key) tiles.
//
// As in the forward over whole sequences, S^T = K . Q^T keeps a row's softmax
// state in its lanes and O^T = V^T . P^T takes P from the score registers; the
// running maximum is raised lazily and the normaliser sums the rounded P. K/V rows
// are gathered: each lane of a load brings a 16-byte chunk from its own row's page
// straight into LDS (8-bit codes go through registers and are widened on the way).
// The rows' cache rows are looked up a tile ahead of their loads.
//
// Bound by the matrix core, the VALU beside it and the waits between them (two waves
// a SIMD): 8192 new tokens of 131072, 16 heads, D = 128 fp16: a call of 155 us, 608
// TFLOP/s (a large matrix product: 1118); two dense chunks of 1000 and 513 tokens among
// 14 single tokens, 16/4 heads, int8 store: 305 us, about 510 TFLOP/s, widening
// included (codes widened on their way from a second stage of them while the next
// loads ran, two turns unrolled: 310 us, eight registers spilled). The fast loop takes no care of
// elements that are not finite in rows that some queries do not see: 0 times them
// leaves NaN in the result, which is looked for once at the end; a wave that finds
// it computes its rows again one by one, over the keys that each sees (careful_row).
#include <stdio.h>

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

// A tile's halves kc0 .. kc1.
template <typename T, int STORE, int D, int BN, int QB, bool MASK>
__device__ __forceinline__ void attend_chunk(const char* tK, const char* tV, const float* ks,
                                             const LaneOffs<D>& lo, const Frag<T> (&qf)[QB][D / 32],
                                             f32x4 (&acc)[D / 16][QB], float (&m_run)[QB],
                                             float (&l_run)[QB], float c2, int g,
                                             const TileMask<QB>& mk, const Frag<T>& one, int kc0, int kc1) {
  // (a loop over the halves would hold the accumulators twice, for its copies)
#pragma unroll
  for (int kc = 0; kc < BN / 32; ++kc) {
    if (kc < kc0 || kc > kc1) continue;
    f32x4 s[2][QB];
    Frag<T> pf[QB];
    tile_scores<T, D, BN, QB, kAhead<D, STORE>>(tK, lo, qf, kc, s);
    chunk_softmax<T, STORE, D, BN, QB, MASK>(s, ks, kc, acc, m_run, l_run, c2, g, mk, one, pf);
    pv_half<T, D, BN, QB, kAhead<D, STORE>>(tV, kc, lo, pf, acc);
  }
}

// Both halves of a tile that every row sees: the second half's scores stand beside
// the first one's exponentials, the first one's P.V beside the second's.
template <typename T, int STORE, int D, int BN, int QB>
__device__ __forceinline__ void attend_whole(const char* tK, const char* tV, const float* ks,
                                             const LaneOffs<D>& lo, const Frag<T> (&qf)[QB][D / 32],
                                             f32x4 (&acc)[D / 16][QB], float (&m_run)[QB],
                                             float (&l_run)[QB], float c2, int g,
                                             const TileMask<QB>& mk, const Frag<T>& one) {
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
  pv_half<T, D, BN, QB, kAhead<D, STORE>>(tV, 0, lo, p0, acc);
  if (__any(high)) {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
      if (__any(!(ps[qb] <= kSumMax)))
        half_rescale<T, D, QB>(s1, qb, c2, acc, m_run, l_run, one, p1[qb], ps[qb]);
  }
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) l_run[qb] += ps[qb];
  pv_half<T, D, BN, QB, kAhead<D, STORE>>(tV, 1, lo, p1, acc);
}

// One query row over the keys of its piece, in fp32, touching only the rows it
// sees: for rows whose tiles hold elements that are not finite. A lane takes a key
// of the tile for the scores, D / 64 columns (or one, below 64) for P.V.
template <typename T, int STORE, int D, int BN>
__device__ __forceinline__ void careful_row(const PagedArgs& a, const Seq& s, const SeqPlan& p, int b,
                                            int hk, int r, int pos, int t_first, int ntot, int nglob,
                                            int gmax, int lo_k, int hi, int nloc, bool bad, int64_t part) {
  constexpr int kCols = D > 64 ? D / 64 : 1;
  const int lane = threadIdx.x & 63;
  const int row_bytes = a.Ds * (STORE == kSame ? 2 : 1);
  const int32_t* pages = a.c.table + b * a.c.table_stride;
  const uint32_t* list = a.list + ((int64_t)b * a.c.H_kv + hk) * a.list_cap;
  const T* q = q_row<T>(a, s, hk, r);
  const int glen = pos >= 0 ? seq_prefix(pos, p) : 0;
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
    const bool loc = it >= nglob;
    const int ts = loc ? lo_k + (nloc - 1 - (it - nglob)) * BN : it * BN;
    const bool sees = lane < BN && (loc ? ts + lane <= pos && ts + lane > pos - p.W && ts + lane < hi
                                        : ts + lane < glen);
    const uint64_t seen = __ballot(sees);
    if (!seen) continue;
    uint32_t slot = 0;
    if (sees) {
      if (!loc && p.rpb > 1)
        slot = list[ts + lane];
      else
        slot = seq_row(pages, loc ? ts + lane : (ts + lane) * p.W, a.c.num_pages, a.c.H_kv, a.c.log_page, hk);
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
  if (part >= 0) {
#pragma unroll
    for (int c = 0; c < kCols; ++c)
      if (lane * kCols + c < D) a.part[part * D + lane * kCols + c] = acc[c];
    if (lane == 0) {
      a.part_ml[2 * part] = m;
      a.part_ml[2 * part + 1] = l;
    }
  } else {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* o = o_row<T>(a, s, hk, r);
#pragma unroll
    for (int c = 0; c < kCols; ++c)
      if (lane * kCols + c < a.D) o[lane * kCols + c] = from_f32<T>(acc[c] * inv);
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
  constexpr bool k8 = STORE != kSame;
  // 16-bit: two stages of K and V tiles, one filled while the other is read. 8-bit:
  // one, and one of the codes as they are loaded: widening empties it before the
  // next tile's loads
  __shared__ __attribute__((aligned(1024))) char stage0[2][Tile::kBytes];
  __shared__ __attribute__((aligned(1024))) char stage1[2][k8 ? 16 : Tile::kBytes];
  __shared__ __attribute__((aligned(1024))) char raw[2][k8 ? BN * D : 16];
  __shared__ __attribute__((aligned(16))) float kscale[2][BN], vscale[2][BN];
  __shared__ uint32_t slots[2][BN];
  __shared__ int2 reach[BM];  // of each row: position, global rows seen (masked tiles read it)

  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) & (NW - 1);
  const ChunkWork w = chunk_work<BM, BN>(a);
  if (w.b < 0) return;
  const int b = w.b, hk = w.hk, tile = w.tile;
  const Seq s = wave_seq(a, b);
  const int rows = s.m * a.grp;
  const SeqPlan p = get_plan(a, s.n);
  const int pos0 = s.n - s.m;
  const int r0 = tile * BM, q0 = r0 + wave * kQW;
  auto pos_of = [&](int r) { return pos0 + row_token(a, r); };
  const int wg_first = pos_of(r0), wg_last = pos_of(min(r0 + BM, rows) - 1);
  const int lo_k = max(0, wg_first - p.W + 1), hi = max(0, wg_last + 1);
  const int gmax = seq_prefix(wg_last, p);
  const int nglob = (gmax + BN - 1) / BN, nloc = (hi - lo_k + BN - 1) / BN;
  const int ntot = min(nglob + (hi > lo_k ? nloc : 0), w.t_end);  // the piece's key tiles end here
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

  // Rows of a tile that this thread fills: the wave's instruction t moves 1 KB, each
  // lane one 16-byte chunk from its own address straight into LDS, at its
  // swizzled place (16-bit) or in order (8-bit codes, which are widened from
  // there; K's scales go to the scores). V is widened times its scale, which rounds
  // it once more: with the scales in P instead (as few_kernel has them) the normaliser,
  // which sums the rounded P on the matrix core, would need a P of its own, and fp16 a
  // reference for each query and tile. The cost: dense int8 chunks of 1000 tokens are
  // off by 2.4e-3 of the result (relative norm) where one rounding of it leaves 1.6e-3.
  constexpr int kPiecesRow = k8 ? D / 16 : Tile::kCPR;
  constexpr int kAll = BN * kPiecesRow, kPer = (kAll + 64 * NW - 1) / (64 * NW);
  const int row_bytes = a.Ds * (k8 ? 1 : 2);
  // cache rows of a tile's rows go through LDS: a thread of the first BN looks up
  // row `tid`, two tiles ahead of its use (one register over the tile in between)
  auto look_up = [&](int it) -> uint32_t {
    if (tid >= BN) return 0u;
    const uint32_t r = slot_of(it, tid);
    bad |= r == kNoRow;
    return r == kNoRow ? 0u : r;
  };
  auto keep = [&](int it, uint32_t r) {
    if (tid < BN) slots[it & 1][tid] = r;
  };
  auto issue = [&](int it, auto& dst) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int t = i * NW + wave;
      if (kAll % (64 * NW) != 0 && t * 64 >= kAll) break;
      const int row = (t * 64 + lane) / kPiecesRow, col = (t * 64 + lane) % kPiecesRow;
      const int chunk = k8 ? col : col ^ Tile::swz(row);
      const int64_t at = (int64_t)slots[it & 1][row] * row_bytes + chunk * 16;
      if (chunk * 16 < row_bytes) {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(a.c.k + at),
                                         CRA_LDS(dst[0] + t * 1024), 16, 0, 0);
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(a.c.v + at),
                                         CRA_LDS(dst[1] + t * 1024), 16, 0, 0);
      }
    }
  };
  auto widen = [&](const float (&vs)[BN]) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int piece = i * 64 * NW + tid, row = piece / kPiecesRow, col = piece % kPiecesRow;
      if (kAll % (64 * NW) != 0 && piece >= kAll) break;
      const uint4 k4 = *reinterpret_cast<const uint4*>(raw[0] + piece * 16);
      const uint4 v4 = *reinterpret_cast<const uint4*>(raw[1] + piece * 16);
      const uint32_t wk[4] = {k4.x, k4.y, k4.z, k4.w}, wv[4] = {v4.x, v4.y, v4.z, v4.w};
      const float sc = vs[row];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint2 x = widen4<T, STORE>(wk[2 * h]), y = widen4<T, STORE>(wk[2 * h + 1]);
        *reinterpret_cast<uint4*>(stage0[0] + Tile::off(row, 2 * col + h)) = make_uint4(x.x, x.y, y.x, y.y);
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = code_value<STORE>(wv[2 * h + j / 4], j % 4) * sc;
        *reinterpret_cast<uint4*>(stage0[1] + Tile::off(row, 2 * col + h)) = pack8<T>(f).w[0];
      }
    }
  };
  float sk = 0.f, sv = 0.f;  // scales of row `tid` of the tile to come
  auto load_scales = [&](int it) {
    if (k8 && tid < BN) {
      const uint32_t r = slots[it & 1][tid];
      sk = a.c.k_scale[r];
      sv = a.c.v_scale[r];
    }
  };
  auto keep_scales = [&](int it) {
    if (k8 && tid < BN) kscale[it & 1][tid] = sk, vscale[it & 1][tid] = sv;
  };
  if (D * (k8 ? 1 : 2) > row_bytes) {  // columns that no load fills
    auto clear = [&](auto& x) {
      for (int i = tid; i < (int)sizeof(x) / 16; i += 64 * NW)
        reinterpret_cast<uint4*>(&x[0][0])[i] = make_uint4(0, 0, 0, 0);
    };
    if constexpr (k8) {
      clear(raw);
    } else {
      clear(stage0);
      clear(stage1);
    }
    __syncthreads();
  }
  LaneOffs<D> lo;
  lo.init(lane);
  Frag<T> qf[QB][D / 32];
  bool counts[QB];
  float m_run[QB], l_run[QB];
  f32x4 acc[D / 16][QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int r = q0 + 16 * qb + l16;
    counts[qb] = r < rows;
    if (g == 0) {
      const int pos = counts[qb] ? pos_of(r) : -1;
      reach[r - r0] = make_int2(pos, pos >= 0 ? seq_prefix(pos, p) : 0);
    }
    const T* qp = q_row<T>(a, s, hk, counts[qb] ? r : 0);
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
      qf[qb][c] = counts[qb] && 32 * c + 8 * g < a.D ? lds_frag_row<T>(qp + 32 * c + 8 * g) : zero_frag<T>();
  }
  const float c2 = a.scale * kLog2e;
  const bool active = q0 < rows;
  const int first = active ? pos_of(q0) : 0;  // positions of the wave's rows: [first, last]
  const int last = active ? pos_of(min(q0 + kQW, rows) - 1) : -1;
  const int w_lo = max(0, first - p.W + 1);
  const int g_all = active ? seq_prefix(first, p) : 0, g_any = active ? seq_prefix(last, p) : 0;
  const Frag<T> one = ones_frag<T>();

#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    m_run[qb] = -kInf;
    l_run[qb] = 0.f;
#pragma unroll
    for (int db = 0; db < D / 16; ++db) acc[db][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  uint32_t ahead = 0;
  if (w.t_first < ntot) {
    keep(w.t_first, look_up(w.t_first));
    if (w.t_first + 1 < ntot) keep(w.t_first + 1, look_up(w.t_first + 1));
    __syncthreads();
    if constexpr (k8)
      issue(w.t_first, raw);
    else
      issue(w.t_first, stage0);
    load_scales(w.t_first);
    keep_scales(w.t_first);
  }
  auto turn = [&](auto second, int it) __attribute__((always_inline)) {
    constexpr bool kS = decltype(second)::value;
    wait_vmem();
    __syncthreads();
    auto refill = [&](auto& dst) {
      if (it + 1 >= ntot) return;
      issue(it + 1, dst);
      load_scales(it + 1);
      if (it + 2 < ntot) ahead = look_up(it + 2);
    };
    if constexpr (k8) {
      widen(vscale[it & 1]);
      __syncthreads();
      refill(raw);
    } else if constexpr (kS) {
      refill(stage0);
    } else {
      refill(stage1);
    }
    const char *tK = stage0[0], *tV = stage0[1];
    if constexpr (!k8 && kS) tK = stage1[0], tV = stage1[1];
    const bool loc = it >= nglob;
    const int ts = tile_start(it);
    const bool work = active && (loc ? ts <= last && ts + BN - 1 >= w_lo : ts < g_any);
    if (work) {
      const bool full = loc ? ts >= last - p.W + 1 && ts + BN - 1 <= first : ts + BN <= g_all;
      const int vis_lo = loc ? max(0, w_lo - ts) : 0, vis_hi = loc ? last - ts : g_any - 1 - ts;
      const int kc0 = vis_lo >> 5, kc1 = min(vis_hi >> 5, BN / 32 - 1);
      TileMask<QB> mk;
      if (full) {
        if constexpr (BN == 64)
          attend_whole<T, STORE, D, BN, QB>(tK, tV, kscale[it & 1], lo, qf, acc, m_run, l_run, c2,
                                            g, mk, one);
        else
          attend_chunk<T, STORE, D, BN, QB, false>(tK, tV, kscale[it & 1], lo, qf, acc,
                                                          m_run, l_run, c2, g, mk, one, 0, 0);
      } else {
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          const int2 e = reach[q0 - r0 + 16 * qb + l16];
          mk.hi[qb] = loc ? e.x - ts : e.y - 1 - ts;
          mk.span[qb] = loc ? (unsigned)(p.W - 1) : 0x7fffffffu;
        }
        attend_chunk<T, STORE, D, BN, QB, true>(tK, tV, kscale[it & 1], lo, qf, acc, m_run,
                                                       l_run, c2, g, mk, one, kc0, kc1);
      }
    }
    if (it + 1 < ntot) keep_scales(it + 1);
    if (it + 2 < ntot) keep(it + 2, ahead);
  };
  if constexpr (k8) {
    for (int it = w.t_first; it < ntot; ++it) turn(std::false_type{}, it);
  } else {
    for (int it = w.t_first; it < ntot; it += 2) {
      turn(std::false_type{}, it);
      if (it + 1 < ntot) turn(std::true_type{}, it + 1);
    }
  }
  bool odd = false;
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    float z = l_run[qb] - l_run[qb];
#pragma unroll
    for (int db = 0; db < D / 16; ++db)
#pragma unroll
      for (int r = 0; r < 4; ++r) z += acc[db][qb][r] - acc[db][qb][r];
    odd |= counts[qb] && !(z == 0.f);
  }
  bad = __syncthreads_or(bad);
  if (__any(odd)) {
    for (int r = q0; r < min(q0 + kQW, rows); ++r) {
      const int64_t at = w.part < 0 ? -1 : w.part + (r - r0);
      careful_row<T, STORE, D, BN>(a, s, p, b, hk, r, pos_of(r), w.t_first, ntot, nglob, gmax, lo_k, hi,
                                   nloc, bad, at);
    }
    return;
  }
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    if (!counts[qb]) continue;
    if (w.part >= 0) {
      const int64_t at = w.part + wave * kQW + 16 * qb + l16;
#pragma unroll
      for (int db = 0; db < D / 16; ++db)
        *reinterpret_cast<f32x4*>(a.part + at * D + 16 * db + 4 * g) = acc[db][qb];
      if (g == 0) {
        a.part_ml[2 * at] = m_run[qb];
        a.part_ml[2 * at + 1] = bad ? __builtin_nanf("") : l_run[qb];
      }
      continue;
    }
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

template <typename T, int D>
__global__ __launch_bounds__(256) void join_kernel(PagedArgs a, uint32_t items) {
  join_chunk<T, 64 * kChunkQB<D>, kChunkBN<D>, D>(a, items);
}

template <typename T, int STORE, int D>
hipError_t run(const PagedArgs& a, uint32_t grid, uint32_t join_tiles, hipStream_t st) {
  chunk_kernel<T, STORE, D><<<grid, 64 * kChunkWaves, 0, st>>>(a);
  if (hipError_t e = hipGetLastError()) return e;
  const uint32_t items = join_tiles * (64 * kChunkQB<D> / join_rows<D>());
  if (items) join_kernel<T, D><<<items < kJoinGrid ? items : kJoinGrid, 256, 0, st>>>(a, items);
  return hipGetLastError();
}
template <typename T, int STORE>
hipError_t run_dim(int Dp, const PagedArgs& a, uint32_t grid, uint32_t join_tiles, hipStream_t st) {
  switch (Dp) {
    case 32: return run<T, STORE, 32>(a, grid, join_tiles, st);
    case 64: return run<T, STORE, 64>(a, grid, join_tiles, st);
    case 128: return run<T, STORE, 128>(a, grid, join_tiles, st);
    default: return run<T, STORE, 256>(a, grid, join_tiles, st);
  }
}

}  // namespace

hipError_t launch_chunk(int dtype, int store, int Dp, const PagedArgs& a, uint32_t grid,
                        uint32_t join_tiles, hipStream_t st) {
  const bool h = dtype == CRA_F16;
  if (store == CRA_STORE_SAME)
    return h ? run_dim<f16, kSame>(Dp, a, grid, join_tiles, st) : run_dim<bf16, kSame>(Dp, a, grid, join_tiles, st);
  if (store == CRA_STORE_E4M3)
    return h ? run_dim<f16, kE4M3>(Dp, a, grid, join_tiles, st) : run_dim<bf16, kE4M3>(Dp, a, grid, join_tiles, st);
  return h ? run_dim<f16, kInt8>(Dp, a, grid, join_tiles, st) : run_dim<bf16, kInt8>(Dp, a, grid, join_tiles, st);
}

}  // namespace cra
