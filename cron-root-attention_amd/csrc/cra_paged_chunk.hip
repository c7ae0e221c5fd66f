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
#include "cra_paged_tiles.hpp"

namespace cra {

namespace {

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
    const KeyTiles keys{pages, list, hk, p.W, p.rpb, nglob, nloc, lo_k};
    for (int r = q0; r < min(q0 + kQW, rows); ++r) {
      const int64_t at = w.part + (r - r0);
      const int pos = pos_of(r);
      careful_row<T, STORE, D, BN>(a, keys, q_row<T>(a, s, hk, r), pos >= 0 ? seq_prefix(pos, p) : 0,
                                   pos - p.W + 1, min(pos, hi - 1), w.t_first, ntot, bad,
                                   w.part < 0 ? nullptr : a.part + at * D, a.part_ml + 2 * at,
                                   o_row<T>(a, s, hk, r));
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
__global__ __launch_bounds__(256) void join_kernel(uint32_t items, PagedArgs a) {
  join_chunk<T, 64 * kChunkQB<D>, kChunkBN<D>, D>(a, items);
}

template <typename T, int STORE, int D>
hipError_t run(const PagedArgs& a, uint32_t grid, uint32_t join_tiles, hipStream_t st) {
  chunk_kernel<T, STORE, D><<<grid, 64 * kChunkWaves, 0, st>>>(a);
  if (hipError_t e = hipGetLastError()) return e;
  const uint32_t items = join_tiles * (64 * kChunkQB<D> / join_rows<D>());
  if (items) join_kernel<T, D><<<items < kJoinGrid ? items : kJoinGrid, 256, 0, st>>>(items, a);
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
