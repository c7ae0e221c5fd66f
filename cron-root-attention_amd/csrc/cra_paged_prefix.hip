// Attention of many sequences' new tokens to a prefix that the sequences share (the same
// rows in the same pages): its rows are read once a kv head for all of them.
//
// A softmax over a set of keys is the sum over a partition of it,
//   o = sum_s e^(m_s - m) o_s / sum_s e^(m_s - m) l_s,  o_s = sum_j e^(x_j - m_s) v_j,
// here of the rows of the prefix (this file) and a sequence's own (few_kernel), joined by
// combine_kernel. The prefix's part of a query's set: its global rows that lie there - of
// blocks that end there for relay rows - and the rows of its window that do.
//
// The queries of all sequences that share stand side by side as rows of one MFMA operand,
// BM at a time (the sequences' at most 16 rows a kv head behind one another), against
// the prefix's key tiles, which are cut into pieces over the grid. Lengths are on the
// device: every workgroup adds up the rows and finds its own.
#include <stdio.h>

#include <type_traits>

#include "cra_paged_dev.hpp"
#include "cra_paged_tiles.hpp"
#include "cra_paged_few.hpp"

namespace cra {

namespace {

constexpr int kPrefixWaves = 8;
constexpr int kLeastTiles = 2;  // key tiles of a piece

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// A row of a tile: where its q lies (head 0 of the kv head's), its window's start, and how
// many global rows it sees. Rows behind the last one see nothing.
struct __attribute__((aligned(16))) PrefixRow {
  int64_t q;
  int ls, glen;
};

// The rows of sequence `lane` of 64 that share, found out from the device's lengths.
struct PrefixSeq {
  Seq s;
  SeqPlan p;
  Share sh;
  int rows;
};
__device__ __forceinline__ PrefixSeq prefix_seq(const PagedArgs& a, const SeqPlan& pp, int b) {
  PrefixSeq x{};
  if (b >= a.c.n_seqs) return x;
  x.s = get_seq(a, b);
  x.p = get_plan(a, x.s.n);
  x.sh = share_of(a, pp, x.s, x.p);
  x.rows = x.sh.P > 0 ? x.s.m * a.grp : 0;
  return x;
}

// The call's work: row tiles, and pieces of each tile's keys.
struct PrefixWork {
  int rows, tiles, pieces;
};
template <int BM, int BN>
__device__ __forceinline__ PrefixWork prefix_work(const PagedArgs& a, const SeqPlan& pp) {
  const int lane = threadIdx.x & 63;
  PrefixWork w{};
  const bool tell = blockIdx.x == 0 && threadIdx.x < 64;  // for combine_kernel
  for (int base = 0; base < a.c.n_seqs; base += 64) {
    const PrefixSeq x = prefix_seq(a, pp, base + lane);
    const int upto = w.rows + (int)wave_upto(x.rows);
    if (tell && base + lane < a.c.n_seqs)
      a.pinfo[base + lane] = x.rows && upto <= a.prefix_most ? upto - x.rows : -1;
    w.rows = __builtin_amdgcn_readlane(upto, 63);
  }
  w.rows = min(w.rows, a.prefix_most);  // offsets of tokens that run backwards may give more
  w.tiles = (w.rows + BM - 1) / BM;
  if (w.tiles > 0) {
    const int keys = (prefix_slots(pp.n, pp.W, pp.rpb) + BN - 1) / BN + (min(pp.n, pp.W) + BN - 1) / BN;
    w.pieces = uniform(max(1, min(a.prefix_grid / (w.tiles * a.c.H_kv), keys / kLeastTiles)));
  }
  if (tell && lane == 0) {
    a.pinfo[a.c.n_seqs] = w.tiles;
    a.pinfo[a.c.n_seqs + 1] = w.pieces;
  }
  return w;
}

// Fills a tile's rows (one wave).
template <int BM>
__device__ __forceinline__ void prefix_rows(const PagedArgs& a, const SeqPlan& pp, int r0, int rows,
                                            PrefixRow (&info)[BM]) {
  const int lane = threadIdx.x & 63;
  for (int i = rows - r0 + lane; i < BM; i += 64) info[i] = PrefixRow{0, pp.n, 0};
  int before = 0;
  for (int base = 0; base < a.c.n_seqs; base += 64) {
    const PrefixSeq x = prefix_seq(a, pp, base + lane);
    const int upto = before + (int)wave_upto(x.rows);
    int at = upto - x.rows - r0;
    for (int t = 0; t < x.s.m && x.rows; ++t) {
      const int pos = x.s.n - x.s.m + t;
      PrefixRow row;
      row.ls = min(pp.n, max(0, pos - x.p.W + 1));
      row.glen = min(x.sh.G0, seq_prefix(pos, x.p));
      row.q = x.s.qb * a.qsb + (int64_t)(x.s.q0 + t) * a.qss;
      for (int h = 0; h < a.grp; ++h, ++at, row.q += a.qsh)
        if (at >= 0 && at < BM) info[at] = row;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
    if (before >= r0 + BM) break;
  }
}

// The tile's keys: all global rows that one of its rows sees, and the prefix's rows from
// the first window on; what all of them see, and what any does.
struct PrefixKeys {
  int gmax, g_all, ls_min, ls_max;
};
template <int BM>
__device__ __forceinline__ PrefixKeys prefix_keys(const PrefixRow (&info)[BM], int first, int count, int n) {
  PrefixKeys k{0, 0x7fffffff, n, 0};
  for (int i = first + (threadIdx.x & 63); i < first + count; i += 64) {
    k.gmax = max(k.gmax, info[i].glen);
    k.g_all = min(k.g_all, info[i].glen);
    k.ls_min = min(k.ls_min, info[i].ls);
    k.ls_max = max(k.ls_max, info[i].ls);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    k.gmax = max(k.gmax, __shfl_xor(k.gmax, o));
    k.g_all = min(k.g_all, __shfl_xor(k.g_all, o));
    k.ls_min = min(k.ls_min, __shfl_xor(k.ls_min, o));
    k.ls_max = max(k.ls_max, __shfl_xor(k.ls_max, o));
  }
  k.gmax = __builtin_amdgcn_readfirstlane(k.gmax);
  k.g_all = __builtin_amdgcn_readfirstlane(k.g_all);
  k.ls_min = __builtin_amdgcn_readfirstlane(k.ls_min);
  k.ls_max = __builtin_amdgcn_readfirstlane(k.ls_max);
  return k;
}

template <int D>
constexpr int kPrefixQB = D > 128 ? 1 : 2;
template <int D>
constexpr int kPrefixBN = D > 128 ? 32 : 64;
template <int D>
constexpr int kPrefixBM = 16 * kPrefixQB<D> * kPrefixWaves;

// One load of every active lane, 16 or 4 bytes from its own address to LDS, lane after lane.
template <int BYTES>
__device__ __forceinline__ void gather_lds(const void* lds, const char* p) {
  const uint32_t at =
      __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)lds);
  if constexpr (BYTES == 16)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(p) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(at), "v"(p) : "memory", "m0");
}
// All but the newest N of the wave's loads have landed, its LDS reads are done, and the
// other waves are as far.
template <int N>
__device__ __forceinline__ void wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// Eight waves of 16 QB rows over K/V tiles in four stages of LDS: a tile's rows are on
// their way while three tiles are computed, the ids of their pages (or list entries) three
// tiles more. Each wave brings eight rows of a tile (with fewer pieces than waves some
// bring the same ones) by loads written as instructions: the compiler would wait for all of
// them before each read of LDS. What bounds it is the softmax beside the MFMAs, as in
// chunk_kernel: a tile of 64 keys x 256 rows at D = 128 takes 2.9 us, its MFMAs 0.9 and its loads
// 1.3. Measured, D = 128: 64 tokens behind 32768 rows, 32/8 heads bf16, dense 62 us (34.5 GFLOP;
// 13 of it write 34 MB of partial rows), with two stages, four waves and two workgroups a CU,
// where it was the loads' latency, 97; 200 behind 15001 over e4m3 106; 48 behind 131072 in the
// sqrt(N) pattern, 16 heads fp16, 19.
constexpr int kStages = 4;

template <typename T, int STORE, int D>
__global__ __launch_bounds__(64 * kPrefixWaves) __attribute__((amdgpu_waves_per_eu(2)))
void prefix_kernel(PagedArgs a) {
  constexpr int NW = kPrefixWaves, QB = kPrefixQB<D>, BN = kPrefixBN<D>, kQW = 16 * QB, BM = kPrefixBM<D>;
  using Tile = SwzTile<D, BN>;
  constexpr bool k8 = STORE != kSame;
  constexpr bool kVS = STORE == kInt8;  // scale_p(): 2.6e-3 of a bf16 result's norm -> 2.4e-3
  // a wave's loads: kPer of K and of V, kRows rows each
  constexpr int kRowBytes = D * (k8 ? 1 : 2), kChunks = kRowBytes / 16, kRows = 64 / kChunks;
  constexpr int kLoads = BN / kRows, kPer = kLoads > NW ? kLoads / NW : 1, kMine = kPer * kRows;
  static_assert(kLoads <= NW || kLoads % NW == 0, "loads of a tile");
  constexpr int kOps = 1 + 2 * kPer + (k8 ? 2 : 0);  // of a tile: ids, rows, scales
  constexpr int kIds = 8;                            // tiles whose ids are held
  __shared__ __attribute__((aligned(1024))) char kt[kStages][BN * kRowBytes];
  __shared__ __attribute__((aligned(1024))) char vt[kStages][BN * kRowBytes];
  __shared__ __attribute__((aligned(1024))) char wide[2][k8 ? Tile::kBytes : 16];
  __shared__ __attribute__((aligned(16))) float kscale[kStages][BN], vscale[kStages][BN];
  __shared__ int32_t ids[kIds][NW][kMine];
  __shared__ PrefixRow info[BM];

  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) & (NW - 1);
  const SeqPlan pp = prefix_plan(a);
  const PrefixWork work = prefix_work<BM, BN>(a, pp);
  const int items = work.tiles * work.pieces * a.c.H_kv;
  const int row_bytes = a.Ds * (k8 ? 1 : 2);
  const float c2 = a.scale * kLog2e;
  const Frag<T> one = ones_frag<T>();
  LaneOffs<D> lo;
  lo.init(lane);
  if (kRowBytes > row_bytes) {  // columns that no load fills
    for (int i = tid; i < (int)sizeof(kt) / 16; i += 64 * NW) {
      reinterpret_cast<uint4*>(&kt[0][0])[i] = make_uint4(0, 0, 0, 0);
      reinterpret_cast<uint4*>(&vt[0][0])[i] = make_uint4(0, 0, 0, 0);
    }
  }
  // the wave's rows of a tile: load i, row j of it
  const int load0 = kLoads < NW ? wave & (kLoads - 1) : wave;
  auto tile_row = [&](int i, int j) { return (i * NW + load0) * kRows + j; };
  // items of one head stand H_kv apart: with a multiple of 8 heads they meet in one XCD's L2
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int rest = uniform((int)div_by(item, a.d_hkv)), hk = item - rest * a.c.H_kv;
    const int piece = uniform(rest / work.tiles), r0 = (rest - piece * work.tiles) * BM;
    __syncthreads();  // the rows of the item before are done with
    if (wave == 0) prefix_rows<BM>(a, pp, r0, work.rows, info);
    __syncthreads();
    const int rows = min(BM, work.rows - r0);
    const PrefixKeys all = prefix_keys<BM>(info, 0, rows, pp.n);
    const int nglob = (all.gmax + BN - 1) / BN, nloc = (pp.n - all.ls_min + BN - 1) / BN;
    const int per = uniform((nglob + nloc + work.pieces - 1) / work.pieces);
    const int t_first = piece * per, ntot = min(nglob + nloc, t_first + per);
    const KeyTiles keys{a.ptable, a.plist + (int64_t)hk * a.plist_cap, hk, pp.W, pp.rpb, nglob, nloc, all.ls_min};
    bool bad = false;

    auto tile_start = [&](int it) {
      return it >= nglob ? all.ls_min + (nloc - 1 - (it - nglob)) * BN : it * BN;
    };
    // row of the prefix, or place in its list, of a tile's row (the last one behind the end)
    auto key_of = [&](int it, int row) {
      return min(tile_start(it) + row, (it < nglob ? all.gmax : pp.n) - 1);
    };
    auto listed = [&](int it) { return it < nglob && pp.rpb > 1; };
    // (what follows from the lane is formed anew for each tile: held over the loop it
    // would leave no registers for the tile's steps)
    auto fetch_ids = [&](int it) __attribute__((always_inline)) {
      it = min(it, ntot - 1);
      const int lane = fresh(threadIdx.x & 63);
      if (lane < kMine) {
        const int i = key_of(it, tile_row(lane / kRows, lane % kRows));
        const int at = listed(it) ? i : (it < nglob ? i * pp.W : i) >> a.c.log_page;
        gather_lds<4>(ids[it & (kIds - 1)][wave],
                      reinterpret_cast<const char*>(listed(it) ? reinterpret_cast<const int32_t*>(keys.list) + at
                                                               : keys.pages + at));
      }
    };
    auto cache_row_of = [&](int it, int i, int j) -> uint32_t {
      const int32_t id = ids[it & (kIds - 1)][wave][i * kRows + j];
      if (listed(it)) return (uint32_t)id;
      const int key = key_of(it, tile_row(i, j)), row = it < nglob ? key * pp.W : key;
      if ((uint32_t)id >= (uint32_t)a.c.num_pages) return kNoRow;
      return cache_row(id, a.c.H_kv, a.c.log_page, hk, row & ((1 << a.c.log_page) - 1));
    };
    auto fill = [&](int it, int s) __attribute__((always_inline)) {
      it = min(it, ntot - 1);
      const int lane = fresh(threadIdx.x & 63);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int j = lane / kChunks, row = tile_row(i, j);
        const int chunk = k8 ? lane % kChunks : (lane % kChunks) ^ Tile::swz(row);
        uint32_t r = cache_row_of(it, i, j);
        bad |= r == kNoRow;
        r = r == kNoRow ? 0u : r;
        const int64_t at = (int64_t)r * row_bytes + chunk * 16;
        const int dst = (i * NW + load0) * 1024;
        if (chunk * 16 < row_bytes) {
          gather_lds<16>(kt[s] + dst, a.c.k + at);
          gather_lds<16>(vt[s] + dst, a.c.v + at);
        }
      }
      if constexpr (k8) {
        static_assert(!k8 || kPer == 1, "one load a wave");
        if (lane < kRows) {
          uint32_t r = cache_row_of(it, 0, lane);
          r = r == kNoRow ? 0u : r;
          gather_lds<4>(kscale[s] + load0 * kRows, reinterpret_cast<const char*>(a.c.k_scale + r));
          gather_lds<4>(vscale[s] + load0 * kRows, reinterpret_cast<const char*>(a.c.v_scale + r));
        }
      }
    };
    // codes of stage s into the 16-bit tile
    auto widen = [&](int s) __attribute__((always_inline)) {
      const int tid = fresh(threadIdx.x);
      constexpr int kAll = BN * kChunks, kEach = (kAll + 64 * NW - 1) / (64 * NW);
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int p = i * 64 * NW + tid, row = p / kChunks, col = p % kChunks;
        if (kAll % (64 * NW) != 0 && p >= kAll) break;
        const uint4 k4 = *reinterpret_cast<const uint4*>(kt[s] + p * 16);
        const uint4 v4 = *reinterpret_cast<const uint4*>(vt[s] + p * 16);
        const uint32_t wk[4] = {k4.x, k4.y, k4.z, k4.w}, wv[4] = {v4.x, v4.y, v4.z, v4.w};
        const float sc = kVS ? scale_of_codes<T>(vscale[s][row]) : vscale[s][row];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint2 x = widen4<T, STORE>(wk[2 * h]), y = widen4<T, STORE>(wk[2 * h + 1]);
          *reinterpret_cast<uint4*>(wide[0] + Tile::off(row, 2 * col + h)) = make_uint4(x.x, x.y, y.x, y.y);
          float f[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = code_value<STORE>(wv[2 * h + j / 4], j % 4) * sc;
          *reinterpret_cast<uint4*>(wide[1] + Tile::off(row, 2 * col + h)) = pack8<T>(f).w[0];
        }
      }
    };
    const int q0 = wave * kQW;  // the wave's rows of the tile
    const bool active = q0 < rows;
    const PrefixKeys mine = prefix_keys<BM>(info, q0, active ? min(kQW, rows - q0) : 0, pp.n);
    Frag<T> qf[QB][D / 32];
    bool counts[QB];
    float m_run[QB], l_run[QB];
    f32x4 acc[D / 16][QB];
    auto q_of = [&](int r) { return static_cast<const T*>(a.q) + info[r].q + (int64_t)hk * a.grp * a.qsh; };
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const int r = q0 + 16 * qb + l16;
      counts[qb] = r < rows;
      const T* qp = q_of(r);
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
        qf[qb][c] = counts[qb] && 32 * c + 8 * g < a.D ? lds_frag_row<T>(qp + 32 * c + 8 * g) : zero_frag<T>();
      m_run[qb] = -kInf;
      l_run[qb] = 0.f;
#pragma unroll
      for (int db = 0; db < D / 16; ++db) acc[db][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    auto turn = [&](int s, int it) __attribute__((always_inline)) {
      wait_barrier<2 * kOps>();  // the tile has landed, and the one before it has been read
      fetch_ids(it + 6);
      fill(it + 3, (s + 3) & 3);
      if constexpr (k8) {
        widen(s);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      }
      const char *tK = k8 ? wide[0] : kt[s], *tV = k8 ? wide[1] : vt[s];
      const bool loc = it >= nglob;
      const int ts = tile_start(it);
      const bool any = active && (loc ? ts + BN > mine.ls_min : ts < mine.gmax);
      if (uniform(any)) {
        const bool full = uniform(loc ? ts >= mine.ls_max && ts + BN <= pp.n : ts + BN <= mine.g_all);
        TileMask<QB> mk;
        if (full) {
          if constexpr (BN == 64)
            attend_whole<T, STORE, D, BN, QB, kVS>(tK, tV, kscale[s], lo, qf, acc, m_run, l_run, c2, g, mk, one,
                                                    vscale[s]);
          else
            attend_chunk<T, STORE, D, BN, QB, false, kVS>(tK, tV, kscale[s], lo, qf, acc, m_run, l_run, c2, g, mk,
                                                          one, 0, 0, vscale[s]);
        }
        // (a branch of its own: with an else the accumulators are held twice)
        if (uniform(fresh(full ? 0 : 1))) {
          const int vis_lo = loc ? max(0, mine.ls_min - ts) : 0, vis_hi = (loc ? pp.n : mine.gmax) - 1 - ts;
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) {
            const PrefixRow r = info[q0 + 16 * qb + l16];
            mk.hi[qb] = loc ? (r.ls < pp.n ? pp.n - 1 - ts : -1) : r.glen - 1 - ts;
            mk.span[qb] = loc ? (unsigned)max(pp.n - 1 - r.ls, 0) : 0x7fffffffu;
          }
          attend_chunk<T, STORE, D, BN, QB, true, kVS>(tK, tV, kscale[s], lo, qf, acc, m_run, l_run, c2, g, mk, one,
                                                  vis_lo >> 5, min(vis_hi >> 5, BN / 32 - 1), vscale[s]);
        }
      }
    };
    if (t_first < ntot) {
#pragma unroll
      for (int i = 0; i < 3; ++i) fetch_ids(t_first + i);
      wait_vmem();  // known to the compiler: q's loads too, or it would wait for all in the loop
#pragma unroll
      for (int i = 0; i < 3; ++i) {  // in the order of the turns, which count the loads
        fetch_ids(t_first + 3 + i);
        fill(t_first + i, i);
      }
      for (int it = t_first; it < ntot; ++it) turn((it - t_first) & (kStages - 1), it);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // tiles past the last one, too
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
    const int64_t part = (int64_t)item * BM;
    if (__any(odd)) {
      for (int r = q0; r < min(q0 + kQW, rows); ++r)
        careful_row<T, STORE, D, BN>(a, keys, q_of(r), info[r].glen, info[r].ls, pp.n - 1, t_first, ntot, bad,
                                     a.ppart + (part + r) * D, a.ppart_ml + 2 * (part + r), static_cast<T*>(nullptr));
      continue;
    }
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      if (!counts[qb]) continue;
      const int64_t at = part + q0 + 16 * qb + l16;
#pragma unroll
      for (int db = 0; db < D / 16; ++db)
        *reinterpret_cast<f32x4*>(a.ppart + at * D + 16 * db + 4 * g) = acc[db][qb];
      if (g == 0) {
        a.ppart_ml[2 * at] = m_run[qb];
        a.ppart_ml[2 * at + 1] = bad ? __builtin_nanf("") : l_run[qb];
      }
    }
  }
}

// fp32, as f32_item (cra_paged_few.hpp): four waves of 16 rows, 32 keys at a time.
template <int STORE, int D>
__global__ __launch_bounds__(256) void prefix_f32_kernel(PagedArgs a) {
  constexpr int BM = kF32Rows, BN = kF32Keys, kStride = D + 4;
  __shared__ __attribute__((aligned(16))) float tK[BN][kStride];
  __shared__ __attribute__((aligned(16))) float tV[BN][kStride];
  __shared__ PrefixRow info[BM];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, g = lane >> 4;
  const SeqPlan pp = prefix_plan(a);
  const PrefixWork work = prefix_work<BM, BN>(a, pp);
  const int items = work.tiles * work.pieces * a.c.H_kv;
  const float c2 = a.scale * kLog2e;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int rest = (int)div_by(item, a.d_hkv), hk = item - rest * a.c.H_kv;
    const int piece = rest / work.tiles, r0 = (rest - piece * work.tiles) * BM;
    __syncthreads();  // the rows of the item before are done with
    if (wave == 0) prefix_rows<BM>(a, pp, r0, work.rows, info);
    __syncthreads();
    const int rows = min(BM, work.rows - r0);
    const PrefixKeys all = prefix_keys<BM>(info, 0, rows, pp.n);
    const int nglob = (all.gmax + BN - 1) / BN, nloc = (pp.n - all.ls_min + BN - 1) / BN;
    const int per = (nglob + nloc + work.pieces - 1) / work.pieces;
    const int t_first = piece * per, t_last = min(nglob + nloc, t_first + per);
    const uint32_t* list = a.plist + (int64_t)hk * a.plist_cap;
    bool bad = false;

    // eight threads a row, D / 8 columns each: quads of them, 32 columns apart
    constexpr int kCols = D / 8;
    const int frow = tid >> 3, fcol = (tid & 7) * 4;
    f32x4 rk[kCols / 4], rv[kCols / 4];
    auto load = [&](int it) {
      const int ts = it >= nglob ? all.ls_min + (it - nglob) * BN : it * BN;
      const int i = min(ts + frow, (it < nglob ? all.gmax : pp.n) - 1);
      uint32_t sl = it < nglob && pp.rpb > 1 ? list[i]
                                             : seq_row(a.ptable, it < nglob ? i * pp.W : i, a.c.num_pages, a.c.H_kv,
                                                       a.c.log_page, hk);
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
    if (t_first < t_last) load(t_first);

    const int q0 = 16 * wave, r = q0 + l16;
    const bool have = r < rows, active = q0 < rows;
    const PrefixRow row = info[r];
    const PrefixKeys mine = prefix_keys<BM>(info, q0, active ? min(16, rows - q0) : 0, pp.n);
    // Q^T operand: MFMA 4 c + i of a 16-column step takes column 16 c + 4 g + i
    f32x4 qf[D / 16];
    const float* qp = static_cast<const float*>(a.q) + row.q + (int64_t)hk * a.grp * a.qsh;
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
      qf[c] = have && 16 * c + 4 * g < a.D ? *reinterpret_cast<const f32x4*>(qp + 16 * c + 4 * g)
                                           : f32x4{0.f, 0.f, 0.f, 0.f};
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
      const int ts = loc ? all.ls_min + (it - nglob) * BN : it * BN;
      if (!(active && (loc ? ts + BN > mine.ls_min : ts < mine.gmax))) continue;
      const bool full = loc ? ts >= mine.ls_max && ts + BN <= pp.n : ts + BN <= mine.g_all;
      const int vis = loc ? (row.ls < pp.n ? pp.n - 1 - ts : -1) : row.glen - 1 - ts;
      const unsigned span = loc ? (unsigned)max(pp.n - 1 - row.ls, 0) : 0x7fffffffu;
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
    if (!have) continue;
    const int64_t at = (int64_t)item * BM + r;
#pragma unroll
    for (int db = 0; db < D / 16; ++db)
      *reinterpret_cast<f32x4*>(a.ppart + at * D + 16 * db + 4 * g) = acc[db];
    if (g == 0) {
      a.ppart_ml[2 * at] = m_run;
      a.ppart_ml[2 * at + 1] = l_run;
    }
  }
}

template <typename T, int STORE, int D>
hipError_t run(const PagedArgs& a, uint32_t combine_grid, uint32_t few_grid, hipStream_t st) {
  if constexpr (std::is_same<T, float>::value)
    prefix_f32_kernel<STORE, D><<<a.prefix_grid, 256, 0, st>>>(a);
  else
    prefix_kernel<T, STORE, D><<<a.prefix_grid, 64 * kPrefixWaves, 0, st>>>(a);
  if (hipError_t e = hipGetLastError()) return e;
  if constexpr (std::is_same<T, float>::value)
    f32_kernel<STORE, D, true, true><<<few_grid, 256, 0, st>>>(a);
  else
    few_kernel<T, STORE, D, true><<<few_grid, 64 * kFewWaves, 0, st>>>(a);
  if (hipError_t e = hipGetLastError()) return e;
  combine_kernel<T, true><<<combine_grid, 256, 0, st>>>(D, a);
  return hipGetLastError();
}
template <typename T, int STORE>
hipError_t run_dim(int Dp, const PagedArgs& a, uint32_t combine_grid, uint32_t few_grid, hipStream_t st) {
  switch (Dp) {
    case 32: return run<T, STORE, 32>(a, combine_grid, few_grid, st);
    case 64: return run<T, STORE, 64>(a, combine_grid, few_grid, st);
    case 128: return run<T, STORE, 128>(a, combine_grid, few_grid, st);
    default: return run<T, STORE, 256>(a, combine_grid, few_grid, st);
  }
}
template <typename T>
hipError_t run_store(int store, int Dp, const PagedArgs& a, uint32_t combine_grid, uint32_t few_grid, hipStream_t st) {
  return store == CRA_STORE_SAME   ? run_dim<T, kSame>(Dp, a, combine_grid, few_grid, st)
         : store == CRA_STORE_E4M3 ? run_dim<T, kE4M3>(Dp, a, combine_grid, few_grid, st)
                                   : run_dim<T, kInt8>(Dp, a, combine_grid, few_grid, st);
}

}  // namespace

PrefixTiles prefix_tiles(int dtype, int Dp) {
  if (dtype == CRA_F32) return PrefixTiles{kF32Rows, kF32Keys};
  return Dp > 128 ? PrefixTiles{kPrefixBM<256>, kPrefixBN<256>} : PrefixTiles{kPrefixBM<128>, kPrefixBN<128>};
}

hipError_t launch_prefix(int dtype, int store, int Dp, const PagedArgs& a, uint32_t combine_grid, uint32_t few_grid,
                         hipStream_t st) {
  if (dtype == CRA_F16) return run_store<f16>(store, Dp, a, combine_grid, few_grid, st);
  if (dtype == CRA_BF16) return run_store<bf16>(store, Dp, a, combine_grid, few_grid, st);
  return run_store<float>(store, Dp, a, combine_grid, few_grid, st);
}

}  // namespace cra
