// New tokens on their way into a paged cache, in one launch: q and k normed and turned
// by their tokens' places in the sequences (or given positions), k and v stored, with
// the C ABI front end. The norm and rotation of cra_rotary.hip (but for the last bit of
// an fp32 sum before its rounding: there the compiler chooses which product of a pair it
// rounds, for each element) with the write of cra_cache.hip behind it:
//   z = x r w,  r = 1 / sqrt(mean(x^2) + eps)             (with the norm)
//   y_a = z_a c - z_b s,  y_b = z_b c + z_a s             c, s of row p of the table,
//   p = n - m + t for new token t of m of a sequence of n
// k is rounded to the rows' type before it is stored: what a cache of that type would
// hold is what 8-bit codes are made of and relay rows are ranked by.
//
// A row belongs to L lanes of two V-element chunks each, a pair's halves in one lane, as
// in the rotation alone. Key rows then pass through LDS to the lanes of the write (8
// consecutive elements each, whose squares are summed in the packed rows' order). The
// rows are loaded before their places are known: finding one takes up to five loads in
// turn (offsets, length, table row; length, page id).
//
// Bound by memory, single tokens by that chain and the launch. Measured, replayed from a
// graph, D = 128, 16 heads of q: 32768 tokens, 16 heads of k, fp16 rows 172 us (805 MB: 157 by
// a copy's rate); 25969 tokens of 16 sequences, 4 heads of k, e4m3 rows 70 (293 MB: 57); one
// token each of 64 sequences, 32 heads and 8 9.
#include <stdio.h>

#include <algorithm>
#include <type_traits>

#include "cra_cache_dev.hpp"
#include "cra_common.hpp"
#include "cra_internal.hpp"
#include "cra_paged.hpp"
#include "cra_turn_dev.hpp"

namespace cra {

int set_error(int code, const char* msg);

namespace {

constexpr int kThreads = kTurnThreads, kHeads = 2;
// Rows of q from which a lane takes two: 32768 x 16 182 -> 172 us, 25969 x 16 142 -> 140; four 177
// and 142, eight 189 and 148. Fewer rows are spread over more workgroups instead.
constexpr int64_t kManyRows = 1 << 14;

struct AppendArgs {
  TurnArgs g;   // t[0]: q into y; t[1]: k, into the cache
  PagedView c;
  const void* v;
  int64_t vsb, vsh, vss;
  float *k_norm, *k_scale, *v_scale;
  int Ds, log_w;  // columns stored, lanes of a row as it is stored
  int heads;      // heads of q an item covers, each
  int64_t xsh, ysh;  // elements behind the one before
};

// Where a new token belongs: its sequence (-1: none), that one's new tokens, and which
// of them it is.
struct Place {
  int b, count, t;
};
// Packed tokens are looked up by the 2^log_l lanes of the row together (a lane alone
// halves the offsets).
__device__ __forceinline__ Place place_of(const PagedView& c, const Item& im, int lane, int log_l) {
  if (!c.cu) return Place{im.b, c.query_len, im.s};
  const int at = threadIdx.x & 63 & ~lane, lanes = 1 << log_l;
  Place p{};
  if (log_l == 0) {
    p.b = seq_of_token(c.cu, c.n_seqs, im.s, 2, [&](int first, int step, int n) {
      return step < n && c.cu[first + step] <= im.s ? 2 : 1;
    });
  } else {
    p.b = seq_of_token(c.cu, c.n_seqs, im.s, lanes, [&](int first, int step, int n) {
      const int64_t i = (int64_t)lane * step;
      const uint64_t m = __ballot(i < n && c.cu[first + (i < n ? i : 0)] <= im.s) >> at;
      return __popcll(lanes == 64 ? m : m & ((1ull << lanes) - 1));
    });
  }
  if (p.b < 0) return p;
  const TokenRange tr = token_range(c.cu, p.b, c.tokens);
  p.count = tr.last - tr.first;
  p.t = im.s - tr.first;
  return p;
}

// turn() with the roundings written out: q and k of one row come out the same.
__device__ __forceinline__ void turn_one(float& x, float& y, float c, float s) {
  const float x0 = x;
  x = __builtin_fmaf(x0, c, -(y * s));
  y = __builtin_fmaf(y, c, x0 * s);
}
template <int V>
__device__ __forceinline__ void turn_rows(float (&a)[V], float (&b)[V], const float (&c)[V],
                                          const float (&s)[V], bool interleaved) {
  if (interleaved) {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      turn_one(a[2 * j], a[2 * j + 1], c[j], s[j]);
      turn_one(b[2 * j], b[2 * j + 1], c[V / 2 + j], s[V / 2 + j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) turn_one(a[i], b[i], c[i], s[i]);
  }
}

// V elements as they lie in memory.
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> raw_vec(const T* p) {
  using raw_t = Vec<T, V>;
  if constexpr (V * sizeof(T) == 16)
    return __builtin_bit_cast(raw_t, *reinterpret_cast<const uint4*>(p));
  else if constexpr (V * sizeof(T) == 8)
    return __builtin_bit_cast(raw_t, *reinterpret_cast<const uint2*>(p));
  else
    return __builtin_bit_cast(raw_t, *reinterpret_cast<const uint32_t*>(p));
}
template <typename T, int V>
__device__ __forceinline__ void widen_vec(const Vec<T, V>& x, bool on, float (&f)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = on ? to_f32(x.v[i]) : 0.f;
}

// A lane's part of one row of k (and the rows of v of its wave), or of U neighbouring heads
// of q, which share place, turns and weights. Loads stand outside of branches, at clamped
// addresses, so that they are on their way together: one in a branch of its own is waited
// for there (25969 tokens and their reading back: 167 us, 142 so). held, dst: rows of k,
// turned, and where they go.
template <typename T, int STORE, int V, int U, bool KV>
__device__ __forceinline__ void append_rows(const AppendArgs& a, uint32_t block, T* held, uint32_t* dst) {
  const TurnArgs& g = a.g;
  const TurnTensor& t = g.t[KV];
  const int log_l = g.log_l, lane = threadIdx.x & ((1 << log_l) - 1), slot = threadIdx.x >> log_l;
  const int rows = kThreads >> log_l;
  const uint32_t it = block * rows + slot;
  const bool on = it < t.items;
  const Item im = item_at(g, t, on ? it : t.items - 1);
  const Unit un = unit_at<V>(g, lane);
  const T* x = static_cast<const T*>(t.x) + im.b * t.xsb + im.s * t.xss + im.h * t.xsh;
  Vec<T, V> rp[U], rq[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    rp[u] = raw_vec<T, V>(x + u * a.xsh + (un.a ? un.ea : 0));
    rq[u] = raw_vec<T, V>(x + u * a.xsh + (un.b ? un.eb : 0));
  }
  // offsets and lengths of up to 63 sequences, a lane each
  const PagedView& c = a.c;
  const int wl = threadIdx.x & 63, seqs = c.n_seqs;
  const bool near = c.cu && seqs < 64;
  int cu = 0, len = 0;
  if (near) {
    cu = c.cu[min(wl, seqs)];
    len = c.lens[min(wl, seqs - 1)];
  }

  // rows of v: as they are stored, up to two a thread (a stored row takes at most
  // twice the lanes of a turned one: cra_cache_append sees to it)
  const int wlane = threadIdx.x & ((1 << a.log_w) - 1), wrow = threadIdx.x >> a.log_w;
  const int wrows = kThreads >> a.log_w;
  const bool have = wlane * 8 < g.D;
  Row8<T> vr[2];
  if constexpr (KV) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const Item vi = item_at(g, t, min(block * rows + min(wrow + j * wrows, rows - 1), t.items - 1));
      const uint4* vp = reinterpret_cast<const uint4*>(static_cast<const T*>(a.v) + vi.b * a.vsb + vi.h * a.vsh +
                                                       vi.s * a.vss + (have ? wlane * 8 : 0));
#pragma unroll
      for (int i = 0; i < (int)(sizeof(T) / 2); ++i) vr[j].w[i] = vp[i];
    }
  }

  // the wave's tokens are most often of one sequence, which all lanes find at once
  Place pl{};
  int n = 0;  // the sequence's length
  bool found = false;
  if (near) {
    const int t0 = __builtin_amdgcn_readfirstlane(im.s);
    const int b = __popcll(__ballot(wl <= seqs && cu <= t0)) - 1;
    if (b >= 0 && b < seqs) {
      const int first = __builtin_amdgcn_readlane(cu, b), last = __builtin_amdgcn_readlane(cu, b + 1);
      if (__all(im.s >= first && im.s < last) && first >= 0 && last <= c.tokens) {
        found = true;
        pl = Place{b, last - first, im.s - first};
        n = __builtin_amdgcn_readlane(len, b);
      }
    }
  }
  if (!found) {
    pl = place_of(c, im, lane, log_l);
    n = c.lens[max(pl.b, 0)];
  }
  const int64_t at = pl.b < 0 ? -1 : (int64_t)n - pl.count + pl.t;
  const int64_t turn_row = g.pos ? table_row(g, im) : at < g.table_rows ? at : -1;
  float cs[V], sn[V], wp[V], wq[V];
#pragma unroll
  for (int i = 0; i < V; ++i) wp[i] = wq[i] = 1.f;
  if (g.rot) {  // (lanes that do not turn, and rows without a place, read the first row)
    const float* tp = g.table + (turn_row >= 0 ? turn_row : 0) * g.rot + (un.turn ? lane * V : 0);
    load_floats<V>(tp, cs);
    load_floats<V>(tp + (g.rot >> 1), sn);
  }
  if (g.norm && t.w) {
    const int ea = un.a ? un.ea : 0, eb = un.b ? un.eb : 0;
    if (g.w_f32) {
      load_floats<V>(static_cast<const float*>(t.w) + ea, wp);
      load_floats<V>(static_cast<const float*>(t.w) + eb, wq);
    } else {
      const Vec<T, V> ra = raw_vec<T, V>(static_cast<const T*>(t.w) + ea), rb = raw_vec<T, V>(static_cast<const T*>(t.w) + eb);
      widen_vec<T, V>(ra, true, wp);
      widen_vec<T, V>(rb, true, wq);
    }
  }
  if (turn_row < 0) {
#pragma unroll
    for (int i = 0; i < V; ++i) cs[i] = sn[i] = __builtin_nanf("");
  }
  auto turned = [&](const Vec<T, V>& x0, const Vec<T, V>& x1, float (&p)[V], float (&q)[V]) {
    widen_vec<T, V>(x0, un.a, p);
    widen_vec<T, V>(x1, un.b, q);
    if (g.norm) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) ss += p[i] * p[i] + q[i] * q[i];
      const float r = rsqrtf(turn_sum(ss, log_l) * g.inv_d + g.eps);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        p[i] *= r * wp[i];
        q[i] *= r * wq[i];
      }
    }
    if (un.turn) turn_rows<V>(p, q, cs, sn, g.interleaved);
  };
  float p[V], q[V];
  if constexpr (!KV) {
    T* y = static_cast<T*>(t.y) + im.b * t.ysb + im.s * t.yss + im.h * t.ysh;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      turned(rp[u], rq[u], p, q);
      if (!on) continue;
      if (pl.b < 0) {  // padding
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = q[i] = 0.f;
      }
      if (un.a) store_vec<T, V>(y + u * a.ysh + un.ea, p);
      if (un.b) store_vec<T, V>(y + u * a.ysh + un.eb, q);
    }
  } else {
    turned(rp[0], rq[0], p, q);
    T* mine = held + slot * (2 * V << log_l);
    if (un.a) store_vec<T, V>(mine + un.ea, p);
    if (un.b) store_vec<T, V>(mine + un.eb, q);
    if (lane == 0) {
      const int row = pl.b < 0 ? -1 : write_row(n, pl.count, pl.t, c.pages_per_seq, c.log_page);
      dst[slot] = on && row >= 0 ? seq_row(c.table + pl.b * c.table_stride, row, c.num_pages, c.H_kv, c.log_page, im.h)
                                 : kNoRow;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = wrow + j * wrows;
      if (r >= rows || dst[r] == kNoRow) continue;  // whole rows: the exchanges stay within one
      Row8<T> kr;
      const uint4* kp = reinterpret_cast<const uint4*>(held + r * (2 * V << log_l) + (have ? wlane * 8 : 0));
      float kx[8], vx[8];
#pragma unroll
      for (int i = 0; i < (int)(sizeof(T) / 2); ++i) {
        kr.w[i] = have ? kp[i] : make_uint4(0, 0, 0, 0);
        vr[j].w[i] = have ? vr[j].w[i] : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        kx[i] = to_f32(reinterpret_cast<const T*>(kr.w)[i]);
        vx[i] = to_f32(reinterpret_cast<const T*>(vr[j].w)[i]);
      }
      const float norm = lanes_sum(square_sum(kx), a.log_w);
      if (wlane == 0) a.k_norm[dst[r]] = norm;
      store_row<T, STORE>(kx, kr, const_cast<char*>(c.k), a.k_scale, dst[r], a.Ds, wlane, a.log_w);
      store_row<T, STORE>(vx, vr[j], const_cast<char*>(c.v), a.v_scale, dst[r], a.Ds, wlane, a.log_w);
    }
  }
}

template <typename T, int STORE, int V, int U>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a) {
  __shared__ __attribute__((aligned(16))) T held[kThreads * 2 * V];
  __shared__ uint32_t dst[kThreads];
  const uint32_t own = a.g.t[1].blocks;
  if (blockIdx.x < own)
    append_rows<T, STORE, V, 1, true>(a, blockIdx.x, held, dst);
  else
    append_rows<T, STORE, V, U, false>(a, blockIdx.x - own, nullptr, nullptr);
}

int err(int code, const char* msg) { return set_error(code, msg); }

template <typename T, int STORE, int V>
hipError_t run(const AppendArgs& a, hipStream_t st) {
  const int blocks = a.g.t[0].blocks + a.g.t[1].blocks;
  if (a.heads == kHeads)
    append_kernel<T, STORE, V, kHeads><<<blocks, kThreads, 0, st>>>(a);
  else
    append_kernel<T, STORE, V, 1><<<blocks, kThreads, 0, st>>>(a);
  return hipGetLastError();
}
template <typename T, int V>
hipError_t run_store(int store, const AppendArgs& a, hipStream_t st) {
  return store == CRA_STORE_SAME   ? run<T, kSame, V>(a, st)
         : store == CRA_STORE_E4M3 ? run<T, kE4M3, V>(a, st)
                                   : run<T, kInt8, V>(a, st);
}
template <typename T>
hipError_t run_type(int V, int store, const AppendArgs& a, hipStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (V == 8) return run_store<T, 8>(store, a, st);
  return V == 4 ? run_store<T, 4>(store, a, st) : run_store<T, 2>(store, a, st);
}

}  // namespace
}  // namespace cra

using namespace cra;

extern "C" {

int cra_cache_append(const cra_cache* c, const cra_batch* b, const cra_turn* p, cra_tensor q,
                     cra_tensor k, cra_tensor v, const void* wq, const void* wk, cra_tensor yq,
                     void* stream) {
  if (int e = check_cache(c)) return e;
  if (int e = check_batch(c, b)) return e;
  if (int e = check_turn(p)) return e;
  if (p->dtype != c->dtype) return err(CRA_E_DTYPE, "q and k must be of the cache's dtype");
  if (p->H_kv != c->H_kv) return err(CRA_E_INVALID, "H_kv differs from the cache's");
  if (p->D < 8 || p->D > c->D || p->D % 8)
    return err(CRA_E_INVALID, "D must be a multiple of 8 up to the row width");
  if (p->B != (b->cu_seqlens ? 1 : b->n_seqs) || p->S != (b->cu_seqlens ? b->tokens : b->query_len))
    return err(CRA_E_INVALID, "B and S differ from the batch's");
  const int esz = p->dtype == CRA_F32 ? 4 : 2, vec = 16 / esz;
  for (const cra_tensor* t : {&q, &k, &v, &yq}) {
    if (!t->ptr) return err(CRA_E_INVALID, "q, k, v or the output is NULL");
    if (reinterpret_cast<uintptr_t>(t->ptr) % 16 || t->sb % vec || t->sh % vec || t->ss % vec)
      return err(CRA_E_LAYOUT, "rows must be 16-byte aligned");
  }
  const cra_tensor* ts[3] = {&q, &k, &yq};
  const void* ws[2] = {p->norm ? wq : nullptr, p->norm ? wk : nullptr};
  TurnShape sh = turn_shape(p, ts, 3, ws);
  if (sh.V < 2) return err(CRA_E_UNSUPPORTED, "weights or turned halves between 4-byte steps are not built");
  AppendArgs a{};
  a.Ds = c->D;
  while ((8 << a.log_w) < c->D) ++a.log_w;
  // a workgroup stores two rows a thread (append_rows): heads far narrower than the cache's
  // rows take more lanes than they have units for
  sh.log_l = std::max(sh.log_l, a.log_w - 1);
  fill_args(a.g, p, sh);
  a.heads = p->H_q % kHeads == 0 && (int64_t)p->B * p->S * p->H_q >= kManyRows ? kHeads : 1;
  a.xsh = q.sh, a.ysh = yq.sh;
  cra_tensor qs = q, ys = yq;  // of `heads` heads together
  qs.sh *= a.heads, ys.sh *= a.heads;
  fill_tensor(a.g.t[0], p, sh, p->H_q / a.heads, qs, nullptr, ys, ws[0]);
  a.g.t[0].head_fast = yq.sh < yq.ss;
  fill_tensor(a.g.t[1], p, sh, p->H_kv, k, nullptr, k, ws[1]);
  a.g.t[1].y = nullptr;
  a.g.norm = p->norm != 0;
  a.c = paged_view(c, b);
  a.v = v.ptr, a.vsb = v.sb, a.vsh = v.sh, a.vss = v.ss;
  a.k_norm = c->k_norm, a.k_scale = c->k_scale, a.v_scale = c->v_scale;
  if (((int64_t)a.g.t[0].blocks + a.g.t[1].blocks) * kThreads >= (int64_t)1 << 32)
    return err(CRA_E_INVALID, "too many rows for one launch");
  const hipStream_t st = (hipStream_t)stream;
  const hipError_t e = p->dtype == CRA_F16    ? run_type<f16>(sh.V, c->store, a, st)
                       : p->dtype == CRA_BF16 ? run_type<bf16>(sh.V, c->store, a, st)
                                              : run_type<float>(sh.V, c->store, a, st);
  if (e == hipSuccess) return CRA_OK;
  char msg[256];
  snprintf(msg, sizeof(msg), "cra_cache_append: %s", hipGetErrorString(e));
  return err(CRA_E_HIP, msg);
}

}  // extern "C"
