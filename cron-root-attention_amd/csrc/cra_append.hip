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
// Bound by memory, single tokens by that chain and the launch.
#include <stdio.h>

#include <type_traits>

#include "cra_cache_dev.hpp"
#include "cra_common.hpp"
#include "cra_internal.hpp"
#include "cra_paged.hpp"
#include "cra_turn_dev.hpp"

namespace cra {

int set_error(int code, const char* msg);

namespace {

constexpr int kThreads = kTurnThreads;

struct AppendArgs {
  TurnArgs g;   // t[0]: q into y; t[1]: k, into the cache
  PagedView c;
  const void* v;
  int64_t vsb, vsh, vss;
  float *k_norm, *k_scale, *v_scale;
  int Ds, log_w;  // columns stored, lanes of a row as it is stored
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

template <typename T, int STORE, int V>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a) {
  __shared__ __attribute__((aligned(16))) T held[kThreads * 2 * V];  // rows of k, turned
  __shared__ uint32_t dst[kThreads];
  const TurnArgs& g = a.g;
  const bool kv = (int)blockIdx.x < g.t[1].blocks;
  const TurnTensor& t = g.t[kv];
  const uint32_t block = blockIdx.x - (kv ? 0 : g.t[1].blocks);
  const int log_l = g.log_l, lane = threadIdx.x & ((1 << log_l) - 1), slot = threadIdx.x >> log_l;
  const int rows = kThreads >> log_l;
  const uint32_t it = block * rows + slot;
  const bool on = it < t.items;
  const Item im = item_at(g, t, on ? it : t.items - 1);
  Unit un[1] = {unit_at<V>(g, lane)};
  const T* x = static_cast<const T*>(t.x) + im.b * t.xsb + im.s * t.xss + im.h * t.xsh;
  float p[1][V], q[1][V];
  load_pair<T, V>(x, un[0], on, p[0], q[0]);

  // rows of v: as they are stored, up to two a thread (a stored row takes at most
  // twice the lanes of a turned one)
  const int wlane = threadIdx.x & ((1 << a.log_w) - 1), wrow = threadIdx.x >> a.log_w;
  const int wrows = kThreads >> a.log_w;
  Row8<T> vr[2];
  if (kv) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int i = 0; i < (int)(sizeof(T) / 2); ++i) vr[j].w[i] = make_uint4(0, 0, 0, 0);
      const int r = wrow + j * wrows;
      const uint32_t at = block * rows + r;
      if (r >= rows || at >= t.items || wlane * 8 >= g.D) continue;
      const Item vi = item_at(g, t, at);
      const uint4* vp = reinterpret_cast<const uint4*>(
          static_cast<const T*>(a.v) + vi.b * a.vsb + vi.h * a.vsh + vi.s * a.vss + wlane * 8);
#pragma unroll
      for (int i = 0; i < (int)(sizeof(T) / 2); ++i) vr[j].w[i] = vp[i];
    }
  }

  const Place pl = place_of(a.c, im, lane, log_l);
  const int64_t at = pl.b < 0 ? -1 : (int64_t)a.c.lens[pl.b] - pl.count + pl.t;
  const int64_t turn_row = g.pos ? table_row(g, im) : at < g.table_rows ? at : -1;
  float c[1][V], s[1][V], wp[1][V], wq[1][V];
  load_turns<V, 1>(g, turn_row, lane, un, c, s);
  if (g.norm) {
    load_weights<T, V, 1>(g, t, un, wp, wq);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) ss += p[0][i] * p[0][i] + q[0][i] * q[0][i];
    const float r = rsqrtf(turn_sum(ss, log_l) * g.inv_d + g.eps);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      p[0][i] *= r * wp[0][i];
      q[0][i] *= r * wq[0][i];
    }
  }
  if (un[0].turn) turn_rows<V>(p[0], q[0], c[0], s[0], g.interleaved);
  if (!kv) {
    if (!on) return;
    T* y = static_cast<T*>(t.y) + im.b * t.ysb + im.s * t.yss + im.h * t.ysh;
    if (pl.b < 0) {  // padding
#pragma unroll
      for (int i = 0; i < V; ++i) p[0][i] = q[0][i] = 0.f;
    }
    if (un[0].a) store_vec<T, V>(y + un[0].ea, p[0]);
    if (un[0].b) store_vec<T, V>(y + un[0].eb, q[0]);
    return;
  }

  T* mine = held + slot * (2 * V << log_l);
  if (un[0].a) store_vec<T, V>(mine + un[0].ea, p[0]);
  if (un[0].b) store_vec<T, V>(mine + un[0].eb, q[0]);
  if (lane == 0) {
    const int row = pl.b < 0 ? -1 : write_row(a.c.lens[pl.b], pl.count, pl.t, a.c.pages_per_seq, a.c.log_page);
    dst[slot] = on && row >= 0 ? seq_row(a.c.table + pl.b * a.c.table_stride, row, a.c.num_pages,
                                         a.c.H_kv, a.c.log_page, im.h)
                               : kNoRow;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = wrow + j * wrows;
    if (r >= rows || dst[r] == kNoRow) continue;  // whole rows: the exchanges stay within one
    const bool have = wlane * 8 < g.D;
    Row8<T> kr;
    const uint4* kp = reinterpret_cast<const uint4*>(held + r * (2 * V << log_l) + wlane * 8);
    float kx[8], vx[8];
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) kr.w[i] = have ? kp[i] : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      kx[i] = to_f32(reinterpret_cast<const T*>(kr.w)[i]);
      vx[i] = to_f32(reinterpret_cast<const T*>(vr[j].w)[i]);
    }
    const float norm = lanes_sum(square_sum(kx), a.log_w);
    if (wlane == 0) a.k_norm[dst[r]] = norm;
    store_row<T, STORE>(kx, kr, const_cast<char*>(a.c.k), a.k_scale, dst[r], a.Ds, wlane, a.log_w);
    store_row<T, STORE>(vx, vr[j], const_cast<char*>(a.c.v), a.v_scale, dst[r], a.Ds, wlane, a.log_w);
  }
}

int err(int code, const char* msg) { return set_error(code, msg); }

template <typename T, int STORE, int V>
hipError_t run(const AppendArgs& a, hipStream_t st) {
  append_kernel<T, STORE, V><<<a.g.t[0].blocks + a.g.t[1].blocks, kThreads, 0, st>>>(a);
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
  const TurnShape sh = turn_shape(p, ts, 3, ws);
  if (sh.V < 2) return err(CRA_E_UNSUPPORTED, "weights or turned halves between 4-byte steps are not built");
  AppendArgs a{};
  fill_args(a.g, p, sh);
  fill_tensor(a.g.t[0], p, sh, p->H_q, q, nullptr, yq, ws[0]);
  fill_tensor(a.g.t[1], p, sh, p->H_kv, k, nullptr, k, ws[1]);
  a.g.t[1].y = nullptr;
  a.g.norm = p->norm != 0;
  a.c = paged_view(c, b);
  a.v = v.ptr, a.vsb = v.sb, a.vsh = v.sh, a.vss = v.ss;
  a.k_norm = c->k_norm, a.k_scale = c->k_scale, a.v_scale = c->v_scale;
  a.Ds = c->D;
  while ((8 << a.log_w) < c->D) ++a.log_w;
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
