// Rotary positions and the norm of heads: arguments of a launch and the pieces of a
// row's work, shared by the operators over tensors (cra_rotary.hip) and over a paged
// cache (cra_append.hip).
#pragma once

#include <algorithm>

#include "../../include/cra.h"
#include "cra_common.hpp"
#include "cra_internal.hpp"

namespace cra {

constexpr int kTurnThreads = 256;  // a workgroup

struct TurnTensor {
  const void* x;   // forward: input; backward: the forward's input (norm) or dy
  const void* dy;  // backward with the norm
  void* y;         // output (backward: dx)
  const void* w;   // norm weights, or null
  float* partial;  // backward: [blocks, D] sums of dw, or null
  int64_t xsb, xsh, xss, dsb, dsh, dss, ysb, ysh, yss;
  int H;           // heads
  int blocks;      // workgroups of this tensor
  uint32_t items;  // rows: B * S * H
  FastDiv dH, dSH;
  int head_fast;   // neighbouring rows are heads of a token (else tokens)
};

struct TurnArgs {
  TurnTensor t[2];  // q, k
  int S, D, rot, interleaved, nturn, log_l;
  FastDiv dS;
  float eps, inv_d;
  int w_f32;  // weights are fp32 (else the rows' type)
  int neg;    // transposed rotation
  int norm;   // (cra_append.hip; the others are compiled with or without)
  const float* table;
  int64_t table_rows;
  const void* pos;
  int pos64;
  int64_t psb, pss;
};

template <typename T, int V>
struct Vec {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&f)[V]) {
  if constexpr (V * sizeof(T) == 16) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const Vec<T, V> x = __builtin_bit_cast(Vec<T, V>, u);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_f32(x.v[i]);
  } else if constexpr (V * sizeof(T) == 8) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const Vec<T, V> x = __builtin_bit_cast(Vec<T, V>, u);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_f32(x.v[i]);
  } else if constexpr (V * sizeof(T) == 4) {
    const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
    const Vec<T, V> x = __builtin_bit_cast(Vec<T, V>, u);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_f32(x.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_f32(p[i]);
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[V]) {
  Vec<T, V> x;
#pragma unroll
  for (int i = 0; i < V; ++i) x.v[i] = from_f32<T>(f[i]);
  if constexpr (V * sizeof(T) == 16)
    *reinterpret_cast<uint4*>(p) = __builtin_bit_cast(uint4, x);
  else if constexpr (V * sizeof(T) == 8)
    *reinterpret_cast<uint2*>(p) = __builtin_bit_cast(uint2, x);
  else if constexpr (V * sizeof(T) == 4)
    *reinterpret_cast<uint32_t*>(p) = __builtin_bit_cast(uint32_t, x);
  else
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = x.v[i];
}

// V floats of the table or of fp32 weights (aligned to min(16, 4 V) bytes).
template <int V>
__device__ __forceinline__ void load_floats(const float* p, float (&f)[V]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const float4 x = reinterpret_cast<const float4*>(p)[i];
      f[4 * i] = x.x, f[4 * i + 1] = x.y, f[4 * i + 2] = x.z, f[4 * i + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = p[i];
  }
}

// The two chunks of a unit: where they start, and which exist.
struct Unit {
  int ea, eb;
  bool turn, a, b;
};
template <int V>
__device__ __forceinline__ Unit unit_at(const TurnArgs& g, int u) {
  Unit n;
  n.turn = u < g.nturn;
  if (n.turn) {
    n.ea = g.interleaved ? 2 * u * V : u * V;
    n.eb = g.interleaved ? n.ea + V : (g.rot >> 1) + n.ea;
    n.a = n.b = true;
  } else {
    n.ea = g.rot + 2 * (u - g.nturn) * V;
    n.eb = n.ea + V;
    n.a = n.ea < g.D;
    n.b = n.eb < g.D;
  }
  return n;
}

// (a, b) <- R (a, b), or its transpose with sines of the other sign.
template <int V>
__device__ __forceinline__ void turn(float (&a)[V], float (&b)[V], const float (&c)[V],
                                     const float (&s)[V], bool interleaved) {
  if (V > 1 && interleaved) {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      const float a0 = a[2 * j], a1 = a[2 * j + 1], b0 = b[2 * j], b1 = b[2 * j + 1];
      a[2 * j] = a0 * c[j] - a1 * s[j];
      a[2 * j + 1] = a1 * c[j] + a0 * s[j];
      b[2 * j] = b0 * c[V / 2 + j] - b1 * s[V / 2 + j];
      b[2 * j + 1] = b1 * c[V / 2 + j] + b0 * s[V / 2 + j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float x = a[i], y = b[i];
      a[i] = x * c[i] - y * s[i];
      b[i] = y * c[i] + x * s[i];
    }
  }
}

__device__ __forceinline__ float turn_sum(float x, int log_l) {
  for (int o = 1 << log_l >> 1; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

struct Item {
  int b, s, h;
};
__device__ __forceinline__ Item item_at(const TurnArgs& g, const TurnTensor& t, uint32_t it) {
  Item r;
  if (t.head_fast) {
    const uint32_t tok = div_by(it, t.dH);
    r.h = (int)(it - tok * t.H);
    r.b = (int)div_by(tok, g.dS);
    r.s = (int)(tok - (uint32_t)r.b * g.S);
  } else {
    r.b = (int)div_by(it, t.dSH);
    const uint32_t rest = it - (uint32_t)r.b * g.S * t.H;
    r.h = (int)div_by(rest, g.dS);
    r.s = (int)(rest - (uint32_t)r.h * g.S);
  }
  return r;
}

// Table row of a token; -1 for a position outside the table (its turned
// elements become NaN: a position cannot be checked before the launch).
__device__ __forceinline__ int64_t table_row(const TurnArgs& g, const Item& it) {
  int64_t p = it.s;
  if (g.pos) {
    const int64_t o = it.b * g.psb + it.s * g.pss;
    p = g.pos64 ? static_cast<const int64_t*>(g.pos)[o] : static_cast<const int32_t*>(g.pos)[o];
  }
  return p >= 0 && p < g.table_rows ? p : -1;
}

template <int V, int U>
__device__ __forceinline__ void load_turns(const TurnArgs& g, int64_t row, int lane,
                                           const Unit (&un)[U], float (&c)[U][V], float (&s)[U][V]) {
#pragma unroll
  for (int j = 0; j < U; ++j) {
    if (un[j].turn && row >= 0) {
      const float* p = g.table + row * g.rot + (lane + j * 64) * V;
      load_floats<V>(p, c[j]);
      load_floats<V>(p + (g.rot >> 1), s[j]);
      if (g.neg) {
#pragma unroll
        for (int i = 0; i < V; ++i) s[j][i] = -s[j][i];
      }
    } else {
      const float nan = __builtin_nanf("");
#pragma unroll
      for (int i = 0; i < V; ++i) c[j][i] = s[j][i] = nan;
    }
  }
}

template <typename T, int V, int U>
__device__ __forceinline__ void load_weights(const TurnArgs& g, const TurnTensor& t,
                                             const Unit (&un)[U], float (&wa)[U][V],
                                             float (&wb)[U][V]) {
#pragma unroll
  for (int j = 0; j < U; ++j) {
#pragma unroll
    for (int i = 0; i < V; ++i) wa[j][i] = wb[j][i] = 1.f;
    if (!t.w) continue;
    if (g.w_f32) {
      const float* w = static_cast<const float*>(t.w);
      if (un[j].a) load_floats<V>(w + un[j].ea, wa[j]);
      if (un[j].b) load_floats<V>(w + un[j].eb, wb[j]);
    } else {
      const T* w = static_cast<const T*>(t.w);
      if (un[j].a) load_vec<T, V>(w + un[j].ea, wa[j]);
      if (un[j].b) load_vec<T, V>(w + un[j].eb, wb[j]);
    }
  }
}

// One chunk pair of row p; absent chunks read as zeros.
template <typename T, int V>
__device__ __forceinline__ void load_pair(const T* p, const Unit& u, bool on, float (&a)[V],
                                          float (&b)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) a[i] = b[i] = 0.f;
  if (on && u.a) load_vec<T, V>(p + u.ea, a);
  if (on && u.b) load_vec<T, V>(p + u.eb, b);
}

inline bool ptr_ok(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
inline bool strides_ok(const cra_tensor& t, int v) { return t.sb % v == 0 && t.sh % v == 0 && t.ss % v == 0; }

struct TurnShape {
  int V, U, log_l, units;
};

// Elements a chunk: the widest load of at most 16 bytes that divides the
// halves of the turned part, the rest of the row and every row's address.
inline TurnShape turn_shape(const cra_turn* p, const cra_tensor* const* ts, int n, const void* const* ws) {
  const int esz = p->dtype == CRA_F32 ? 4 : 2;
  int V = 16 / esz;
  auto fits = [&](int v) {
    if (p->rot % (2 * v) || (p->D - p->rot) % v) return false;
    for (int i = 0; i < n; ++i)
      if (!ptr_ok(ts[i]->ptr, v * esz) || !strides_ok(*ts[i], v)) return false;
    for (int i = 0; i < 2; ++i)
      if (ws[i] && !ptr_ok(ws[i], std::min(16, v * (p->weight_dtype == CRA_F32 ? 4 : esz)))) return false;
    return p->rot == 0 || ptr_ok(p->table, std::min(16, 4 * v));
  };
  while (V > 1 && !fits(V)) V >>= 1;
  TurnShape s;
  s.V = V;
  s.units = p->rot / (2 * V) + ((p->D - p->rot) + 2 * V - 1) / (2 * V);
  s.log_l = 0;
  while (s.log_l < 6 && (1 << s.log_l) < s.units) ++s.log_l;
  if (V == 1) s.log_l = 6;  // two units a lane
  s.U = V == 1 ? 2 : 1;
  return s;
}

inline void fill_args(TurnArgs& g, const cra_turn* p, const TurnShape& sh) {
  g = TurnArgs{};
  g.S = p->S;
  g.D = p->D;
  g.rot = p->rot;
  g.interleaved = p->interleaved != 0;
  g.nturn = p->rot / (2 * sh.V);
  g.log_l = sh.log_l;
  g.dS = fast_div(p->S);
  g.eps = p->eps;
  g.inv_d = 1.f / p->D;
  g.w_f32 = p->weight_dtype == CRA_F32;
  g.table = p->table;
  g.table_rows = p->table_rows;
  g.pos = p->positions;
  g.pos64 = p->positions_64;
  g.psb = p->psb;
  g.pss = p->pss;
}

inline void fill_tensor(TurnTensor& t, const cra_turn* p, const TurnShape& sh, int H, const cra_tensor& x,
                 const cra_tensor* dy, const cra_tensor& y, const void* w) {
  t.x = x.ptr;
  t.xsb = x.sb, t.xsh = x.sh, t.xss = x.ss;
  if (dy) t.dy = dy->ptr, t.dsb = dy->sb, t.dsh = dy->sh, t.dss = dy->ss;
  t.y = y.ptr;
  t.ysb = y.sb, t.ysh = y.sh, t.yss = y.ss;
  t.w = w;
  t.H = H;
  t.items = (uint32_t)p->B * p->S * H;
  t.dH = fast_div(H);
  t.dSH = fast_div((uint32_t)p->S * H);
  t.head_fast = y.sh < y.ss;
  const int slots = kTurnThreads >> sh.log_l;
  t.blocks = (int)((t.items + slots - 1) / slots);
}

// Checks of the C ABI (CRA_OK or an error with its text set).
int check_turn(const cra_turn* p);

}  // namespace cra
