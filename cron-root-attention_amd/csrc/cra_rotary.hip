// Rotary positions of query and key heads, alone or behind a norm of each head
// (forward and backward), and the C ABI front end of both.
//
// A head row x of D elements at position p (fp32 arithmetic, one rounding):
//   z = x                                      (rotation alone)
//   z = x * r * w,  r = 1 / sqrt(mean(x^2) + eps)   (with the norm; w may be absent)
//   y_a = z_a c_i - z_b s_i,  y_b = z_b c_i + z_a s_i   for the pairs (a, b) of
//   the first `rot` elements, (i, i + rot/2) or interleaved (2i, 2i + 1), with
//   c_i, s_i of row p of the table; elements from `rot` on pass.
// Backward: dz = the transposed rotation of dy (s -> -s), and with the norm
//   dw = sum over rows of dz * xhat,  xhat = x r,
//   dx = r (g - xhat mean(g xhat)),  g = dz * w.
//
// Bound by memory: x in, y out (backward: x and dy in, dx out): S=32768 H=16/4 D=128
// bf16 with the norm 73 us (4.8 TB/s) and 122 us + 6 us for dw (4.3 TB/s). A row belongs
// to L lanes of a wave, each with the two V-element chunks of a pair of 16-byte
// (or 8-, 4-byte) loads, so the rotation needs no exchange between lanes and
// the norm's sum is log2(L) shuffles. Neighbouring rows of a wave are heads or
// tokens, whichever lie closer in memory; the table row of a token is read again
// for each head, from the caches. One row a thread: with several (table row and
// weights loaded once for them) the registers cost more waves than the loads
// save (S=32768 H=16/4 D=128 bf16, a training step with 1, 2, 4 heads a thread in
// the backward: 218, 240, 270 us; in the forward 219, 217, 218).
#include <stdio.h>

#include <algorithm>

#include "../../include/cra.h"
#include "cra_common.hpp"
#include "cra_internal.hpp"

namespace cra {

int set_error(int code, const char* msg);

namespace {

constexpr int kThreads = 256;      // a workgroup
constexpr int kMaxPartials = 2048;  // workgroups (and partial rows) of a backward with weights

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

__device__ __forceinline__ float lanes_sum(float x, int log_l) {
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

// V elements a chunk, U units a lane (more than one only for V = 1).
template <typename T, int V, int U, bool NORM>
__global__ __launch_bounds__(kThreads) void turn_fwd_kernel(TurnArgs g) {
  const bool second = (int)blockIdx.x >= g.t[0].blocks;
  const TurnTensor& t = g.t[second];
  const uint32_t block = blockIdx.x - (second ? g.t[0].blocks : 0);
  const int lane = threadIdx.x & ((1 << g.log_l) - 1), slot = threadIdx.x >> g.log_l;
  const uint32_t it = block * (kThreads >> g.log_l) + slot;
  const bool on = it < t.items;
  const Item im = item_at(g, t, on ? it : t.items - 1);
  Unit un[U];
#pragma unroll
  for (int j = 0; j < U; ++j) un[j] = unit_at<V>(g, lane + 64 * j);

  const T* x = static_cast<const T*>(t.x) + im.b * t.xsb + im.s * t.xss + im.h * t.xsh;
  float a[U][V], b[U][V];
#pragma unroll
  for (int j = 0; j < U; ++j) load_pair<T, V>(x, un[j], on, a[j], b[j]);
  float c[U][V], s[U][V], wa[U][V], wb[U][V];
  load_turns<V, U>(g, table_row(g, im), lane, un, c, s);
  if (NORM) {
    load_weights<T, V, U>(g, t, un, wa, wb);
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < U; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) ss += a[j][i] * a[j][i] + b[j][i] * b[j][i];
    const float r = rsqrtf(lanes_sum(ss, g.log_l) * g.inv_d + g.eps);
#pragma unroll
    for (int j = 0; j < U; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        a[j][i] *= r * wa[j][i];
        b[j][i] *= r * wb[j][i];
      }
  }
  if (!on) return;
  T* y = static_cast<T*>(t.y) + im.b * t.ysb + im.s * t.yss + im.h * t.ysh;
#pragma unroll
  for (int j = 0; j < U; ++j) {
    if (un[j].turn) turn<V>(a[j], b[j], c[j], s[j], g.interleaved);
    if (un[j].a) store_vec<T, V>(y + un[j].ea, a[j]);
    if (un[j].b) store_vec<T, V>(y + un[j].eb, b[j]);
  }
}

// Backward of norm + rotation. The workgroups of a tensor stride over its
// rows; each thread keeps the sums of dw of its chunks, added over the
// workgroup's rows in a fixed order and stored as one partial row.
template <typename T, int V, int U>
__global__ __launch_bounds__(kThreads) void turn_bwd_kernel(TurnArgs g) {
  __shared__ float red[kThreads * 2 * V * U];
  const bool second = (int)blockIdx.x >= g.t[0].blocks;
  const TurnTensor& t = g.t[second];
  const uint32_t block = blockIdx.x - (second ? g.t[0].blocks : 0);
  const int lane = threadIdx.x & ((1 << g.log_l) - 1), slot = threadIdx.x >> g.log_l;
  const int slots = kThreads >> g.log_l;
  Unit un[U];
#pragma unroll
  for (int j = 0; j < U; ++j) un[j] = unit_at<V>(g, lane + 64 * j);
  float wa[U][V], wb[U][V], da[U][V], db[U][V];
  load_weights<T, V, U>(g, t, un, wa, wb);
#pragma unroll
  for (int j = 0; j < U; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) da[j][i] = db[j][i] = 0.f;

  // every thread of the workgroup takes the same number of turns (the shuffles
  // need whole waves)
  for (uint32_t base = block * slots; base < t.items; base += t.blocks * slots) {
    const uint32_t it = base + slot;
    const bool on = it < t.items;
    const Item im = item_at(g, t, on ? it : t.items - 1);
    const T* x = static_cast<const T*>(t.x) + im.b * t.xsb + im.s * t.xss + im.h * t.xsh;
    const T* dy = static_cast<const T*>(t.dy) + im.b * t.dsb + im.s * t.dss + im.h * t.dsh;
    float xa[U][V], xb[U][V], ga[U][V], gb[U][V], c[U][V], s[U][V];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      load_pair<T, V>(x, un[j], on, xa[j], xb[j]);
      load_pair<T, V>(dy, un[j], on, ga[j], gb[j]);
    }
    load_turns<V, U>(g, table_row(g, im), lane, un, c, s);
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < U; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) ss += xa[j][i] * xa[j][i] + xb[j][i] * xb[j][i];
    // 0 behind the last row: its zeros times rsqrt(0 + eps) are NaN where eps is 0, and
    // the sums of dw go on below
    const float mean = lanes_sum(ss, g.log_l) * g.inv_d, r = on ? rsqrtf(mean + g.eps) : 0.f;
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (un[j].turn && on) turn<V>(ga[j], gb[j], c[j], s[j], g.interleaved);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        xa[j][i] *= r;
        xb[j][i] *= r;
        da[j][i] += ga[j][i] * xa[j][i];
        db[j][i] += gb[j][i] * xb[j][i];
        ga[j][i] *= wa[j][i];
        gb[j][i] *= wb[j][i];
        dot += ga[j][i] * xa[j][i] + gb[j][i] * xb[j][i];
      }
    }
    dot = lanes_sum(dot, g.log_l) * g.inv_d;
    if (!on) continue;
    T* y = static_cast<T*>(t.y) + im.b * t.ysb + im.s * t.yss + im.h * t.ysh;
#pragma unroll
    for (int j = 0; j < U; ++j) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        ga[j][i] = r * (ga[j][i] - xa[j][i] * dot);
        gb[j][i] = r * (gb[j][i] - xb[j][i] * dot);
      }
      if (un[j].a) store_vec<T, V>(y + un[j].ea, ga[j]);
      if (un[j].b) store_vec<T, V>(y + un[j].eb, gb[j]);
    }
  }
  if (!t.partial) return;
#pragma unroll
  for (int j = 0; j < U; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (un[j].a) red[slot * g.D + un[j].ea + i] = da[j][i];
      if (un[j].b) red[slot * g.D + un[j].eb + i] = db[j][i];
    }
  __syncthreads();
  for (int e = threadIdx.x; e < g.D; e += kThreads) {
    float sum = 0.f;
    for (int i = 0; i < slots; ++i) sum += red[i * g.D + e];
    t.partial[(int64_t)block * g.D + e] = sum;
  }
}

// dw = sum of the partial rows: 64 interleaved sequences of them, each in row
// order, then the sequences in order. One workgroup: 16 columns of one tensor.
constexpr int kDwSeqs = 64;
template <typename W>
__global__ __launch_bounds__(16 * kDwSeqs) void turn_dw_kernel(const float* pq, int nq, W* dwq,
                                                               const float* pk, int nk, W* dwk, int D) {
  __shared__ float red[kDwSeqs][17];
  const float* p = blockIdx.y ? pk : pq;
  W* dw = blockIdx.y ? dwk : dwq;
  const int n = blockIdx.y ? nk : nq;
  if (!dw) return;
  const int col = threadIdx.x & 15, seq = threadIdx.x >> 4, e = blockIdx.x * 16 + col;
  float sum = 0.f;
  if (e < D) {
#pragma unroll 8
    for (int r = seq; r < n; r += kDwSeqs) sum += p[(int64_t)r * D + e];
  }
  red[seq][col] = sum;
  __syncthreads();
  if (seq == 0 && e < D) {
    for (int i = 1; i < kDwSeqs; ++i) sum += red[i][col];
    dw[e] = from_f32<W>(sum);
  }
}

int err(int code, const char* msg) { return set_error(code, msg); }

int check_turn(const cra_turn* p) {
  if (!p) return err(CRA_E_INVALID, "turn is NULL");
  if (p->dtype != CRA_F16 && p->dtype != CRA_BF16 && p->dtype != CRA_F32)
    return err(CRA_E_DTYPE, "unknown dtype code");
  if (p->B < 1 || p->S < 1 || p->H_q < 1 || p->H_kv < 0)
    return err(CRA_E_INVALID, "B, S and H_q must be >= 1, H_kv >= 0");
  if (p->D < 1) return err(CRA_E_INVALID, "head dim must be >= 1");
  if (p->D > 256) return err(CRA_E_UNSUPPORTED, "head dim above 256 is not built");
  if (p->rot < 0 || p->rot > p->D || p->rot % 2)
    return err(CRA_E_INVALID, "rot must be even, from 0 to the head dim");
  if (p->rot > 0 && (!p->table || p->table_rows < 1))
    return err(CRA_E_INVALID, "a rotation needs a table");
  if (p->norm != 0 && p->norm != 1) return err(CRA_E_INVALID, "norm must be 0 or 1");
  if (p->norm && !(p->eps >= 0.f)) return err(CRA_E_INVALID, "eps must be >= 0");
  if (p->norm && p->weight_dtype != p->dtype && p->weight_dtype != CRA_F32)
    return err(CRA_E_DTYPE, "weights must be of the rows' type or fp32");
  if ((int64_t)p->B * p->S * std::max(p->H_q, p->H_kv) > (int64_t)1 << 31)
    return err(CRA_E_INVALID, "B*S*H exceeds 2^31");
  return CRA_OK;
}

bool ptr_ok(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
bool strides_ok(const cra_tensor& t, int v) { return t.sb % v == 0 && t.sh % v == 0 && t.ss % v == 0; }

struct Shape {
  int V, U, log_l, units;
};

// Elements a chunk: the widest load of at most 16 bytes that divides the
// halves of the turned part, the rest of the row and every row's address.
Shape shape_of(const cra_turn* p, const cra_tensor* const* ts, int n, const void* const* ws) {
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
  Shape s;
  s.V = V;
  s.units = p->rot / (2 * V) + ((p->D - p->rot) + 2 * V - 1) / (2 * V);
  s.log_l = 0;
  while (s.log_l < 6 && (1 << s.log_l) < s.units) ++s.log_l;
  if (V == 1) s.log_l = 6;  // two units a lane
  s.U = V == 1 ? 2 : 1;
  return s;
}

void fill_args(TurnArgs& g, const cra_turn* p, const Shape& sh) {
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

void fill_tensor(TurnTensor& t, const cra_turn* p, const Shape& sh, int H, const cra_tensor& x,
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
  const int slots = kThreads >> sh.log_l;
  t.blocks = (int)((t.items + slots - 1) / slots);
}

template <typename F>
hipError_t with_type(int dtype, F f) {
  return dtype == CRA_F16 ? f(f16()) : dtype == CRA_BF16 ? f(bf16()) : f(float());
}

// A launch holds at most 2^32 threads a dimension.
bool grid_fits(const TurnArgs& g) {
  return ((int64_t)g.t[0].blocks + g.t[1].blocks) * kThreads < (int64_t)1 << 32;
}

template <typename T, int V, int U>
hipError_t run_fwd(const TurnArgs& g, bool norm, hipStream_t st) {
  const int grid = g.t[0].blocks + g.t[1].blocks;
  if (norm)
    turn_fwd_kernel<T, V, U, true><<<grid, kThreads, 0, st>>>(g);
  else
    turn_fwd_kernel<T, V, U, false><<<grid, kThreads, 0, st>>>(g);
  return hipGetLastError();
}
template <typename T, int V, int U>
hipError_t run_bwd(const TurnArgs& g, hipStream_t st) {
  turn_bwd_kernel<T, V, U><<<g.t[0].blocks + g.t[1].blocks, kThreads, 0, st>>>(g);
  return hipGetLastError();
}

template <bool BWD>
hipError_t launch(int dtype, const Shape& s, const TurnArgs& g, bool norm, hipStream_t st) {
  return with_type(dtype, [&](auto z) {
    using T = decltype(z);
    auto go = [&](auto v, auto u) {
      constexpr int V = decltype(v)::value, U = decltype(u)::value;
      if constexpr (BWD)
        return run_bwd<T, V, U>(g, st);
      else
        return run_fwd<T, V, U>(g, norm, st);
    };
    using I1 = std::integral_constant<int, 1>;
    if constexpr (sizeof(T) == 2)
      if (s.V == 8) return go(std::integral_constant<int, 8>(), I1());
    if (s.V == 4) return go(std::integral_constant<int, 4>(), I1());
    if (s.V == 2) return go(std::integral_constant<int, 2>(), I1());
    return go(I1(), std::integral_constant<int, 2>());
  });
}

int hip_err(hipError_t e, const char* where) {
  if (e == hipSuccess) return CRA_OK;
  char msg[256];
  snprintf(msg, sizeof(msg), "%s: %s", where, hipGetErrorString(e));
  return err(CRA_E_HIP, msg);
}

int check_rows(const char* name, const cra_tensor& t, int esz) {
  if (t.ptr && reinterpret_cast<uintptr_t>(t.ptr) % esz == 0) return CRA_OK;
  char msg[96];
  snprintf(msg, sizeof(msg), "%s: NULL or misaligned pointer", name);
  return err(t.ptr ? CRA_E_LAYOUT : CRA_E_INVALID, msg);
}

// Workgroups of the two tensors of a backward with the norm: at most
// kMaxPartials together, shared by their items.
void share_blocks(TurnArgs& g) {
  const int64_t want = (int64_t)g.t[0].blocks + g.t[1].blocks;
  if (want <= kMaxPartials) return;
  for (TurnTensor& t : g.t)
    if (t.blocks) t.blocks = std::max<int>(1, (int)(t.blocks * (int64_t)(kMaxPartials - 1) / want));
}

}  // namespace
}  // namespace cra

using namespace cra;

extern "C" {

int cra_rotary(const cra_turn* p, cra_tensor q, cra_tensor k, const void* wq, const void* wk,
               cra_tensor yq, cra_tensor yk, int32_t transpose, void* stream) {
  if (int e = check_turn(p)) return e;
  if (transpose && p->norm) return err(CRA_E_INVALID, "transpose is for the rotation alone");
  const int esz = p->dtype == CRA_F32 ? 4 : 2;
  const cra_tensor* ts[4] = {&q, &yq, &k, &yk};
  const char* names[4] = {"q", "q output", "k", "k output"};
  const int n = p->H_kv ? 4 : 2;
  for (int i = 0; i < n; ++i)
    if (int e = check_rows(names[i], *ts[i], esz)) return e;
  const void* ws[2] = {p->norm ? wq : nullptr, p->norm && p->H_kv ? wk : nullptr};
  const Shape sh = shape_of(p, ts, n, ws);
  TurnArgs g;
  fill_args(g, p, sh);
  g.neg = transpose != 0;
  fill_tensor(g.t[0], p, sh, p->H_q, q, nullptr, yq, ws[0]);
  if (p->H_kv) fill_tensor(g.t[1], p, sh, p->H_kv, k, nullptr, yk, ws[1]);
  if (!grid_fits(g)) return err(CRA_E_INVALID, "too many rows for one launch");
  return hip_err(launch<false>(p->dtype, sh, g, p->norm, (hipStream_t)stream), "cra_rotary");
}

size_t cra_rotary_bwd_workspace_bytes(const cra_turn* p) {
  return check_turn(p) ? 0 : (size_t)kMaxPartials * p->D * sizeof(float);
}

int cra_norm_rotary_bwd(const cra_turn* p, cra_tensor q, cra_tensor k, const void* wq,
                        const void* wk, cra_tensor dyq, cra_tensor dyk, cra_tensor dq,
                        cra_tensor dk, void* dwq, void* dwk, void* workspace,
                        size_t workspace_bytes, void* stream) {
  if (int e = check_turn(p)) return e;
  if (!p->norm) return err(CRA_E_INVALID, "without the norm the backward is cra_rotary with transpose");
  const int esz = p->dtype == CRA_F32 ? 4 : 2;
  const cra_tensor* ts[6] = {&q, &dyq, &dq, &k, &dyk, &dk};
  const char* names[6] = {"q", "dyq", "dq", "k", "dyk", "dk"};
  const int n = p->H_kv ? 6 : 3;
  for (int i = 0; i < n; ++i)
    if (int e = check_rows(names[i], *ts[i], esz)) return e;
  if (!p->H_kv) wk = dwk = nullptr;
  if ((dwq && !wq) || (dwk && !wk)) return err(CRA_E_INVALID, "dw without weights");
  const void* ws[2] = {wq, wk};
  Shape sh = shape_of(p, ts, n, ws);
  const bool sums = dwq || dwk;
  if (sums) {
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16)
      return err(CRA_E_INVALID, "workspace: NULL or misaligned pointer");
    if (workspace_bytes < cra_rotary_bwd_workspace_bytes(p))
      return err(CRA_E_WORKSPACE, "workspace too small (cra_rotary_bwd_workspace_bytes)");
  }
  TurnArgs g;
  fill_args(g, p, sh);
  g.neg = 1;
  fill_tensor(g.t[0], p, sh, p->H_q, q, &dyq, dq, wq);
  if (p->H_kv) fill_tensor(g.t[1], p, sh, p->H_kv, k, &dyk, dk, wk);
  share_blocks(g);
  float* part = static_cast<float*>(workspace);
  if (dwq) g.t[0].partial = part;
  if (dwk) g.t[1].partial = part + (int64_t)g.t[0].blocks * p->D;
  hipStream_t st = (hipStream_t)stream;
  if (int e = hip_err(launch<true>(p->dtype, sh, g, true, st), "cra_norm_rotary_bwd")) return e;
  if (!sums) return CRA_OK;
  const dim3 grid((p->D + 15) / 16, 2);
  return hip_err(with_type(p->weight_dtype, [&](auto z) {
    using W = decltype(z);
    turn_dw_kernel<W><<<grid, 16 * kDwSeqs, 0, st>>>(g.t[0].partial, g.t[0].blocks, static_cast<W*>(dwq),
                                            g.t[1].partial, g.t[1].blocks, static_cast<W*>(dwk), p->D);
    return hipGetLastError();
  }), "cra_norm_rotary_bwd (weights)");
}

}  // extern "C"
