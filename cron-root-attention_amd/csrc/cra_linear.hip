// Products in 8-bit floating point: y = x w^T (+ bias), both operands e4m3 codes with a
// power-of-two scale, x for each row and block of 128 columns, w for each block of
// 128 x 128; and the bringing of rows and weights into that form. C ABI front end.
//
// Block b of a row with m = max |x| is held as codes c and a scale s:
//   s = the smallest power of two with m <= 448 s, at least 2^-126;  c = RNE(x / s)
// (x / s and c s are exact but for that rounding, whatever the block's magnitude), and
//   y_ij = sum_b s_ib t_jb (sum_{k in b} c_ik d_jk) + bias_j.
// The scale is its exponent byte, as the matrix instruction takes it: the 16x16x128 MFMA
// multiplies by both operands' scales on the way, so a block of 128 is one instruction
// and no scaling is left to the VALU. A block that holds an infinity or NaN gets NaN
// codes: its row of y is NaN.
//
// Sums: the 8-bit MFMA cuts the products it adds at about 2^-16 of the largest (measured:
// 1.4e-5 of the result's norm for random operands, whatever K; its accumulator is fp32).
// That is below the rounding of 16-bit results (fp16: 2e-4). fp32 results take the codes
// widened to bf16 with their scales (exact: w_shift) through the bf16 MFMA instead, at half
// its rate or less: 3e-7.
#include <stdio.h>

#include <algorithm>
#include <type_traits>

#include "../../include/cra.h"
#include "cra_cache_dev.hpp"
#include "cra_common.hpp"
#include "cra_internal.hpp"
#include "cra_paged.hpp"

namespace cra {

int set_error(int code, const char* msg);

namespace {

constexpr int kBlock = 128;
typedef int i32x8 __attribute__((ext_vector_type(8)));

__host__ __device__ inline int up(int64_t n, int m) { return (int)((n + m - 1) / m); }

// ---------------------------------------------------------------------------
// Into 8 bits.
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, bool wide, float (&x)[8]) {
  if (wide) {
    const Row8<T> r = *reinterpret_cast<const Row8<T>*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(reinterpret_cast<const T*>(r.w)[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < n ? to_f32(p[i]) : 0.f;
  }
}
__device__ __forceinline__ uint32_t largest(const float (&x)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  return m;
}
// Codes of eight elements of a block whose largest magnitude has the bits m, and the
// block's exponent byte.
__device__ __forceinline__ uint2 codes8(const float (&x)[8], uint32_t m, uint8_t& e) {
  const float s = row_scale<kE4M3>(m);
  e = s == s ? (uint8_t)(__float_as_uint(s) >> 23) : 127;
  return s == s ? make_uint2(codes4<kE4M3>(x, s), codes4<kE4M3>(x + 4, s))
                : make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
}

struct RowsArgs {
  const void* x;
  int64_t ldx;
  uint8_t* codes;   // [M, 128 Kb]
  uint8_t* scales;  // [M, Ks]
  uint32_t blocks;  // M * Kb
  int K, Kb, Ks;
  FastDiv dKb;
  int wide;         // rows lie between 16-byte addresses
};

// 16 lanes a block of a row, eight elements each.
template <typename T>
__global__ __launch_bounds__(256) void rows_kernel(RowsArgs a) {
  const uint32_t i = blockIdx.x * 16u + (threadIdx.x >> 4);
  if (i >= a.blocks) return;  // whole rows of lanes
  const uint32_t row = div_by(i, a.dKb);
  const int b = (int)(i - row * a.Kb), lane = threadIdx.x & 15, col = b * kBlock + lane * 8;
  float x[8];
  load8<T>(static_cast<const T*>(a.x) + row * a.ldx + col, a.K - col, a.wide && col + 8 <= a.K, x);
  uint8_t e;
  const uint2 c = codes8(x, lanes_max(largest(x), 4), e);
  *reinterpret_cast<uint2*>(a.codes + (int64_t)row * a.Kb * kBlock + col) = c;
  if (lane == 0) a.scales[(int64_t)row * a.Ks + b] = e;
}

// A workgroup a block of 128 x 128: two threads a row.
template <typename T>
__global__ __launch_bounds__(256) void weight_kernel(const T* w, int64_t ldw, int N, int K, int Kb, int Ks,
                                                     int wide, uint8_t* codes, uint8_t* scales) {
  __shared__ uint32_t most[4];
  const int row = blockIdx.y * kBlock + (threadIdx.x >> 1);
  const int col0 = blockIdx.x * kBlock + (threadIdx.x & 1) * 64;
  float x[8][8];
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int col = col0 + 8 * j;
    load8<T>(w + (int64_t)min(row, N - 1) * ldw + col, row < N ? K - col : 0, wide && row < N && col + 8 <= K, x[j]);
    m = max(m, largest(x[j]));
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
  if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = m;
  __syncthreads();
  m = max(max(most[0], most[1]), max(most[2], most[3]));
  uint8_t e;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint2 c = codes8(x[j], m, e);
    if (row < N) *reinterpret_cast<uint2*>(codes + (int64_t)row * Kb * kBlock + col0 + 8 * j) = c;
  }
  if (threadIdx.x == 0) scales[(int64_t)blockIdx.y * Ks + blockIdx.x] = e;
}

// ---------------------------------------------------------------------------
// Products. A wave holds w as the MFMA's rows and x as its columns: a lane's four
// results are neighbours of one row of y.
// ---------------------------------------------------------------------------
struct LinearArgs {
  const void* x;       // rows as they are (few rows)
  int64_t ldx;
  const uint8_t *xc, *xs;  // codes [M, Kp] and exponents [M, Ks]
  const uint8_t *wc, *ws;  // codes [N, Kp] and exponents [ceil(N / 128), Ks]
  const void* bias;
  void* y;
  int64_t ldy;
  int64_t M;
  int N, K, Kb, Kp, Ks;  // blocks of a row; columns of codes; exponents of a row
  int tiles_m, tiles_n;
  int per;               // blocks of a piece of the tiles
  float* part;           // sums of pieces [piece, M, ldp], or null
  int64_t ldp;
  int wide_x, wide_y, wide_y8;  // rows of x between 16-byte addresses; four and eight results of y as one store
};

// 32 codes of a row of a block: the same columns for both operands, in any order.
struct Frag8 {
  uint4 lo, hi;
};

// One 16 x 16 x 128 step: rows of w, columns of x, exponents of both in byte 0.
__device__ __forceinline__ f32x4 mma8(f32x4 c, const Frag8& w, const Frag8& x, uint32_t sw, uint32_t sx) {
  i32x8 a, b;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i] = reinterpret_cast<const int*>(&w.lo)[i];
    a[4 + i] = reinterpret_cast<const int*>(&w.hi)[i];
    b[i] = reinterpret_cast<const int*>(&x.lo)[i];
    b[4 + i] = reinterpret_cast<const int*>(&x.hi)[i];
  }
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, (int)sw, 0, (int)sx);
}

// The codes as bf16 numbers, times 2^(e - 127).
struct Wide {
  Frag<bf16> f[4];
};
__device__ __forceinline__ Wide widen(const Frag8& c, uint32_t e) {
  const float s = __uint_as_float((e & 0xffu) << 23);
  Wide r;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t w = i < 4 ? reinterpret_cast<const uint32_t*>(&c.lo)[i] : reinterpret_cast<const uint32_t*>(&c.hi)[i - 4];
    uint32_t* o = reinterpret_cast<uint32_t*>(r.f[i / 2].w) + 2 * (i & 1);
    o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, s, false));
    o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, s, true));
  }
  return r;
}
__device__ __forceinline__ f32x4 mma_wide(f32x4 c, const Wide& w, const Wide& x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = mma(c, w.f[i], x.f[i]);
  return c;
}

// Codes reach down to 2^-9 and scales to 2^-126, bf16 to 2^-133, so one operand's scale goes
// into it four times as large and the other's a quarter (the product is the same): w's where
// its own is small (up to 2^-123; what x loses then is below 2^-200 in the product), else x's -
// unless a row of the wave stands too high for that (a scale from 2^118), and elements
// below 2^-133 beside it round to multiples of that. The power of two that w takes:
__device__ __forceinline__ int w_shift(uint32_t ew, bool high) {
  return (ew & 0xffu) <= 4u ? 2 : __any(high) ? 0 : -2;
}
__device__ __forceinline__ bool high_row(uint32_t ex) { return (ex & 0xffu) > 244u; }
__device__ __forceinline__ Wide widen_w(const Frag8& c, uint32_t ew, int shift) { return widen(c, (ew & 0xffu) + shift); }
__device__ __forceinline__ Wide widen_x(const Frag8& c, uint32_t ex, int shift) {
  return widen(c, max((int)(ex & 0xffu) - shift, 0));
}

// Four results of row m, columns n .. n + 3.
template <typename T>
__device__ __forceinline__ f32x4 bias4(const LinearArgs& a, int n) {
  const T* bias = static_cast<const T*>(a.bias);
  f32x4 b = f32x4{0.f, 0.f, 0.f, 0.f};
  if (bias) {
#pragma unroll
    for (int r = 0; r < 4; ++r) b[r] = to_f32(bias[min(n + r, a.N - 1)]);
  }
  return b;
}
template <typename T>
__device__ __forceinline__ void store4(const LinearArgs& a, int64_t m, int n, f32x4 c, f32x4 b) {
  if (m >= a.M || n >= a.N) return;
  T e[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) e[r] = from_f32<T>(c[r] + b[r]);
  T* p = static_cast<T*>(a.y) + m * a.ldy + n;
  if (a.wide_y) {
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(e);
    else
      *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(e);
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < a.N) p[r] = e[r];
  }
}

// ROWS x 128 codes in LDS, 16-byte chunks XOR-swizzled so that 16 lanes reading one chunk
// of 16 rows hit every bank once. A wave's instruction brings eight rows.
template <int ROWS, int NW>
struct CodeTile {
  static constexpr int kBytes = ROWS * kBlock;
  static constexpr int kPer = kBytes / 1024 / NW;  // instructions of a wave
  static_assert(kPer * NW * 1024 == kBytes && NW % 2 == 0, "the swizzle repeats every 16 rows");
  __device__ __forceinline__ static int off(int row, int chunk) {
    return row * kBlock + ((chunk ^ (row >> 1 & 7)) << 4);
  }
  __device__ __forceinline__ static int lane_off(int wave, int lane, int Kp) {
    const int row = wave * 8 + (lane >> 3);
    return row * Kp + (((lane & 7) ^ (row >> 1 & 7)) << 4);
  }
  // 32 codes of row 16 blk + lane % 16: chunks g and g + 4
  __device__ __forceinline__ static Frag8 frag(const char* lds, int blk, int lane) {
    const int row = lane & 15, g = lane >> 4;
    const char* p = lds + blk * 16 * kBlock;
    return Frag8{*reinterpret_cast<const uint4*>(p + off(row, g)), *reinterpret_cast<const uint4*>(p + off(row, g + 4))};
  }
};

// Tile of a workgroup: the dispatcher sends workgroup i to XCD i % 8; each XCD takes a
// contiguous eighth of the tiles, which go down four row tiles before the next column
// tile, so that its L2 holds what its workgroups share (16384 x 6144 x 4096 with four,
// eight, sixteen: 297, 316, 320 us).
__device__ __forceinline__ void tile_of(const LinearArgs& a, int& tm, int& tn) {
  const int all = a.tiles_m * a.tiles_n, x = blockIdx.x & 7, base = all >> 3, extra = all & 7;
  const int i = x * base + min(x, extra) + (blockIdx.x >> 3);
  constexpr int kDown = 4;
  const int group = i / (kDown * a.tiles_n), first = group * kDown, down = min(kDown, a.tiles_m - first);
  const int j = i - group * kDown * a.tiles_n;
  tn = __builtin_amdgcn_readfirstlane(j / down);  // what follows from them stays scalar
  tm = __builtin_amdgcn_readfirstlane(first + j - tn * down);
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// Buffer resource over `bytes` bytes at `base`, in scalar registers.
__device__ __forceinline__ u32x4 resource(const void* base, uint32_t bytes) {
  const uint64_t p = reinterpret_cast<uint64_t>(base);
  u32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((uint32_t)p);
  r[1] = __builtin_amdgcn_readfirstlane((uint32_t)(p >> 32) & 0xffffu);
  r[2] = __builtin_amdgcn_readfirstlane(bytes);
  r[3] = 0x00020000;
  return r;
}
__device__ __forceinline__ uint32_t lds_at(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}
// One load of every lane, 16 or 4 bytes each, from resource + off + soff to LDS, lane after
// lane. A row behind the resource's last byte loads as zeros: soff stays below one row.
template <int BYTES>
__device__ __forceinline__ void to_lds(uint32_t lds, u32x4 rsrc, int off, int soff) {
  static_assert(BYTES == 16 || BYTES == 4, "a lane's load");
  if constexpr (BYTES == 16)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :: "s"(lds), "v"(off), "s"(rsrc), "s"(soff) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds"
                 :: "s"(lds), "v"(off), "s"(rsrc), "s"(soff) : "memory", "m0");
}
// All but the newest N loads of the wave have landed, its LDS reads are done, and the other
// waves are as far.
template <int N>
__device__ __forceinline__ void wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
typedef const __attribute__((address_space(4))) uint32_t* ConstWords;  // read by scalar loads

// WM x WN waves of (16 FM) x (16 FN) results over LDS tiles of a block of 128 columns, in
// kStages stages: a block's loads run while the others are multiplied. Bound by the
// latency of those loads where a workgroup has few blocks, and by the matrix core and
// LDS reads (a fragment serves two to four MFMAs) where it has many. Few tiles are cut
// along K (gridDim.y), whose sums join_kernel adds in their order.
// Measured, bf16 with the rows' own way into 8 bits: 1024 x 4096 x 4096 (tiles of 128) 31.8 us,
// 512 (of 64) 23.7, 64 (of 64, K in eight pieces) 16; 16384 x 6144 x 4096 fp32 (of 256) 700-735; two stages and no pieces 42.5, 28.0, 19.
template <typename T, int WM, int WN, int FM, int FN, int kStages>
__global__ __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(WM * WN / 4)))
void linear_kernel(LinearArgs a) {
  constexpr bool kWide = std::is_same<T, float>::value;
  constexpr int NW = WM * WN, BM = 16 * FM * WM, BN = 16 * FN * WN;
  static_assert(16 * FN <= kBlock && kBlock % (16 * FN) == 0, "one exponent of w a wave");
  static_assert(16 * FM <= 64, "a wave's exponents of x are one load");
  using TX = CodeTile<BM, NW>;
  using TW = CodeTile<BN, NW>;
  constexpr int kOps = TX::kPer + TW::kPer + 1;  // loads of a block
  __shared__ __attribute__((aligned(1024))) char xt[kStages][TX::kBytes], wt[kStages][TW::kBytes];
  __shared__ uint32_t exps[kStages][NW][16 * FM];
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;
  int tm, tn;
  tile_of(a, tm, tn);
  const int64_t m0 = (int64_t)tm * BM;
  const int n0 = tn * BN;
  const int mrows = (int)min((int64_t)BM, a.M - m0), nrows = min(BN, a.N - n0);
  const u32x4 rx = resource(a.xc + m0 * a.Kp, (uint32_t)mrows * a.Kp);
  const u32x4 rw = resource(a.wc + (int64_t)n0 * a.Kp, (uint32_t)nrows * a.Kp);
  const u32x4 re = resource(a.xs + m0 * a.Ks, (uint32_t)mrows * a.Ks);
  const int ox = TX::lane_off(wave, lane, a.Kp), ow = TW::lane_off(wave, lane, a.Kp);
  const int oe = (wm * 16 * FM + lane) * a.Ks;
  const int nb = min((n0 + 16 * FN * wn) / kBlock, (a.N - 1) / kBlock);
  const ConstWords sw = (ConstWords)(a.ws + (int64_t)nb * a.Ks);
  const int k0 = blockIdx.y * a.per, k1 = min(a.Kb, k0 + a.per);  // blocks of this piece
  auto fill = [&](int kb, int s) __attribute__((always_inline)) {
    kb = min(kb, k1 - 1);
#pragma unroll
    for (int i = 0; i < TX::kPer; ++i)
      to_lds<16>(lds_at(xt[s]) + (i * NW + wave) * 1024, rx, ox + i * NW * 8 * a.Kp, kb * kBlock);
#pragma unroll
    for (int i = 0; i < TW::kPer; ++i)
      to_lds<16>(lds_at(wt[s]) + (i * NW + wave) * 1024, rw, ow + i * NW * 8 * a.Kp, kb * kBlock);
    if (lane < 16 * FM) to_lds<4>(lds_at(exps[s][wave]), re, oe, kb & ~3);
  };
  f32x4 acc[FN][FM];
#pragma unroll
  for (int n = 0; n < FN; ++n)
#pragma unroll
    for (int m = 0; m < FM; ++m) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fill(k0 + i, i);
  for (int kb = k0; kb < k1; ++kb) {
    const int s = (kb - k0) & (kStages - 1);
    wait_barrier<(kStages - 2) * kOps>();  // the block has landed, and the one before it has been read
    fill(kb + kStages - 1, (s + kStages - 1) & (kStages - 1));
    const int shift = 8 * (kb & 3);
    const uint32_t ew = sw[kb >> 2] >> shift;
    const char *tx = xt[s] + wm * FM * 16 * kBlock, *tw = wt[s] + wn * FN * 16 * kBlock;
    uint32_t ex[FM];
#pragma unroll
    for (int m = 0; m < FM; ++m) ex[m] = exps[s][wave][16 * m + l16] >> shift;
    if constexpr (kWide) {
      bool high = false;
#pragma unroll
      for (int m = 0; m < FM; ++m) high |= high_row(ex[m]);
      const int shift = w_shift(ew, high);
      Wide xf[FM];
#pragma unroll
      for (int m = 0; m < FM; ++m) xf[m] = widen_x(TX::frag(tx, m, lane), ex[m], shift);
#pragma unroll
      for (int n = 0; n < FN; ++n) {
        const Wide wf = widen_w(TW::frag(tw, n, lane), ew, shift);
#pragma unroll
        for (int m = 0; m < FM; ++m) acc[n][m] = mma_wide(acc[n][m], wf, xf[m]);
      }
    } else {
      Frag8 xf[FM], wf[2];
      wf[0] = TW::frag(tw, 0, lane);
#pragma unroll
      for (int m = 0; m < FM; ++m) xf[m] = TX::frag(tx, m, lane);
#pragma unroll
      for (int n = 0; n < FN; ++n) {
        if (n + 1 < FN) wf[(n + 1) & 1] = TW::frag(tw, n + 1, lane);
#pragma unroll
        for (int m = 0; m < FM; ++m) acc[n][m] = mma8(acc[n][m], wf[n & 1], xf[m], ew, ex[m]);
      }
    }
  }
  f32x4 bias[FN];
#pragma unroll
  for (int n = 0; n < FN; ++n) bias[n] = bias4<T>(a, n0 + 16 * (wn * FN + n) + 4 * g);
  wait_vmem();  // loads past the last block, too
#pragma unroll
  for (int m = 0; m < FM; ++m)
#pragma unroll
    for (int n = 0; n < FN; ++n) {
      const int64_t row = m0 + 16 * (wm * FM + m) + l16;
      const int col = n0 + 16 * (wn * FN + n) + 4 * g;
      if (!a.part)
        store4<T>(a, row, col, acc[n][m], bias[n]);
      else if (row < a.M && col < a.N)  // rows of N up to a multiple of four
        *reinterpret_cast<f32x4*>(a.part + ((int64_t)blockIdx.y * a.M + row) * a.ldp + col) = acc[n][m];
    }
}

// Adds the pieces of a product cut along K: a thread four columns of a row.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(LinearArgs a, int pieces, uint32_t quads, FastDiv d_quads) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  const uint32_t row = div_by(i, d_quads);
  const int col = (int)(i - row * quads) * 4;
  if (row >= a.M) return;
  const float* p = a.part + (int64_t)row * a.ldp + col;
  const f32x4 b = bias4<T>(a, col);
  f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int k = 0; k < pieces; ++k) s += *reinterpret_cast<const f32x4*>(p + (int64_t)k * a.M * a.ldp);
  store4<T>(a, row, col, s, b);
}

// Large 16-bit products: 256 x 256 results a workgroup, eight waves of 64 x 128, two waves
// a SIMD, one workgroup a CU (132 KB of LDS). A block of 128 columns is 64 MFMAs a SIMD
// (2048 cycles) beside 24 LDS reads of 1 KB a wave and 64 KB of loads.
//
// What bounds it is the loads' latency: with each block's loads issued a block ahead and
// waited for at one barrier the kernel stood at 1.7 PFLOP/s (2.7 without the loads). So the
// two stages are refilled piece by piece, as soon as a piece has been read: a block is two
// halves with a barrier each; x is read into registers during the half before it is used,
// so its place is free for the block after the next at the first barrier, a half of w
// (64 of each wave's 128 columns) half a block after its reading. Every piece is on its way
// for one and a half blocks, and a barrier waits for all but the newest eight of a wave's
// loads. The loads are written as instructions: the compiler would wait for all of
// them before each read of LDS.
//
// Measured, 8192 x 8192 x 8192 bf16: 384 us, 2.86 PFLOP/s; 16384 x 6144 x 4096: 297-350 us by
// box, 2.4-2.8 (library products of one scale: 2.66 and 2.98).
template <typename T>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2)))
void large_kernel(LinearArgs a) {
  constexpr int FM = 4, FN = 8, NW = 8, WN = 2, BM = 256, BN = 256;
  using TX = CodeTile<BM, NW>;
  using TW = CodeTile<BN, NW>;
  __shared__ __attribute__((aligned(1024))) char x0[TX::kBytes], x1[TX::kBytes], w00[TW::kBytes / 2], w01[TW::kBytes / 2], w10[TW::kBytes / 2], w11[TW::kBytes / 2];
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;
  int tm, tn;
  tile_of(a, tm, tn);
  const int64_t m0 = (int64_t)tm * BM;
  const int n0 = tn * BN;
  const int mrows = (int)min((int64_t)BM, a.M - m0), nrows = min(BN, a.N - n0);
  const u32x4 rx = resource(a.xc + m0 * a.Kp, (uint32_t)mrows * a.Kp);
  const u32x4 rw = resource(a.wc + (int64_t)n0 * a.Kp, (uint32_t)nrows * a.Kp);
  const u32x4 re = resource(a.xs + m0 * a.Ks, (uint32_t)mrows * a.Ks);
  __shared__ uint32_t exps[2][NW][64];
  const int ox = TX::lane_off(wave, lane, a.Kp), ow = TW::lane_off(wave, lane, a.Kp);
  const int nb = min((n0 + 16 * FN * wn) / kBlock, (a.N - 1) / kBlock);
  const ConstWords sw = (ConstWords)(a.ws + (int64_t)nb * a.Ks);
  uint32_t ex[FM], ew;
  const int oe = (wm * 64 + lane) * a.Ks;
  f32x4 acc[FN][FM];
#pragma unroll
  for (int n = 0; n < FN; ++n)
#pragma unroll
    for (int m = 0; m < FM; ++m) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int row8 = NW * 8 * a.Kp;
  auto fill_x = [&](char* dst, int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) to_lds<16>(lds_at(dst) + (i * NW + wave) * 1024, rx, ox + i * row8, kb * kBlock);
  };
  // half h of the columns of each of the two column waves: 64 of every 128 rows of w
  auto fill_w = [&](char* dst, int h, int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) to_lds<16>(lds_at(dst) + (i * NW + wave) * 1024, rw, ow + (2 * i + h) * row8, kb * kBlock);
  };
  auto fill_e = [&](int s, int q) __attribute__((always_inline)) { to_lds<4>(lds_at(exps[s][wave]), re, oe, 4 * q); };
  const int last = a.Kb - 1, lastq = a.Ks / 4 - 1;
  fill_e(0, 0);
  fill_x(x0, 0);
  fill_w(w00, 0, 0);
  fill_x(x1, min(1, last));
  fill_w(w01, 1, 0);
  fill_w(w10, 0, min(1, last));
  int q = 0;
  Frag8 xf[2][FM];
  wait_barrier<8>();  // x of the first block (ten loads are newer)
#pragma unroll
  for (int m = 0; m < FM; ++m) xf[0][m] = TX::frag(x0 + wm * FM * 16 * kBlock, m, lane);
  auto step = [&](auto second, int kb) __attribute__((always_inline)) {
    constexpr bool kS = decltype(second)::value;
    const char* txn = (kS ? x0 : x1) + wm * FM * 16 * kBlock;
    const char* tw0 = (kS ? w10 : w00) + wn * 64 * kBlock;
    const char* tw1 = (kS ? w11 : w01) + wn * 64 * kBlock;
    wait_barrier<8>();  // the first half of w has landed; x and the other stage's second half have been read
    Frag8 wf[2];
#pragma unroll
    for (int n = 0; n < 1; ++n) wf[n] = TW::frag(tw0, n, lane);
    fill_x(kS ? x1 : x0, min(kb + 2, last));
    fill_w(kS ? w01 : w11, 1, min(kb + 1, last));
    if (!kS && (kb & 2) == 0) {
#pragma unroll
      for (int i = 0; i < FM; ++i) ex[i] = exps[q & 1][wave][16 * i + l16];
      ew = sw[q];
      q = min(q + 1, lastq);
      fill_e(q & 1, q);
    } else {
#pragma unroll
      for (int i = 0; i < FM; ++i) ex[i] >>= 8;
      ew >>= 8;
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if (n + 1 < 4) wf[(n + 1) & 1] = TW::frag(tw0, n + 1, lane);
#pragma unroll
      for (int m = 0; m < FM; ++m) acc[n][m] = mma8(acc[n][m], wf[n & 1], xf[kS][m], ew, ex[m]);
      __builtin_amdgcn_sched_barrier(0);
    }
    wait_barrier<8>();  // the second half of w and the next x have landed; the first half has been read
#pragma unroll
    for (int n = 0; n < 1; ++n) wf[n] = TW::frag(tw1, n, lane);
    fill_w(kS ? w10 : w00, 0, min(kb + 2, last));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if (n + 1 < 4) wf[(n + 1) & 1] = TW::frag(tw1, n + 1, lane);
      xf[!kS][n] = TX::frag(txn, n, lane);
#pragma unroll
      for (int m = 0; m < FM; ++m) acc[4 + n][m] = mma8(acc[4 + n][m], wf[n & 1], xf[kS][m], ew, ex[m]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  for (int kb = 0; kb < a.Kb; kb += 2) {
    step(std::false_type{}, kb);
    if (kb + 1 < a.Kb) step(std::true_type{}, kb + 1);
  }
  wait_vmem();  // loads past the last block, too: LDS is used again
  if (a.wide_y8) {
    // rows of y leave as whole 256-byte pieces: through LDS, 64 rows of 128 columns a
    // wave, chunks of 16 bytes swizzled by row
    __syncthreads();
    char* mine = wave < 2   ? x0 + wave * 16384
                 : wave < 4 ? x1 + (wave - 2) * 16384
                 : wave < 6 ? (wave == 4 ? w00 : w01)
                            : (wave == 6 ? w10 : w11);
#pragma unroll
    for (int n = 0; n < FN; ++n) {
      const f32x4 bias = bias4<T>(a, n0 + 16 * (wn * FN + n) + 4 * g);
#pragma unroll
      for (int m = 0; m < FM; ++m) {
        const int row = 16 * m + l16, chunk = 2 * n + (g >> 1);
        T e[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) e[r] = from_f32<T>(acc[n][m][r] + bias[r]);
        *reinterpret_cast<uint2*>(mine + row * 256 + ((chunk ^ l16) << 4) + (g & 1) * 8) =
            *reinterpret_cast<const uint2*>(e);
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int row = 4 * i + g;
      const uint4 v = *reinterpret_cast<const uint4*>(mine + row * 256 + ((l16 ^ (row & 15)) << 4));
      const int64_t m = m0 + wm * 64 + row;
      const int n = n0 + wn * 128 + l16 * 8;
      if (m < a.M && n < a.N) *reinterpret_cast<uint4*>(static_cast<T*>(a.y) + m * a.ldy + n) = v;
    }
    return;
  }
#pragma unroll
  for (int n = 0; n < FN; ++n) {
    const int col = n0 + 16 * (wn * FN + n) + 4 * g;
    const f32x4 bias = bias4<T>(a, col);
#pragma unroll
    for (int m = 0; m < FM; ++m) store4<T>(a, m0 + 16 * (wm * FM + m) + l16, col, acc[n][m], bias);
  }
}

// Few rows of x: bound by the reading of w. A workgroup takes 16 columns of y and all
// rows (kFewRowsMost at most), its waves a share of the blocks each, straight from memory
// into registers, the first ones' loads on their way before x is looked at; they add up
// through LDS in their order. RAW: x comes as it is, and each wave brings its blocks of the
// at most kRawRows rows into 8 bits for itself, kRawPairs blocks of rows at most.
// Measured, bf16, one row: 6144 x 4096 8.0 us (25 MB of codes: 4.9 by a copy's rate).
constexpr int kFewWaves = 8, kAheadBlocks = 4, kRawRows = 4, kRawPairs = 32;
constexpr int kFewRowsMost = 16, kLargeTiles = 128, kMediumTiles = 140;

template <typename T, bool RAW>
__global__ __launch_bounds__(64 * kFewWaves) void few_rows_kernel(LinearArgs a) {
  constexpr bool kWide = std::is_same<T, float>::value;
  constexpr int NW = kFewWaves, R = kFewRowsMost;
  constexpr int kRawBytes = RAW ? kRawPairs * kBlock : 16;
  __shared__ __attribute__((aligned(16))) char raw[NW][kRawBytes];
  __shared__ uint8_t raw_e[NW][RAW ? kRawPairs : 4];
  __shared__ float sums[NW][R][17];
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * 16, M = (int)a.M;
  const int per = (a.Kb + NW - 1) / NW, k0 = wave * per, k1 = min(a.Kb, k0 + per);
  const uint8_t* wp = a.wc + (int64_t)min(n0 + l16, a.N - 1) * a.Kp + 16 * g;
  const uint8_t* sw = a.ws + (int64_t)(n0 / kBlock) * a.Ks;
  auto load_w = [&](int kb) {
    const uint4* p = reinterpret_cast<const uint4*>(wp + (int64_t)kb * kBlock);
    return Frag8{p[0], p[4]};
  };
  Frag8 wf[kAheadBlocks];
  uint32_t ew[kAheadBlocks];
#pragma unroll
  for (int i = 0; i < kAheadBlocks; ++i) {
    const int kb = max(min(k0 + i, k1 - 1), 0);
    wf[i] = load_w(kb);
    ew[i] = sw[kb];
  }
  if constexpr (RAW) {
    const int n = (k1 - k0) * M;  // (block, row) pairs, four at a time
    for (int i = g; i < n; i += 4) {
      const int b = i / M, row = i - b * M, col = (k0 + b) * kBlock + l16 * 8;
      float x[8];
      load8<T>(static_cast<const T*>(a.x) + row * a.ldx + col, a.K - col, a.wide_x && col + 8 <= a.K, x);
      uint8_t e;
      const uint2 c = codes8(x, lanes_max(largest(x), 4), e);
      *reinterpret_cast<uint2*>(raw[wave] + i * kBlock + l16 * 8) = c;
      if (l16 == 0) raw_e[wave][i] = e;
    }
    __builtin_amdgcn_wave_barrier();  // the wave's own LDS, in order
  }
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int base = k0; base < k1; base += kAheadBlocks) {
#pragma unroll
    for (int i = 0; i < kAheadBlocks; ++i) {
      const int kb = base + i;
      if (kb >= k1) break;
      Frag8 xf;
      uint32_t ex;
      if constexpr (RAW) {
        const int at = (kb - k0) * M + min(l16, M - 1);
        const uint4* p = reinterpret_cast<const uint4*>(raw[wave] + at * kBlock + 16 * g);
        xf = Frag8{p[0], p[4]};
        ex = raw_e[wave][at];
      } else {
        const int64_t row = min(l16, M - 1);
        const uint4* p = reinterpret_cast<const uint4*>(a.xc + row * a.Kp + (int64_t)kb * kBlock + 16 * g);
        xf = Frag8{p[0], p[4]};
        ex = a.xs[row * a.Ks + kb];
      }
      const Frag8 w = wf[i];
      const uint32_t e = ew[i];
      if (kb + kAheadBlocks < k1) {
        wf[i] = load_w(kb + kAheadBlocks);
        ew[i] = sw[kb + kAheadBlocks];
      }
      if constexpr (kWide) {
        const int shift = w_shift(__builtin_amdgcn_readfirstlane(e), high_row(ex));
        acc = mma_wide(acc, widen_w(w, e, shift), widen_x(xf, ex, shift));
      } else {
        acc = mma8(acc, w, xf, e, ex);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) sums[wave][l16][4 * g + r] = acc[r];
  const f32x4 bias = bias4<T>(a, n0 + (tid & 3) * 4);
  __syncthreads();
  for (int i = tid; i < 4 * R; i += 64 * NW) {
    const int row = i >> 2, c = (i & 3) * 4;
    f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[r] += sums[w][row][c + r];
    store4<T>(a, row, n0 + c, s, bias);
  }
}

int err(int code, const char* msg) { return set_error(code, msg); }

int hip_err(hipError_t e, const char* where) {
  if (e == hipSuccess) return CRA_OK;
  char msg[256];
  snprintf(msg, sizeof(msg), "%s: %s", where, hipGetErrorString(e));
  return err(CRA_E_HIP, msg);
}

bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <typename F>
hipError_t with_type(int dtype, F f) {
  return dtype == CRA_F16 ? f(f16()) : dtype == CRA_BF16 ? f(bf16()) : f(float());
}

int check_type(int dtype) {
  return dtype == CRA_F16 || dtype == CRA_BF16 || dtype == CRA_F32 ? CRA_OK : err(CRA_E_DTYPE, "unknown dtype code");
}

int check_linear(const cra_linear* p) {
  if (!p) return err(CRA_E_INVALID, "linear is NULL");
  if (int e = check_type(p->dtype)) return e;
  if (p->M < 1 || p->N < 1 || p->K < 1) return err(CRA_E_INVALID, "M, N and K must be >= 1");
  if (p->K > 1 << 22) return err(CRA_E_INVALID, "K above 2^22 is not built");  // a tile's rows within 2^31 bytes
  if (p->M * (int64_t)up(p->K, kBlock) >= (int64_t)1 << 32) return err(CRA_E_INVALID, "M * K / 128 exceeds 2^32");
  return CRA_OK;
}

// What a call launches.
struct Plan {
  int Kb, Kp, Ks;
  bool few, raw;
  int tile;  // 64, 128, 256
  int64_t tiles_m;
  int tiles_n, pieces;
  size_t code_bytes, scale_bytes, part_bytes;
  size_t bytes() const { return code_bytes + scale_bytes + part_bytes; }
};
Plan plan_of(const cra_linear* p) {
  Plan l{};
  l.Kb = up(p->K, kBlock);
  l.Kp = l.Kb * kBlock;
  l.Ks = up(l.Kb, 4) * 4;
  // where the sides cross (bf16, us): x as it is against brought into 8 bits first, 4 x 4096
  // x 4096 8.2 and 8.7, 4 x 1024 x 16384 17.5 and 12.7 (one and two rows, which stay: 1 x 128 x
  // 4096 5.0 and 8.0, 1 x 1024 x 16384 11.3 and 11.0, 2 x 1024 x 16384 13.2 and 11.6); rows straight from memory against
  // tiles cut along K, 16 x 4096 x 4096 10.5 and 11.4, 16 x 1024 x 16384 23.2 and 13.2, 16 x
  // 16384 x 4096 24.8 and 19.1, 32 x 4096 x 4096 13.2 and 12.7
  l.raw = p->M <= kRawRows && p->M * up(l.Kb, kFewWaves) <= kRawPairs;
  l.few = l.raw || (p->M <= kFewRowsMost && up(p->N, 16) >= 192 && up(p->N, 16) <= 512);
  // tiles: 2048 x 4096 x 4096 (128 of 256) 54.4 us, in tiles of 128 55.1; 1024 x 4096 x 4096 (64
  // and 256) 49.6 and 31.4; 512 x 4096 x 4096 (128 of 128) 26.5, in tiles of 64 24.0; 600 x
  // 4096 x 4096 (160 of 128) 29.6 and 34.4
  auto tiles = [&](int t) { return (int64_t)up(p->M, t) * up(p->N, t); };
  l.tile = tiles(256) >= kLargeTiles ? 256 : tiles(128) >= kMediumTiles ? 128 : 64;
  l.tiles_m = up(p->M, l.tile);
  l.tiles_n = up(p->N, l.tile);
  l.pieces = 1;
  // pieces of K: as many as leave all workgroups resident (two a CU). 128 x 2304 x 4096 (72
  // tiles) in seven 16.8 us, eight 18.3; 300 x 4096 x 4096 (320) in one 22.1, two 26.5
  if (!l.few && l.tile == 64 && tiles(64) <= 256) {
    const int want = std::max(1, std::min(512 / (int)tiles(64), l.Kb / 4));
    l.pieces = up(l.Kb, up(l.Kb, want));
  }
  if (!l.raw) {
    auto up256 = [](size_t n) { return (n + 255) / 256 * 256; };
    l.code_bytes = up256((size_t)p->M * l.Kp);
    l.scale_bytes = up256((size_t)p->M * l.Ks);
    if (l.pieces > 1) l.part_bytes = up256((size_t)l.pieces * p->M * up(p->N, 4) * 16);
  }
  return l;
}

template <typename T>
hipError_t run_rows(const RowsArgs& r, hipStream_t st) {
  rows_kernel<T><<<(r.blocks + 15) / 16, 256, 0, st>>>(r);
  return hipGetLastError();
}

template <typename T>
hipError_t run_linear(const LinearArgs& a, const Plan& l, hipStream_t st) {
  if (l.few) {
    const uint32_t grid = (uint32_t)up(a.N, 16);
    if (l.raw)
      few_rows_kernel<T, true><<<grid, 64 * kFewWaves, 0, st>>>(a);
    else
      few_rows_kernel<T, false><<<grid, 64 * kFewWaves, 0, st>>>(a);
    return hipGetLastError();
  }
  const dim3 grid((uint32_t)(l.tiles_m * l.tiles_n), l.pieces);
  if (l.tile == 256) {
    if constexpr (std::is_same<T, float>::value)
      linear_kernel<T, 4, 2, 4, 8, 2><<<grid, 512, 0, st>>>(a);
    else
      large_kernel<T><<<grid, 512, 0, st>>>(a);
  } else if (l.tile == 128) {
    linear_kernel<T, 4, 2, 2, 4, 4><<<grid, 512, 0, st>>>(a);
  } else {
    linear_kernel<T, 2, 2, 2, 2, 4><<<grid, 256, 0, st>>>(a);
  }
  if (hipError_t e = hipGetLastError()) return e;
  if (l.pieces > 1) {
    const uint32_t quads = (uint32_t)up(a.N, 4);
    join_kernel<T><<<(uint32_t)up((int64_t)quads * a.M, 256), 256, 0, st>>>(a, l.pieces, quads, fast_div(quads));
  }
  return hipGetLastError();
}

}  // namespace
}  // namespace cra

using namespace cra;

extern "C" {

int cra_e4m3_rows(const void* x, int64_t ldx, int64_t M, int32_t K, int32_t dtype, void* codes,
                  void* scales, void* stream) {
  const cra_linear p{M, 1, K, dtype};
  if (int e = check_linear(&p)) return e;
  if (!x || !codes || !scales) return err(CRA_E_INVALID, "x, codes or scales is NULL");
  const int esz = dtype == CRA_F32 ? 4 : 2;
  if (!aligned(x, esz) || !aligned(codes, 16) || !aligned(scales, 4))
    return err(CRA_E_LAYOUT, "x, codes or scales: misaligned pointer");
  RowsArgs r{};
  r.x = x, r.ldx = ldx;
  r.codes = static_cast<uint8_t*>(codes);
  r.scales = static_cast<uint8_t*>(scales);
  r.K = K, r.Kb = up(K, kBlock), r.Ks = up(r.Kb, 4) * 4;
  r.blocks = (uint32_t)(M * r.Kb);
  r.dKb = fast_div(r.Kb);
  r.wide = aligned(x, 16) && ldx * esz % 16 == 0;
  if ((uint64_t)r.blocks * 16 >= (uint64_t)1 << 32) return err(CRA_E_INVALID, "too many rows for one launch");
  return hip_err(with_type(dtype, [&](auto z) { return run_rows<decltype(z)>(r, (hipStream_t)stream); }),
                 "cra_e4m3_rows");
}

int cra_e4m3_weight(const void* w, int64_t ldw, int32_t N, int32_t K, int32_t dtype, void* codes,
                    void* scales, void* stream) {
  const cra_linear p{1, N, K, dtype};
  if (int e = check_linear(&p)) return e;
  if (!w || !codes || !scales) return err(CRA_E_INVALID, "w, codes or scales is NULL");
  const int esz = dtype == CRA_F32 ? 4 : 2;
  if (!aligned(w, esz) || !aligned(codes, 16) || !aligned(scales, 4))
    return err(CRA_E_LAYOUT, "w, codes or scales: misaligned pointer");
  const int Kb = up(K, kBlock), Ks = up(Kb, 4) * 4;
  if (up(N, kBlock) > 65535) return err(CRA_E_INVALID, "N above 2^23 is not built");
  const int wide = aligned(w, 16) && ldw * esz % 16 == 0;
  const dim3 grid(Kb, up(N, kBlock));
  return hip_err(with_type(dtype, [&](auto z) {
    using T = decltype(z);
    weight_kernel<T><<<grid, 256, 0, (hipStream_t)stream>>>(static_cast<const T*>(w), ldw, N, K, Kb, Ks, wide,
                                                            static_cast<uint8_t*>(codes),
                                                            static_cast<uint8_t*>(scales));
    return hipGetLastError();
  }), "cra_e4m3_weight");
}

size_t cra_linear_e4m3_workspace_bytes(const cra_linear* p) {
  if (check_linear(p)) return 0;
  const Plan l = plan_of(p);
  return l.bytes();
}

int cra_linear_e4m3(const cra_linear* p, const void* x, int64_t ldx, const void* w_codes,
                    const void* w_scales, const void* bias, void* y, int64_t ldy, void* workspace,
                    size_t workspace_bytes, void* stream) {
  if (int e = check_linear(p)) return e;
  if (!x || !w_codes || !w_scales || !y) return err(CRA_E_INVALID, "x, w or y is NULL");
  const int esz = p->dtype == CRA_F32 ? 4 : 2;
  if (!aligned(x, esz) || !aligned(y, esz) || !aligned(bias, esz) || !aligned(w_codes, 16) || !aligned(w_scales, 4))
    return err(CRA_E_LAYOUT, "x, w, bias or y: misaligned pointer");
  const Plan l = plan_of(p);
  const size_t need = l.bytes();
  if (need && (!workspace || !aligned(workspace, 16)))
    return err(CRA_E_INVALID, "workspace: NULL or misaligned pointer");
  if (workspace_bytes < need) return err(CRA_E_WORKSPACE, "workspace too small (cra_linear_e4m3_workspace_bytes)");
  if (l.tiles_m * l.tiles_n >= (int64_t)1 << 22) return err(CRA_E_INVALID, "too many tiles for one launch");
  hipStream_t st = (hipStream_t)stream;
  LinearArgs a{};
  a.x = x, a.ldx = ldx;
  a.wc = static_cast<const uint8_t*>(w_codes);
  a.ws = static_cast<const uint8_t*>(w_scales);
  a.bias = bias;
  a.y = y, a.ldy = ldy;
  a.M = p->M, a.N = p->N, a.K = p->K;
  a.Kb = l.Kb, a.Kp = l.Kp, a.Ks = l.Ks;
  a.tiles_m = (int)l.tiles_m, a.tiles_n = l.tiles_n;
  a.wide_x = aligned(x, 16) && ldx * esz % 16 == 0;
  a.wide_y = p->N % 4 == 0 && ldy % 4 == 0 && aligned(y, 4 * esz);
  a.wide_y8 = p->N % 8 == 0 && ldy % 8 == 0 && aligned(y, 16);
  if (!l.raw) {
    char* ws = static_cast<char*>(workspace);
    if (int e = cra_e4m3_rows(x, ldx, p->M, p->K, p->dtype, ws, ws + l.code_bytes, stream)) return e;
    a.xc = reinterpret_cast<const uint8_t*>(ws);
    a.xs = reinterpret_cast<const uint8_t*>(ws + l.code_bytes);
    if (l.pieces > 1) a.part = reinterpret_cast<float*>(ws + l.code_bytes + l.scale_bytes);
    a.per = up(l.Kb, l.pieces);
    a.ldp = (int64_t)up(p->N, 4) * 4;
  }
  return hip_err(with_type(p->dtype, [&](auto z) { return run_linear<decltype(z)>(a, l, st); }), "cra_linear_e4m3");
}

}  // extern "C"
