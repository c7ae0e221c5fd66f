// Rows on their way into a paged cache: the sum of squares of a key, 8-bit codes and
// scales. Shared by the write (cra_cache.hip) and the append (cra_append.hip).
#pragma once

#include "cra_common.hpp"
#include "cra_paged.hpp"

namespace cra {

template <typename T>
struct Row8 {
  uint4 w[sizeof(T) / 2];
};

template <typename F>
__device__ __forceinline__ uint32_t lanes_fold(uint32_t x, int log_l, F f) {
  if (log_l > 4) x = f(x, from_lane_xor<16>(x));
  if (log_l > 3) x = f(x, from_lane_xor<8>(x));
  if (log_l > 2) x = f(x, from_lane_xor<4>(x));
  if (log_l > 1) x = f(x, from_lane_xor<2>(x));
  if (log_l > 0) x = f(x, from_lane_xor<1>(x));
  return x;
}
__device__ __forceinline__ uint32_t lanes_max(uint32_t x, int log_l) {
  return lanes_fold(x, log_l, [](uint32_t a, uint32_t b) { return max(a, b); });
}
__device__ __forceinline__ float lanes_sum(float x, int log_l) {
  return __uint_as_float(lanes_fold(__float_as_uint(x), log_l, [](uint32_t a, uint32_t b) {
    return __float_as_uint(__fadd_rn(__uint_as_float(a), __uint_as_float(b)));
  }));
}

// Sum of a lane's squares: left to right by fused multiply-adds.
__device__ __forceinline__ float square_sum(const float (&x)[8]) {
  float s = x[0] * x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) s = __builtin_fmaf(x[i], x[i], s);
  return s;
}

// Scale of a row from the bits of max |x| (which order as the values do, NaN
// above infinity).
template <int STORE>
__device__ __forceinline__ float row_scale(uint32_t m) {
  if (m >= 0x7f800000u) return __builtin_nanf("");
  if (STORE == kE4M3) {
    const int e = (int)(m >> 23) - 127 - 8 + ((m & 0x7fffffu) > 0x600000u ? 1 : 0);
    return __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
  }
  return fmaxf(__uint_as_float(m) * (1.f / 127.f), 0x1p-126f);
}

// Four codes of x / s.
template <int STORE>
__device__ __forceinline__ uint32_t codes4(const float* x, float s) {
  if (STORE == kE4M3) {
    const float inv = __fdiv_rn(1.f, s);  // a power of two: exact
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false);
    c = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, c, true);
    return (uint32_t)c;
  }
  // RNE(x / s) by a multiplication: x times the reciprocal (one ulp off) is within
  // 2^-14 of x / s (at most 127), so the integers agree unless that is nearer than
  // 2^-12 to halfway between two; a wave that meets such an element divides. Adding
  // 1.5 * 2^23 rounds to the integer and leaves it in the low byte.
  constexpr float kMagic = 12582912.f;
  const float inv = __builtin_amdgcn_rcpf(s);
  float q[4], off = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float y = x[i] * inv;
    q[i] = y + kMagic;
    off = fmaxf(off, fabsf(y - (q[i] - kMagic)));
  }
  if (__any(off > 0.5f - 0x1p-12f)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = __fadd_rn(__fdiv_rn(x[i], s), kMagic);
  }
  const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(q[1]), __float_as_uint(q[0]), 0x0c0c0400);
  const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(q[3]), __float_as_uint(q[2]), 0x04000c0c);
  return lo | hi;
}

template <typename T, int STORE>
__device__ __forceinline__ void store_row(const float (&x)[8], const Row8<T>& raw, void* base,
                                          float* scale, uint32_t row, int Ds, int lane, int log_l) {
  const int64_t at = (int64_t)row * Ds + lane * 8;
  if constexpr (STORE == kSame) {
    if (lane * 8 < Ds) {
      uint4* p = reinterpret_cast<uint4*>(static_cast<T*>(base) + at);
#pragma unroll
      for (int i = 0; i < (int)(sizeof(T) / 2); ++i) p[i] = raw.w[i];
    }
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    const float s = row_scale<STORE>(lanes_max(m, log_l));
    if (lane * 8 < Ds)  // codes themselves are finite: the scale says what is not
      *reinterpret_cast<uint2*>(static_cast<char*>(base) + at) =
          s == s ? make_uint2(codes4<STORE>(x, s), codes4<STORE>(x + 4, s)) : make_uint2(0, 0);
    if (lane == 0) scale[row] = s;
  }
}

}  // namespace cra
