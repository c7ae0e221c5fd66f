// Paged key/value cache: writing the rows of new tokens (as they are, or with 8
// bits an element) and reading sequences back, with the C ABI front end.
//
// A key row is stored with the sum of its squares, which the relay rows are
// ranked by: 4 bytes a row instead of a pass over all keys whenever blocks are
// formed for another length. The sum is that of the packed-row kernel of whole
// sequences, bit for bit (8 elements left to right by fused multiply-adds, then a
// butterfly over the D/8 lanes), so both choose the same rows.
//
// 8 bits: row x with m = max |x| is held as codes c and a scale s.
//   e4m3: s = the smallest power of two with m <= 448 s, c = RNE(x / s). x / s
//         and c s are exact, codes keep their 3 bits whatever the row's scale.
//   int8: s = m times the fp32 1/127 (so |x| / s stays below 127.5), c = RNE(x / s).
// s is at least 2^-126. A row that holds an infinity or NaN gets s = NaN.
//
// Bound by memory, 8-bit writes nearly as much by the VALU; a row belongs to D/8
// lanes (a power of two), 16 bytes of k and of v each. Measured, D = 128 16-bit:
// writes of 32768 tokens of 16 heads as they are 106 us (539 MB, 5.1 TB/s), as int8
// 100 us (409 MB, 4.1 TB/s; dividing each element and exchanging by LDS shuffles
// 146 us); of 26000 ragged tokens of 4 heads as they are 21 us (107 MB), as e4m3 31
// us (81 MB; the VALU is busy for about 16 of them, and waves wait for two thirds of
// their time, offsets, length and page id of a row in turn); reads 155 us (814 MB,
// 5.2 TB/s) and 44 us (16 sequences of up to 9001 rows, padded: 322 MB). Two or four rows a thread gave nothing (146, 159
// against 146 us), nor did neighbouring tokens in place of heads (152-160 us).
#include <stdio.h>

#include <algorithm>

#include "cra_common.hpp"
#include "cra_internal.hpp"
#include "cra_cache_dev.hpp"
#include "cra_paged.hpp"

namespace cra {

int set_error(int code, const char* msg);

namespace {

constexpr int kThreads = 256;

struct WriteArgs {
  PagedView c;
  const void *k, *v;
  int64_t ksb, ksh, kss, vsb, vsh, vss;
  float *k_norm, *k_scale, *v_scale;
  int Din, Ds, log_l;    // columns given, columns stored, lanes of a row
  uint32_t rows;         // tokens * H_kv
  FastDiv dH, dT, dM;    // H_kv; tokens; tokens per sequence
  int head_fast;
};

template <typename T, int STORE>
__global__ __launch_bounds__(kThreads) void cache_write_kernel(WriteArgs a) {
  const int lane = threadIdx.x & ((1 << a.log_l) - 1);
  const uint32_t r = blockIdx.x * (uint32_t)(kThreads >> a.log_l) + (threadIdx.x >> a.log_l);
  if (r >= a.rows) return;  // whole rows leave: the shuffles stay within a row
  int t, h;
  if (a.head_fast) {
    t = (int)div_by(r, a.dH);
    h = (int)(r - (uint32_t)t * a.c.H_kv);
  } else {
    h = (int)div_by(r, a.dT);
    t = (int)(r - (uint32_t)h * a.c.tokens);
  }
  // the rows are loaded before the place they go to is known: finding it takes four
  // loads in turn (offsets, length, page id)
  const int tb = a.c.cu ? 0 : (int)div_by(t, a.dM), ts = a.c.cu ? t : t - tb * a.c.query_len;
  Row8<T> kr, vr;
  float kx[8], vx[8];
  const bool have = lane * 8 < a.Din;
  const T* kp = static_cast<const T*>(a.k) + tb * a.ksb + h * a.ksh + ts * a.kss + lane * 8;
  const T* vp = static_cast<const T*>(a.v) + tb * a.vsb + h * a.vsh + ts * a.vss + lane * 8;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); ++i) {
    kr.w[i] = have ? reinterpret_cast<const uint4*>(kp)[i] : make_uint4(0, 0, 0, 0);
    vr.w[i] = have ? reinterpret_cast<const uint4*>(vp)[i] : make_uint4(0, 0, 0, 0);
  }
  int b = tb, first = tb * a.c.query_len, count = a.c.query_len;  // sequence, its first token and tokens
  if (a.c.cu) {
    const int at = threadIdx.x & 63 & ~lane;  // the row's lanes within the wave
    b = seq_of_token(a.c.cu, a.c.n_seqs, t, 1 << a.log_l, [&](int first, int step, int n) {
      const int64_t i = (int64_t)lane * step;
      const uint64_t m = __ballot(i < n && a.c.cu[first + (i < n ? i : 0)] <= t) >> at;
      return __popcll(m & ((1ull << (1 << a.log_l)) - 1));
    });
    if (b < 0) return;
    const TokenRange tr = token_range(a.c.cu, b, a.c.tokens);
    first = tr.first, count = tr.last - tr.first;
  }
  const int row = write_row(a.c.lens[b], count, t - first, a.c.pages_per_seq, a.c.log_page);
  const uint32_t dst = row >= 0 ? seq_row(a.c.table + b * a.c.table_stride, row, a.c.num_pages,
                                          a.c.H_kv, a.c.log_page, h)
                                : kNoRow;
  if (dst == kNoRow) return;  // nothing of the row is written
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    kx[i] = to_f32(reinterpret_cast<const T*>(kr.w)[i]);
    vx[i] = to_f32(reinterpret_cast<const T*>(vr.w)[i]);
  }
  const float norm = lanes_sum(square_sum(kx), a.log_l);
  if (lane == 0) a.k_norm[dst] = norm;
  store_row<T, STORE>(kx, kr, const_cast<char*>(a.c.k), a.k_scale, dst, a.Ds, lane, a.log_l);
  store_row<T, STORE>(vx, vr, const_cast<char*>(a.c.v), a.v_scale, dst, a.Ds, lane, a.log_l);
}

struct ReadArgs {
  PagedView c;
  void *k, *v;   // [n_seqs, H_kv, L, D]
  int L, D, Ds;  // rows and columns read; columns stored
  int chunks;    // V-element chunks of a row
  uint32_t total;
  FastDiv dC, dL, dH;
};

// V elements of a stored row times its scale.
template <typename T, int STORE, int V>
__device__ __forceinline__ void read_chunk(const char* base, const float* scale, uint32_t row,
                                           int64_t at, T (&y)[V]) {
  if constexpr (STORE == kSame) {
    const T* p = reinterpret_cast<const T*>(base) + at;
    if constexpr (V == 8) {
      const Row8<T> w = *reinterpret_cast<const Row8<T>*>(p);
#pragma unroll
      for (int i = 0; i < V; ++i) y[i] = reinterpret_cast<const T*>(w.w)[i];
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) y[i] = p[i];
    }
  } else {
    const float s = scale[row];
    uint32_t w[(V + 3) / 4];
    if constexpr (V == 8) {
      const uint2 u = *reinterpret_cast<const uint2*>(base + at);
      w[0] = u.x, w[1] = u.y;
    } else {
      w[0] = *reinterpret_cast<const uint8_t*>(base + at);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float c;
      if (STORE == kE4M3) {
        const uint32_t byte = w[i / 4] >> (8 * (i % 4)) & 0xffu;
        c = __builtin_amdgcn_cvt_f32_fp8((int)byte, 0);
      } else {
        c = (float)(int8_t)(w[i / 4] >> (8 * (i % 4)) & 0xffu);
      }
      y[i] = from_f32<T>(c * s);
    }
  }
}

template <typename T, int STORE, int V>
__global__ __launch_bounds__(kThreads) void cache_read_kernel(ReadArgs a) {
  const uint32_t i = blockIdx.x * (uint32_t)kThreads + threadIdx.x;
  if (i >= a.total) return;
  const uint32_t line = div_by(i, a.dC);  // (sequence, head, row)
  const int chunk = (int)(i - line * a.chunks);
  const uint32_t bh = div_by(line, a.dL);
  const int row = (int)(line - bh * a.L);
  const int b = (int)div_by(bh, a.dH), h = (int)(bh - (uint32_t)b * a.c.H_kv);
  const int n = seq_length(a.c.lens[b], a.c.pages_per_seq, a.c.log_page);
  T ky[V], vy[V];
#pragma unroll
  for (int j = 0; j < V; ++j) ky[j] = vy[j] = from_f32<T>(0.f);
  if (row < n) {
    const uint32_t src =
        seq_row(a.c.table + b * a.c.table_stride, row, a.c.num_pages, a.c.H_kv, a.c.log_page, h);
    if (src != kNoRow) {
      const int64_t at = (int64_t)src * a.Ds + chunk * V;
      read_chunk<T, STORE, V>(a.c.k, a.c.k_scale, src, at, ky);
      read_chunk<T, STORE, V>(a.c.v, a.c.v_scale, src, at, vy);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) ky[j] = vy[j] = from_f32<T>(__builtin_nanf(""));
    }
  }
  T* kp = static_cast<T*>(a.k) + (int64_t)line * a.D + chunk * V;
  T* vp = static_cast<T*>(a.v) + (int64_t)line * a.D + chunk * V;
  if constexpr (V == 8) {
    *reinterpret_cast<Row8<T>*>(kp) = __builtin_bit_cast(Row8<T>, ky);
    *reinterpret_cast<Row8<T>*>(vp) = __builtin_bit_cast(Row8<T>, vy);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) kp[j] = ky[j], vp[j] = vy[j];
  }
}

int err(int code, const char* msg) { return set_error(code, msg); }

int hip_err(hipError_t e, const char* where) {
  if (e == hipSuccess) return CRA_OK;
  char msg[256];
  snprintf(msg, sizeof(msg), "%s: %s", where, hipGetErrorString(e));
  return err(CRA_E_HIP, msg);
}

bool misaligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

template <typename F>
hipError_t with_type(int dtype, F f) {
  return dtype == CRA_F16 ? f(f16()) : dtype == CRA_BF16 ? f(bf16()) : f(float());
}
template <int S>
using Int = std::integral_constant<int, S>;
template <typename F>
hipError_t with_store(int store, F f) {
  return store == CRA_STORE_SAME ? f(Int<kSame>()) : store == CRA_STORE_E4M3 ? f(Int<kE4M3>()) : f(Int<kInt8>());
}

}  // namespace

int check_cache(const cra_cache* c) {
  if (!c) return err(CRA_E_INVALID, "cache is NULL");
  if (c->dtype != CRA_F16 && c->dtype != CRA_BF16 && c->dtype != CRA_F32)
    return err(CRA_E_DTYPE, "unknown dtype code");
  if (c->store != CRA_STORE_SAME && c->store != CRA_STORE_E4M3 && c->store != CRA_STORE_INT8)
    return err(CRA_E_DTYPE, "unknown storage code");
  if (c->num_pages < 1 || c->H_kv < 1) return err(CRA_E_INVALID, "num_pages and H_kv must be >= 1");
  if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)))
    return err(CRA_E_INVALID, "page size must be a power of two from 16 to 1024");
  if (c->D < 16 || c->D > 256 || c->D % 16)
    return err(CRA_E_UNSUPPORTED, "row width must be a multiple of 16 up to 256");
  if ((int64_t)c->num_pages * c->H_kv * c->page_size >= (int64_t)1 << 31)
    return err(CRA_E_INVALID, "the cache has 2^31 rows or more");
  if (!c->k || !c->v || !c->k_norm) return err(CRA_E_INVALID, "cache: NULL pointer");
  if (c->store != CRA_STORE_SAME && (!c->k_scale || !c->v_scale))
    return err(CRA_E_INVALID, "an 8-bit cache needs scales");
  if (misaligned(c->k, 16) || misaligned(c->v, 16) || misaligned(c->k_norm, 16) ||
      misaligned(c->k_scale, 4) || misaligned(c->v_scale, 4))
    return err(CRA_E_LAYOUT, "cache: misaligned pointer");
  return CRA_OK;
}

int check_batch(const cra_cache* c, const cra_batch* b) {
  if (!b) return err(CRA_E_INVALID, "batch is NULL");
  if (b->n_seqs < 1 || b->pages_per_seq < 1)
    return err(CRA_E_INVALID, "n_seqs and pages_per_seq must be >= 1");
  if (!b->page_table || !b->seq_lens) return err(CRA_E_INVALID, "page_table or seq_lens is NULL");
  if (misaligned(b->page_table, 4) || misaligned(b->seq_lens, 4) || misaligned(b->cu_seqlens, 4))
    return err(CRA_E_LAYOUT, "batch: misaligned pointer");
  if (b->cu_seqlens ? b->tokens < 1 : b->query_len < 1)
    return err(CRA_E_INVALID, "a batch without new tokens");
  if (!b->cu_seqlens && (int64_t)b->n_seqs * b->query_len >= (int64_t)1 << 31)
    return err(CRA_E_INVALID, "2^31 new tokens or more");
  return CRA_OK;
}

PagedView paged_view(const cra_cache* c, const cra_batch* b) {
  PagedView v{};
  v.k = static_cast<const char*>(c->k);
  v.v = static_cast<const char*>(c->v);
  v.k_norm = c->k_norm;
  v.k_scale = c->k_scale;
  v.v_scale = c->v_scale;
  v.table = b->page_table;
  v.table_stride = b->table_stride;
  v.lens = b->seq_lens;
  v.cu = b->cu_seqlens;
  v.num_pages = c->num_pages;
  v.H_kv = c->H_kv;
  v.log_page = __builtin_ctz((unsigned)c->page_size);
  v.n_seqs = b->n_seqs;
  v.pages_per_seq = b->pages_per_seq;
  v.tokens = b->cu_seqlens ? b->tokens : b->n_seqs * b->query_len;
  v.query_len = b->query_len;
  return v;
}

}  // namespace cra

using namespace cra;

extern "C" {

int cra_cache_write(const cra_cache* c, const cra_batch* b, cra_tensor k, cra_tensor v, int32_t D,
                    void* stream) {
  if (int e = check_cache(c)) return e;
  if (int e = check_batch(c, b)) return e;
  if (D < 8 || D > c->D || D % 8) return err(CRA_E_INVALID, "D must be a multiple of 8 up to the row width");
  const int vec = c->dtype == CRA_F32 ? 4 : 8;
  for (const cra_tensor* t : {&k, &v}) {
    if (!t->ptr) return err(CRA_E_INVALID, "k or v is NULL");
    if (misaligned(t->ptr, 16) || t->sb % vec || t->sh % vec || t->ss % vec)
      return err(CRA_E_LAYOUT, "rows of k and v must be 16-byte aligned");
  }
  WriteArgs a{};
  a.c = paged_view(c, b);
  if ((int64_t)a.c.tokens * c->H_kv >= (int64_t)1 << 31) return err(CRA_E_INVALID, "2^31 new rows or more");
  a.k = k.ptr, a.ksb = k.sb, a.ksh = k.sh, a.kss = k.ss;
  a.v = v.ptr, a.vsb = v.sb, a.vsh = v.sh, a.vss = v.ss;
  a.k_norm = c->k_norm, a.k_scale = c->k_scale, a.v_scale = c->v_scale;
  a.Din = D, a.Ds = c->D;
  while ((8 << a.log_l) < c->D) ++a.log_l;
  a.rows = (uint32_t)a.c.tokens * c->H_kv;
  a.dH = fast_div(c->H_kv);
  a.dT = fast_div(a.c.tokens);
  a.dM = fast_div(std::max(1, b->query_len));
  a.head_fast = k.sh < k.ss;
  const uint32_t slots = kThreads >> a.log_l, grid = (a.rows + slots - 1) / slots;
  if ((uint64_t)grid * kThreads >= (uint64_t)1 << 32) return err(CRA_E_INVALID, "too many rows for one launch");
  return hip_err(with_type(c->dtype, [&](auto z) {
    return with_store(c->store, [&](auto s) {
      cache_write_kernel<decltype(z), decltype(s)::value><<<grid, kThreads, 0, (hipStream_t)stream>>>(a);
      return hipGetLastError();
    });
  }), "cra_cache_write");
}

int cra_cache_read(const cra_cache* c, const cra_batch* b, int32_t length, int32_t D, void* k,
                   void* v, void* stream) {
  if (int e = check_cache(c)) return e;
  if (!b) return err(CRA_E_INVALID, "batch is NULL");
  cra_batch one = *b;  // a read takes no new tokens
  one.cu_seqlens = nullptr;
  one.query_len = 1;
  if (int e = check_batch(c, &one)) return e;
  if (D < 1 || D > c->D) return err(CRA_E_INVALID, "D must be from 1 to the row width");
  if (length < 1) return err(CRA_E_INVALID, "length must be >= 1");
  if (!k || !v) return err(CRA_E_INVALID, "k or v is NULL");
  if (misaligned(k, 16) || misaligned(v, 16)) return err(CRA_E_LAYOUT, "k or v is not 16-byte aligned");
  ReadArgs a{};
  a.c = paged_view(c, &one);
  a.k = k, a.v = v;
  a.L = length, a.D = D, a.Ds = c->D;
  const bool wide = D % 8 == 0;
  a.chunks = wide ? D / 8 : D;
  const int64_t total = (int64_t)b->n_seqs * c->H_kv * length * a.chunks;
  if (total >= (int64_t)0xffffff00) return err(CRA_E_INVALID, "too many rows for one launch");
  a.total = (uint32_t)total;
  a.dC = fast_div(a.chunks);
  a.dL = fast_div(length);
  a.dH = fast_div(c->H_kv);
  const uint32_t grid = (uint32_t)((total + kThreads - 1) / kThreads);
  return hip_err(with_type(c->dtype, [&](auto z) {
    return with_store(c->store, [&](auto s) {
      using T = decltype(z);
      constexpr int S = decltype(s)::value;
      if (wide)
        cache_read_kernel<T, S, 8><<<grid, kThreads, 0, (hipStream_t)stream>>>(a);
      else
        cache_read_kernel<T, S, 1><<<grid, kThreads, 0, (hipStream_t)stream>>>(a);
      return hipGetLastError();
    });
  }), "cra_cache_read");
}

}  // extern "C"
