"""The paged cache and its attention without a GPU: the geometry header against
plain Python, refusals of the C ABI before any launch, and of the Python layer."""
import ctypes
import math
import os
import shutil
import subprocess

import pytest
import torch

import cron_root_attention as cra
from cron_root_attention import _native as N

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "cron-root-attention_amd", "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

CHECKER = r"""
#include "cra_paged.hpp"
#include <cstdio>
#include <vector>
using namespace cra;
int main() {
  long bad = 0, cases = 0;
  // ceil(sqrt(n)) around every square up to 2^31
  for (int64_t r = 0; r <= 46341; ++r)
    for (int64_t n = r * r - 1; n <= r * r + 1; ++n) {
      if (n < 0 || n > 0x7fffffff) continue;
      ++cases;
      const int64_t c = ceil_sqrt((int)n);
      bad += !(c * c >= n && (c == 0 || (c - 1) * (c - 1) < n));
    }
  // the prefix of global rows counts the strided rows below the window and the
  // relay rows of the blocks that end before it
  for (int n = 1; n < 220; ++n)
    for (int window : {0, 1, 2, 7, 64, 1000})
      for (int relay : {0, 1}) {
        const SeqPlan p = seq_plan(n, window, relay, 2);
        if (p.W < 1 || p.W > n) { ++bad; continue; }
        for (int i = 0; i < n; ++i) {
          ++cases;
          const int ls = i - p.W + 1 > 0 ? i - p.W + 1 : 0;
          int want = 0;
          for (int r = 0; r * p.W < ls; ++r) want += 1 + (relay && (r + 1) * p.W <= ls ? 2 : 0);
          bad += seq_prefix(i, p) != want;
        }
      }
  bad += seq_plan(2048, 0, -1, 2).rpb != 1 || seq_plan(2049, 0, -1, 2).rpb != 3;
  bad += seq_plan(0, 0, -1, 2).W != 1 || seq_prefix(-5, seq_plan(100, 0, 1, 2)) != 0;
  // lengths and token ranges stay within the tables whatever the device holds
  bad += seq_length(-3, 4, 4) != 0 || seq_length(64, 4, 4) != 64 || seq_length(65, 4, 4) != 64;
  bad += seq_length(0x7fffffff, 0x7fffffff, 10) != 0x7fffffff;
  const int32_t junk[][2] = {{-5, 3}, {3, -5}, {90, 200}, {4, 2}, {0, 10}, {-2147483647 - 1, 2147483647}};
  for (auto& c : junk) {
    const TokenRange t = token_range(c, 0, 10);
    bad += t.first < 0 || t.first > t.last || t.last > 10;
    ++cases;
  }
  // the tiles of any sequence stay within what the launch reserves for the longest
  for (int most : {1, 5, 16, 100, 676, 677, 2047, 2100, 2500, 5000})
    for (int window : {0, 1, 3, 64, 700, 100000})
      for (int relay : {-1, 0, 1}) {
        const PlanMost pm = plan_most(most, window, relay, 3);
        for (int n = 0; n <= most; ++n) {
          const SeqPlan p = seq_plan(n, window, relay, 3);
          bad += n > 0 && seq_prefix(n - 1, p) > pm.globals;
          bad += p.W > pm.W;
          for (int m : {1, 2, 16}) {
            ++cases;
            bad += few_tile_count(n, m, p) > few_tile_most(pm, 16);
          }
          for (int bn : {32, 64}) bad += chunk_tile_count(n, 10, bn, p) > chunk_tile_most(pm, 10, bn);
        }
      }
  // the sequence of a token, empty sequences among them
  const std::vector<int32_t> cu = {2, 2, 5, 5, 5, 9, 9};
  const int want[] = {-1, -1, 1, 1, 1, 4, 4, 4, 4, -1, -1};
  auto find = [](const std::vector<int32_t>& cu, int t, int lanes) {
    const int n_seqs = (int)cu.size() - 1;
    return seq_of_token(cu.data(), n_seqs, t, lanes, [&](int first, int step, int n) {
      int c = 0;
      for (int i = 0; i < lanes && (int64_t)i * step < n; ++i) c += cu[first + i * step] <= t;
      return c;
    });
  };
  for (int lanes : {2, 4, 32})
    for (int t = 0; t < 11; ++t) bad += find(cu, t, lanes) != want[t];
  for (int n_seqs : {1, 2, 3, 15, 16, 17, 64, 65, 300, 1025}) {
    std::vector<int32_t> many(1, 3);
    std::vector<int> owner(3, -1);
    for (int b = 0; b < n_seqs; ++b) {
      const int m = b * 7 % 5;
      owner.insert(owner.end(), m, b);
      many.push_back(many.back() + m);
    }
    owner.insert(owner.end(), 2, -1);
    for (int lanes : {2, 4, 8, 16, 32})
      for (int t = 0; t < (int)owner.size(); ++t, ++cases) bad += find(many, t, lanes) != owner[t];
  }
  // offsets that run backwards: some sequence of the batch
  const std::vector<int32_t> back = {0, 90, 5, 70, -4, 2147483647, 3, 60, 20, 100};
  for (int lanes : {2, 4, 8})
    for (int t = 0; t < 100; ++t) {
      const int b = find(back, t, lanes);
      bad += b < 0 || b > 8;
    }
  // rows of pages: in the page's place, and none of a page outside the cache
  const int32_t pages[] = {7, -1, 12, 11, 2147483647, -2147483647 - 1};
  bad += seq_row(pages, 5, 12, 3, 4, 2) != (7u * 3 + 2) * 16 + 5;
  bad += seq_row(pages, 16, 12, 3, 4, 2) != kNoRow || seq_row(pages, 33, 12, 3, 4, 0) != kNoRow;
  bad += seq_row(pages, 63, 12, 3, 4, 0) != (11u * 3) * 16 + 15;
  bad += seq_row(pages, 64, 12, 3, 4, 0) != kNoRow || seq_row(pages, 95, 12, 3, 4, 0) != kNoRow;
  // a cache of almost 2^31 rows keeps its row numbers apart from kNoRow
  const int32_t far[] = {8388606};
  bad += seq_row(far, 15, 8388607, 16, 4, 15) != 8388606u * 256 + 15 * 16 + 15;
  printf("%ld %ld\n", cases, bad);
  return 0;
}
"""


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")
def test_geometry_on_the_host(tmp_path):
    src, exe = tmp_path / "paged.cpp", tmp_path / "paged"
    src.write_text(CHECKER)
    subprocess.run([HIPCC, "-std=c++17", "-O1", "-I", CSRC, str(src), "-o", str(exe)], check=True,
                   capture_output=True, timeout=300)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=120)
    cases, bad = map(int, out.stdout.split())
    assert cases > 300000 and bad == 0


P = 0x10000
CACHE = dict(k=P, v=P, k_norm=P, k_scale=None, v_scale=None, num_pages=10, H_kv=2, page_size=64, D=128,
             dtype=0, store=0)
BATCH = dict(page_table=P, table_stride=5, seq_lens=P, cu_seqlens=None, n_seqs=3, pages_per_seq=5, tokens=0,
             query_len=4)
PLAN = dict(H_q=8, D=128, window=0, relay=-1, top_k=2, max_query_len=4, max_seqlen=320, zero_outside=0, scale=0.1)
T = N.CraTensor(P, 1 << 16, 128, 1024)


def structs(**kw):
    out = []
    for cls, base in ((N.CraCache, CACHE), (N.CraBatch, BATCH), (N.CraPagedPlan, PLAN)):
        over = {k: v for k, v in kw.items() if k in base and not (cls is N.CraPagedPlan and k == "D")}
        if cls is N.CraPagedPlan and "qD" in kw:  # the plan's columns, not the cache's
            over["D"] = kw["qD"]
        out.append(ctypes.byref(cls(**{**base, **over})))
    return out


COMMON = [
    (dict(D=24), N.E_UNSUPPORTED, "multiple of 16"),
    (dict(D=272), N.E_UNSUPPORTED, "multiple of 16"),
    (dict(dtype=3), N.E_DTYPE, "dtype"),
    (dict(store=3), N.E_DTYPE, "storage"),
    (dict(num_pages=0), N.E_INVALID, "num_pages"),
    (dict(H_kv=0), N.E_INVALID, "H_kv"),
    (dict(page_size=48), N.E_INVALID, "power of two"),
    (dict(page_size=8), N.E_INVALID, "power of two"),
    (dict(page_size=2048), N.E_INVALID, "power of two"),
    (dict(num_pages=1 << 24, H_kv=2, page_size=64), N.E_INVALID, "2^31"),
    (dict(k=None), N.E_INVALID, "NULL"),
    (dict(k_norm=None), N.E_INVALID, "NULL"),
    (dict(store=1), N.E_INVALID, "scales"),
    (dict(v=P + 4), N.E_LAYOUT, "misaligned"),
    (dict(n_seqs=0), N.E_INVALID, "n_seqs"),
    (dict(pages_per_seq=0), N.E_INVALID, "pages_per_seq"),
    (dict(page_table=None), N.E_INVALID, "NULL"),
    (dict(seq_lens=None), N.E_INVALID, "NULL"),
    (dict(seq_lens=P + 2), N.E_LAYOUT, "misaligned"),
]


@pytest.mark.parametrize("kw,code,msg", COMMON + [
    (dict(query_len=0), N.E_INVALID, "new tokens"),
    (dict(cu_seqlens=P, tokens=0), N.E_INVALID, "new tokens"),
    (dict(n_seqs=1 << 16, query_len=1 << 15), N.E_INVALID, "2^31"),
])
def test_write_and_attention_reject(kw, code, msg):
    lib = N.load_library()
    c, b, p = structs(**kw)
    assert lib.cra_cache_write(c, b, T, T, 128, None) == code
    assert msg in lib.cra_last_error().decode()
    assert lib.cra_fwd_paged(c, b, p, T, T, None, 0, None) == code
    assert msg in lib.cra_last_error().decode()
    assert lib.cra_fwd_paged_workspace_bytes(c, b, p) == 0


@pytest.mark.parametrize("kw,code,msg", COMMON)
def test_read_rejects(kw, code, msg):
    lib = N.load_library()
    c, b, _ = structs(**kw)
    assert lib.cra_cache_read(c, b, 10, 128, P, P, None) == code
    assert msg in lib.cra_last_error().decode()


@pytest.mark.parametrize("kw,msg", [
    (dict(H_q=7), "multiple"), (dict(H_q=0), "multiple"), (dict(qD=130), "multiple of 8"),
    (dict(qD=136), "multiple of 8"), (dict(qD=0), "multiple of 8"), (dict(window=-1), "window"),
    (dict(relay=2), "relay"), (dict(relay=-2), "relay"), (dict(top_k=0), "top_k"), (dict(top_k=5), "top_k"),
    (dict(relay=1, top_k=9), "top_k"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(max_seqlen=0), "max_seqlen"), (dict(cu_seqlens=P, tokens=5, max_query_len=0), "max_query_len"),
    (dict(n_seqs=1 << 14, query_len=1 << 15), "2^30"),
    (dict(window=1 << 30, max_seqlen=1 << 30, pages_per_seq=1 << 24, table_stride=1 << 24), "2^30 keys"),
    (dict(max_seqlen=(1 << 31) - 1, pages_per_seq=1 << 25, table_stride=1 << 25), "2^31"),
])
def test_attention_rejects_plans(kw, msg):
    lib = N.load_library()
    c, b, p = structs(**kw)
    assert lib.cra_fwd_paged(c, b, p, T, T, P, 1 << 30, None) == N.E_INVALID
    assert msg in lib.cra_last_error().decode()


def test_rows_and_workspace():
    lib = N.load_library()
    odd, null = N.CraTensor(P + 2, 0, 0, 0), N.CraTensor(None, 0, 0, 0)
    skew = N.CraTensor(P, 1 << 16, 132, 1024)
    c, b, p = structs()
    for bad, code in ((odd, N.E_LAYOUT), (skew, N.E_LAYOUT), (null, N.E_INVALID)):
        assert lib.cra_cache_write(c, b, bad, T, 128, None) == code
        assert lib.cra_cache_write(c, b, T, bad, 128, None) == code
        assert lib.cra_fwd_paged(c, b, p, bad, T, P, 1 << 30, None) == code
        assert lib.cra_fwd_paged(c, b, p, T, bad, P, 1 << 30, None) == code
    for D in (0, 4, 12, 136):
        assert lib.cra_cache_write(c, b, T, T, D, None) == N.E_INVALID
    assert lib.cra_cache_read(c, b, 0, 128, P, P, None) == N.E_INVALID
    assert lib.cra_cache_read(c, b, 4, 129, P, P, None) == N.E_INVALID
    assert lib.cra_cache_read(c, b, 4, 128, P + 4, P, None) == N.E_LAYOUT
    assert lib.cra_cache_read(c, b, 1 << 30, 128, P, P, None) == N.E_INVALID
    c, b, p = structs(max_seqlen=100000, pages_per_seq=5000)  # relay rows to list
    need = lib.cra_fwd_paged_workspace_bytes(c, b, p)
    assert need > 0
    assert lib.cra_fwd_paged(c, b, p, T, T, None, need, None) == N.E_INVALID
    assert lib.cra_fwd_paged(c, b, p, T, T, P, need - 1, None) == N.E_WORKSPACE
    assert str(need) in lib.cra_last_error().decode()
    c, b, p = structs(n_seqs=1 << 23, query_len=1)
    assert lib.cra_fwd_paged(c, b, p, T, T, P, 1 << 60, None) == N.E_INVALID
    assert "one launch" in lib.cra_last_error().decode()


def test_workspace_covers_the_list_of_any_length():
    """The list holds the global rows of every length up to the bound, under the rule and under fixed windows."""
    lib = N.load_library()
    for top in (2049, 3000, 4096, 4097, 40000, 131072):
        for window in (0, 1, 5, 363, 4096):
            for relay in (-1, 1):
                c, b, p = structs(max_seqlen=top, pages_per_seq=4096, window=window, relay=relay, n_seqs=1,
                                  query_len=64)  # 256 rows: no partial results in the workspace
                ws = lib.cra_fwd_paged_workspace_bytes(c, b, p)
                for n in {top, top - 1, top // 2, top // 3 + 1, 2049}:
                    W = min(n, window) if window else math.isqrt(n - 1) + 1
                    ls = max(0, n - W)
                    rows = 3 * (ls // W) + (1 if ls % W else 0)
                    if n <= top and (relay == 1 or n > 2048):
                        assert 2 * 4 * rows <= ws, (top, window, n)


def test_python_refusals_without_a_gpu():
    with pytest.raises(RuntimeError, match="GPU"):
        cra.PagedKVCache(4, 2, 64, device="cpu")
    k = torch.zeros(4, 2, 16, 64)
    n = torch.zeros(4, 2, 16)
    with pytest.raises(RuntimeError, match="GPU"):
        cra.PagedKVCache.from_tensors(k, k, n)
    for bad, exc in ((dict(page_size=24), ValueError), (dict(page_size=2048), ValueError),
                     (dict(num_pages=0), ValueError), (dict(head_dim=257), NotImplementedError),
                     (dict(head_dim=0), NotImplementedError), (dict(dtype=torch.float64), TypeError),
                     (dict(storage=torch.float8_e5m2), TypeError), (dict(storage=torch.float16), TypeError)):
        with pytest.raises(exc):
            cra.PagedKVCache(**{**dict(num_pages=4, n_kv_heads=2, head_dim=64, device="cpu"), **bad})
    with pytest.raises(ValueError, match="width"):
        cra.PagedKVCache.from_tensors(k, k, n, head_dim=48)
    with pytest.raises(ValueError, match="k_norm"):
        cra.PagedKVCache.from_tensors(k, k, n[:3])
    with pytest.raises(ValueError, match="alike"):
        cra.PagedKVCache.from_tensors(k, k[:3], n)
    with pytest.raises(ValueError, match="scales"):
        cra.PagedKVCache.from_tensors(k, k, n, n, n)


WRITE_ROWS = r"""
#include "cra_paged.hpp"
#include <cstdio>
using namespace cra;
int main() {
  long bad = 0;
  for (int pages : {1, 2, 5})
    for (int len = -3; len <= 100; ++len)
      for (int count : {1, 2, 17, 200})
        for (int t = 0; t < count; ++t) {
          const int row = len - count + t, cap = pages * 16;
          bad += write_row(len, count, t, pages, 4) != (len > 0 && row >= 0 && row < cap && row < len ? row : -1);
        }
  // the ends of the range
  bad += write_row(0x7fffffff, 1, 0, 4, 4) != -1 || write_row(-0x7fffffff - 1, 0x7fffffff, 0, 4, 4) != -1;
  bad += write_row(0x7fffffff, 5, 1, 0x7fffffff, 10) != 0x7ffffffb || write_row(64, 0x7fffffff, 0x7ffffffe, 4, 4) != 63;
  // offsets that run backwards: a token outside its sequence's range stays inside the table
  for (int t : {-0x7fffffff - 1, -70, 3, 70, 0x7fffffff})
    for (int len : {1, 64, 0x7fffffff}) {
      const int row = write_row(len, 2, t, 4, 4);
      bad += row < -1 || row >= 64;
    }
  printf("%ld\n", bad);
  return 0;
}
"""


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")
def test_rows_that_new_tokens_are_written_to(tmp_path):
    src, exe = tmp_path / "rows.cpp", tmp_path / "rows"
    src.write_text(WRITE_ROWS)
    subprocess.run([HIPCC, "-std=c++17", "-O1", "-I", CSRC, str(src), "-o", str(exe)], check=True,
                   capture_output=True, timeout=300)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=120)
    assert int(out.stdout) == 0


def test_a_head_dim_of_zero_is_no_default():
    k, n = torch.zeros(4, 2, 16, 64), torch.zeros(4, 2, 16)
    with pytest.raises(NotImplementedError, match="head dim 0"):
        cra.PagedKVCache.from_tensors(k, k, n, head_dim=0)
