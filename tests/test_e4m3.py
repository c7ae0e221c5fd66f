"""8-bit products, appending and shared prefixes without a GPU: refusals of the C ABI
before any launch, and of the Python layer; the split of global rows at a prefix."""
import ctypes
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
lib = N.load_library()
PTR = 1 << 20  # an aligned address that is never used


def error():
    return lib.cra_last_error().decode()


def linear(M=4, N_=8, K=128, dtype=N.BF16):
    return N.CraLinear(M, N_, K, dtype)


@pytest.mark.parametrize("change,code", [
    (dict(M=0), N.E_INVALID), (dict(N_=0), N.E_INVALID), (dict(K=0), N.E_INVALID), (dict(K=(1 << 22) + 1), N.E_INVALID),
    (dict(dtype=7), N.E_DTYPE), (dict(M=1 << 33), N.E_INVALID)])
def test_product_sizes(change, code):
    p = linear(**change)
    assert lib.cra_linear_e4m3(ctypes.byref(p), PTR, 128, PTR, PTR, None, PTR, 8, PTR, 1 << 40, None) == code
    assert lib.cra_linear_e4m3_workspace_bytes(ctypes.byref(p)) == 0
    assert error()


def test_product_pointers_and_workspace():
    p = linear(M=100)
    need = lib.cra_linear_e4m3_workspace_bytes(ctypes.byref(p))
    assert need >= 100 * 128 + 100 * 4

    def call(x=PTR, w=PTR, s=PTR, bias=None, y=PTR, ws=PTR, n=need):
        return lib.cra_linear_e4m3(ctypes.byref(p), x, 128, w, s, bias, y, 8, ws, n, None)
    for kw in (dict(x=None), dict(w=None), dict(s=None), dict(y=None), dict(ws=None), dict(ws=PTR + 8)):
        assert call(**kw) == N.E_INVALID
    for kw in (dict(x=PTR + 1), dict(w=PTR + 8), dict(s=PTR + 2), dict(bias=PTR + 1), dict(y=PTR + 1)):
        assert call(**kw) == N.E_LAYOUT
    assert call(n=need - 1) == N.E_WORKSPACE
    assert lib.cra_linear_e4m3(None, PTR, 128, PTR, PTR, None, PTR, 8, PTR, need, None) == N.E_INVALID
    assert lib.cra_linear_e4m3_workspace_bytes(ctypes.byref(linear(M=1))) == 0  # few rows need none


def test_weights_and_rows():
    assert lib.cra_e4m3_weight(None, 8, 8, 8, N.F16, PTR, PTR, None) == N.E_INVALID
    assert lib.cra_e4m3_weight(PTR, 8, 0, 8, N.F16, PTR, PTR, None) == N.E_INVALID
    assert lib.cra_e4m3_weight(PTR, 8, 8, 8, 9, PTR, PTR, None) == N.E_DTYPE
    assert lib.cra_e4m3_weight(PTR, 8, 8, 8, N.F16, PTR + 4, PTR, None) == N.E_LAYOUT
    assert lib.cra_e4m3_weight(PTR, 8, 1 << 24, 8, N.F16, PTR, PTR, None) == N.E_INVALID
    assert lib.cra_e4m3_rows(PTR, 8, 8, 8, N.F16, None, PTR, None) == N.E_INVALID
    assert lib.cra_e4m3_rows(PTR + 1, 8, 8, 8, N.F16, PTR, PTR, None) == N.E_LAYOUT


def cache(**kw):
    a = dict(k=PTR, v=PTR, k_norm=PTR, k_scale=None, v_scale=None, num_pages=8, H_kv=2, page_size=16, D=64, dtype=N.BF16,
             store=0) | kw
    return N.CraCache(*a.values())


def batch(**kw):
    a = dict(page_table=PTR, table_stride=4, seq_lens=PTR, cu_seqlens=None, n_seqs=2, pages_per_seq=4, tokens=0,
             query_len=1) | kw
    return N.CraBatch(*a.values())


def turn(**kw):
    a = dict(B=2, H_q=4, H_kv=2, S=1, D=64, rot=64, interleaved=0, norm=0, dtype=N.BF16, weight_dtype=N.BF16, positions_64=0,
             eps=1e-6, table=PTR, table_rows=64, positions=None, psb=0, pss=0) | kw
    return N.CraTurn(*a.values())


def rows(ptr=PTR, s=64):
    return N.CraTensor(ptr, s, s, s)


@pytest.mark.parametrize("c,b,p,code", [
    (dict(page_size=8), {}, {}, N.E_INVALID), ({}, dict(n_seqs=0), {}, N.E_INVALID), ({}, {}, dict(rot=63), N.E_INVALID),
    ({}, {}, dict(dtype=N.F16), N.E_DTYPE), ({}, {}, dict(H_kv=1), N.E_INVALID), ({}, {}, dict(D=60), N.E_INVALID),
    ({}, {}, dict(D=128), N.E_INVALID), ({}, {}, dict(B=1), N.E_INVALID), ({}, {}, dict(S=2), N.E_INVALID),
    ({}, {}, dict(table=None), N.E_INVALID), ({}, {}, dict(norm=1, eps=-1.0), N.E_INVALID),
    ({}, dict(cu_seqlens=PTR, tokens=5), dict(B=1, S=4), N.E_INVALID), ({}, {}, dict(rot=6), N.E_UNSUPPORTED)])
def test_append_arguments(c, b, p, code):
    args = cache(**c), batch(**b), turn(**p)
    r = lib.cra_cache_append(*map(ctypes.byref, args), rows(), rows(), rows(), None, None, rows(), None)
    assert r == code and error()


def test_append_rows():
    args = [ctypes.byref(x) for x in (cache(), batch(), turn())]
    for i in range(4):
        t = [rows()] * 4
        for bad, code in ((rows(None), N.E_INVALID), (rows(PTR + 8), N.E_LAYOUT), (rows(s=60), N.E_LAYOUT)):
            t[i] = bad
            assert lib.cra_cache_append(*args, t[0], t[1], t[2], None, None, t[3], None) == code


def plan(**kw):
    a = dict(H_q=4, D=64, window=64, relay=-1, top_k=2, max_query_len=1, max_seqlen=64, zero_outside=1, scale=0.125) | kw
    return N.CraPagedPlan(*a.values())


def test_shared_prefix_arguments():
    c, b = cache(), batch()

    def call(x, p=None, n=1 << 40):
        p = p or plan()
        return lib.cra_fwd_paged_shared(ctypes.byref(c), ctypes.byref(b), ctypes.byref(p), None if x is None else ctypes.byref(x),
                                        rows(), rows(), PTR, n, None)
    good = N.CraPrefix(PTR, PTR, 2)
    assert call(None) == N.E_INVALID
    assert call(good, plan(window=0)) == N.E_INVALID and "window" in error()
    for bad, code in ((N.CraPrefix(None, PTR, 2), N.E_INVALID), (N.CraPrefix(PTR, None, 2), N.E_INVALID),
                      (N.CraPrefix(PTR + 2, PTR, 2), N.E_LAYOUT), (N.CraPrefix(PTR, PTR, 0), N.E_INVALID),
                      (N.CraPrefix(PTR, PTR, 1 << 27), N.E_INVALID)):
        assert call(bad) == code
    # keys of a query: global rows of blocks of the window, and the window
    long = N.CraPrefix(PTR, PTR, (1 << 29) // c.page_size)
    assert call(long, plan(window=1)) == N.E_INVALID and "2^30" in error()
    assert call(long, plan(window=1, relay=0), n=0) == N.E_WORKSPACE
    need = lib.cra_fwd_paged_shared_workspace_bytes(*map(ctypes.byref, (c, b, plan(), good)))
    assert need > lib.cra_fwd_paged_workspace_bytes(*map(ctypes.byref, (c, b, plan())))
    assert call(good, n=need - 1) == N.E_WORKSPACE


PROGRAM = r"""
#include "cra_paged.hpp"
#include <cstdio>
using namespace cra;
int main() {
  long bad = 0, cases = 0;
  for (int W : {1, 2, 7, 16, 50})
    for (int rpb : {1, 3, 5})
      for (int P = 0; P < 120; ++P) {
        // a prefix's slots: first rows below P, and relay rows of blocks that end there
        int want = 0;
        for (int r = 0; r * W < P; ++r) want += 1 + ((r + 1) * W <= P ? rpb - 1 : 0);
        bad += prefix_slots(P, W, rpb) != want;
        for (int n = P + 1; n < P + 100; n += 3)
          for (int m = 1; m <= 3 && m <= n - P; ++m) {
            ++cases;
            const SeqPlan p{n, W < n ? W : n, rpb};
            const int G0 = p.W < n ? prefix_slots(P, W, rpb) : 0, G = seq_prefix(n - 1, p);
            const int pos0 = n - m, lo = pos0 - p.W + 1;
            const int own = (G > G0 ? (G - G0 + 31) / 32 : 0) + (n - (lo > P ? lo : P) + 31) / 32;
            bad += few_tile_count(n, m, p, P, G0) != own || own < 1 || own > few_tile_count(n, m, p);
          }
      }
  printf("%ld %ld\n", bad, cases);
  return bad != 0;
}
"""


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not found")
def test_global_rows_split_at_a_prefix(tmp_path):
    src = tmp_path / "c.cpp"
    src.write_text(PROGRAM)
    exe = tmp_path / "c"
    subprocess.run([HIPCC, "-x", "hip", "--offload-arch=gfx950", "-O1", "-std=c++17", "-w", f"-I{CSRC}", str(src), "-o", str(exe)],
                   check=True, capture_output=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout


def test_python_refusals_without_a_gpu():
    w = torch.zeros(4, 4)
    with pytest.raises(RuntimeError, match="GPU"):
        cra.E4M3Weight.from_dense(w)
    with pytest.raises(TypeError):
        cra.E4M3Weight.from_dense(w.long())
    with pytest.raises(ValueError):
        cra.E4M3Weight.from_dense(w[0])
    with pytest.raises(TypeError):
        cra.E4M3Weight(4, 4, w, w)
    with pytest.raises(ValueError):
        cra.E4M3Weight(4, 4, torch.zeros(4, 4, dtype=torch.uint8), torch.zeros(1, 4, dtype=torch.uint8))
    with pytest.raises(TypeError):
        cra.linear_e4m3(w, w)
    with pytest.raises(RuntimeError):
        cra.CronRootAttention(64, 2).to_e4m3()


def test_a_layer_pickled_before_it_could_hold_a_joint_projection():
    torch.manual_seed(0)
    layer = cra.CronRootAttention(64, 2).eval()
    state = {k: v for k, v in layer.__dict__.items() if k != "qkv_proj"}
    other = cra.CronRootAttention.__new__(cra.CronRootAttention)
    other.__setstate__(state)
    x = torch.randn(1, 9, 64)
    with torch.no_grad():
        assert torch.equal(other(x), layer(x))
    assert "qkv_proj" not in other.state_dict()
