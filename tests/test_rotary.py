"""Rotary tables and the refusals of the rotary operators (no GPU needed): the
frequencies against their formulas, angles of far positions, argument checks of
the Python layer and of the C ABI before any launch."""
import ctypes
import math

import pytest
import torch

import cron_root_attention as cra
from cron_root_attention import _native as N
from cron_root_attention.rotary import rotary_frequencies


def test_frequencies_without_scaling():
    f, mul = rotary_frequencies(64, 500000.0)
    assert mul == 1.0
    assert torch.equal(f, torch.tensor([500000.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64))


def test_linear_and_ntk_scaling():
    f, _ = rotary_frequencies(64)
    lin, mul = rotary_frequencies(64, scaling={"type": "linear", "factor": 4})
    assert mul == 1.0 and torch.allclose(lin, f / 4, rtol=1e-15)
    ntk, _ = rotary_frequencies(64, scaling={"type": "ntk", "factor": 4})
    assert ntk[0] == 1.0
    # the slowest pair is stretched by exactly the factor
    assert math.isclose(float(ntk[-1]), float(f[-1]) / 4, rel_tol=1e-12)


def test_yarn_scaling_keeps_fast_pairs_and_stretches_slow_ones():
    n, d, factor = 4096, 128, 8.0
    f, _ = rotary_frequencies(d)
    y, mul = rotary_frequencies(d, scaling={"type": "yarn", "factor": factor, "original_positions": n})
    turns = f * n / (2 * math.pi)
    assert torch.equal(y[turns > 40], f[turns > 40])
    assert torch.allclose(y[turns < 0.8], f[turns < 0.8] / factor, rtol=1e-15)
    assert bool((y[1:] <= y[:-1]).all()) and bool((y <= f).all()) and bool((y >= f / factor * (1 - 1e-15)).all())
    assert math.isclose(mul, 0.1 * math.log(8.0) + 1)
    assert rotary_frequencies(d, scaling={"type": "yarn", "factor": factor, "original_positions": n,
                                          "attention_factor": 1.25})[1] == 1.25


@pytest.mark.parametrize("scaling", [{"type": "other", "factor": 2}, {"type": "linear", "factor": 0},
                                     {"type": "linear", "factor": 2, "original_positions": 5},
                                     {"type": "ntk", "factor": -1}])
def test_unknown_scalings_are_refused(scaling):
    with pytest.raises(ValueError):
        rotary_frequencies(64, scaling=scaling)


def test_table_of_far_positions():
    """A row of the table is the fp64 angle's cosine and sine rounded once: with
    p f in fp32 the angle at position 10^6 would be off by 0.03."""
    t = cra.RotaryTable(32, 1_000_003)
    assert t.table.shape == (1_000_003, 32) and t.max_positions == 1_000_003
    f, _ = rotary_frequencies(32)
    for p in (0, 1, 77777, 1_000_002):
        for i in range(16):
            a = p * float(f[i])
            assert abs(float(t.table[p, i]) - math.cos(a)) <= 2.0 ** -24
            assert abs(float(t.table[p, 16 + i]) - math.sin(a)) <= 2.0 ** -24
    assert t.to("cpu") is t


@pytest.mark.parametrize("dim,n", [(3, 10), (-2, 10), (4, 0)])
def test_bad_tables(dim, n):
    with pytest.raises(ValueError):
        cra.RotaryTable(dim, n)


def test_cpu_tensors_are_refused():
    t = cra.RotaryTable(8, 16)
    q = torch.zeros(1, 2, 4, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        cra.rotary_embedding(q, q, t)
    with pytest.raises(RuntimeError, match="GPU"):
        cra.qk_norm_rotary(q, q, None, None, t)
    with pytest.raises(ValueError, match=r"\[B, H, S, D\]"):
        cra.rotary_embedding(q[0], None, t)


# ------------------------------------------------------------------ C ABI
GOOD = dict(B=1, H_q=4, H_kv=2, S=10, D=64, rot=64, interleaved=0, norm=0, dtype=0, weight_dtype=0,
            positions_64=0, eps=1e-6, table=0x10000, table_rows=100, positions=None, psb=0, pss=0)
T = N.CraTensor(0x10000, 1 << 16, 64, 256)


def turn(**kw):
    return ctypes.byref(N.CraTurn(**{**GOOD, **kw}))


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dtype=5), N.E_DTYPE, "dtype"),
    (dict(B=0), N.E_INVALID, ">= 1"),
    (dict(S=0), N.E_INVALID, ">= 1"),
    (dict(H_q=0), N.E_INVALID, ">= 1"),
    (dict(H_kv=-1), N.E_INVALID, ">= 0"),
    (dict(D=257, rot=0), N.E_UNSUPPORTED, "256"),
    (dict(rot=63), N.E_INVALID, "even"),
    (dict(rot=66), N.E_INVALID, "even"),
    (dict(rot=-2), N.E_INVALID, "even"),
    (dict(table=None), N.E_INVALID, "table"),
    (dict(table_rows=0), N.E_INVALID, "table"),
    (dict(norm=2), N.E_INVALID, "norm"),
    (dict(norm=1, eps=-1.0), N.E_INVALID, "eps"),
    (dict(norm=1, eps=float("nan")), N.E_INVALID, "eps"),
    (dict(norm=1, weight_dtype=1), N.E_DTYPE, "weights"),
    (dict(B=1 << 20, S=1 << 20), N.E_INVALID, "2^31"),
    (dict(B=1 << 10, S=1 << 18, D=255, rot=0, H_q=8), N.E_INVALID, "one launch"),
])
def test_rotary_rejects(kw, code, msg):
    lib = N.load_library()
    assert lib.cra_rotary(turn(**kw), T, T, None, None, T, T, 0, None) == code
    assert msg in lib.cra_last_error().decode()


def test_rotary_rejects_pointers_and_misuse():
    lib = N.load_library()
    null, odd = N.CraTensor(None, 0, 0, 0), N.CraTensor(0x10001, 0, 0, 0)
    assert lib.cra_rotary(turn(), null, T, None, None, T, T, 0, None) == N.E_INVALID
    assert lib.cra_rotary(turn(), T, T, None, None, T, null, 0, None) == N.E_INVALID
    assert lib.cra_rotary(turn(), T, odd, None, None, T, T, 0, None) == N.E_LAYOUT
    assert lib.cra_rotary(turn(norm=1), T, T, None, None, T, T, 1, None) == N.E_INVALID
    assert lib.cra_rotary(None, T, T, None, None, T, T, 0, None) == N.E_INVALID
    bwd = lib.cra_norm_rotary_bwd
    assert bwd(turn(), T, T, None, None, T, T, T, T, None, None, None, 0, None) == N.E_INVALID
    assert bwd(turn(norm=1), T, T, None, None, T, T, T, T, 0x10000, None, 0x10000, 1 << 30, None) == N.E_INVALID
    need = lib.cra_rotary_bwd_workspace_bytes(turn(norm=1))
    assert need > 0
    w = 0x10000
    assert bwd(turn(norm=1), T, T, w, w, T, T, T, T, w, w, None, need, None) == N.E_INVALID
    assert bwd(turn(norm=1), T, T, w, w, T, T, T, T, w, w, w, need - 1, None) == N.E_WORKSPACE
    assert lib.cra_rotary_bwd_workspace_bytes(turn(D=300)) == 0
