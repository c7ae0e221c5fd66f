"""Rotary positions of query and key heads, alone or behind a norm of each head.

The reference leaves positions and head norms to its callers; here they are one
pass over q and k between the projections and the attention
(``csrc/cra_rotary.hip``): read once, written once, with the angles from a table
and fp32 arithmetic.  Both operators take and give ``[B, H, S, D]`` tensors in
any layout with D contiguous (a slice of a fused projection is read in place)
and are differentiable once, in reverse mode; the gradients of the norm weights are
summed in a fixed order.
"""
from __future__ import annotations

import functools
import math
from typing import Optional, Tuple

import torch

from . import _native

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


def rotary_frequencies(rotary_dim: int, base: float = 10000.0,
                       scaling: Optional[dict] = None) -> Tuple[torch.Tensor, float]:
    """(angle per position of each pair, fp64 [rotary_dim / 2]; multiplier of cos and sin).

    ``scaling`` stretches the positions for contexts beyond the trained ones:
    ``{"type": "linear", "factor": f}`` divides every frequency by f;
    ``{"type": "ntk", "factor": f}`` raises the base to base * f^(d / (d - 2));
    ``{"type": "yarn", "factor": f, "original_positions": n}`` keeps the pairs
    that make more than ``beta_fast`` (32) turns over n positions, divides those
    that make fewer than ``beta_slow`` (1) by f, and goes linearly between; cos
    and sin are multiplied by ``attention_factor`` (0.1 ln f + 1).
    """
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and >= 0, got {rotary_dim}")
    if not base > 0:
        raise ValueError(f"base must be > 0, got {base}")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    kind = "none" if scaling is None else scaling.get("type")
    if kind == "none":
        return base ** (-2.0 * i / max(rotary_dim, 1)), 1.0
    if kind not in ("linear", "ntk", "yarn"):
        raise ValueError(f"unknown scaling type {kind!r}: linear, ntk or yarn")
    known = {"type", "factor"} | ({"original_positions", "beta_fast", "beta_slow",
                                   "attention_factor"} if kind == "yarn" else set())
    if set(scaling) - known:
        raise ValueError(f"unknown keys in a {kind} scaling: {sorted(set(scaling) - known)}")
    factor = float(scaling["factor"])
    if not factor > 0:
        raise ValueError(f"scaling factor must be > 0, got {factor}")
    if kind == "ntk":
        if rotary_dim > 2:
            base = base * factor ** (rotary_dim / (rotary_dim - 2))
        return base ** (-2.0 * i / max(rotary_dim, 1)), 1.0
    f = base ** (-2.0 * i / max(rotary_dim, 1))
    if kind == "linear":
        return f / factor, 1.0
    n = float(scaling["original_positions"])

    def pair_with(turns: float) -> float:
        return rotary_dim * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))
    lo = max(0, math.floor(pair_with(float(scaling.get("beta_fast", 32.0)))))
    hi = min(rotary_dim - 1, math.ceil(pair_with(float(scaling.get("beta_slow", 1.0)))))
    slow = ((i - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
    mul = scaling.get("attention_factor")
    if mul is None:
        mul = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return f * (1 - slow) + f / factor * slow, float(mul)


class RotaryTable:
    """cos and sin of positions 0 .. max_positions - 1, fp32 ``[max_positions, rotary_dim]``
    (row p: rotary_dim / 2 cosines, then as many sines), with the way pairs lie in
    a head. Angles are formed in 64 bits: p * f of a far position has no bits left
    behind the point in 32."""

    def __init__(self, rotary_dim: int, max_positions: int, base: float = 10000.0,
                 scaling: Optional[dict] = None, interleaved: bool = False, device=None):
        if max_positions < 1:
            raise ValueError(f"max_positions must be >= 1, got {max_positions}")
        freq, mul = rotary_frequencies(rotary_dim, base, scaling)
        self.rotary_dim = int(rotary_dim)
        self.interleaved = bool(interleaved)
        angle = torch.arange(max_positions, dtype=torch.float64,
                             device=device)[:, None] * freq.to(device)
        self.table = torch.cat([angle.cos() * mul, angle.sin() * mul], 1).to(torch.float32)

    @property
    def max_positions(self) -> int:
        return self.table.shape[0]

    @property
    def device(self) -> torch.device:
        return self.table.device

    def to(self, device) -> "RotaryTable":
        """This table on another device (itself if it is there already)."""
        table = self.table.to(device)
        if table is self.table:
            return self
        other = object.__new__(RotaryTable)
        other.rotary_dim, other.interleaved, other.table = self.rotary_dim, self.interleaved, table
        return other


def _check_rows(q, k):
    for name, t in (("q", q), ("k", k)):
        if t is None:
            continue
        if t.dim() != 4:
            raise ValueError(f"{name} must be [B, H, S, D]")
        if t.device.type != "cuda":
            raise RuntimeError(f"the rotary operators run on ROCm GPU tensors only (got {t.device})")
        if t.dtype not in _DTYPES:
            raise TypeError(f"unsupported dtype {t.dtype}; use float16, bfloat16 or float32")
        if min(t.shape) < 1:
            raise ValueError(f"{name} has an empty dimension: {tuple(t.shape)}")
        if max(t.shape) > 2**31 - 1:
            raise ValueError(f"{name} has a dimension of 2^31 or more: {tuple(t.shape)}")
    if k is not None:
        if (q.shape[0], q.shape[2], q.shape[3]) != (k.shape[0], k.shape[2], k.shape[3]):
            raise ValueError(f"k shape {tuple(k.shape)} does not match q {tuple(q.shape)}")
        if q.dtype != k.dtype:
            raise TypeError(f"q and k dtypes differ: {q.dtype}, {k.dtype}")
        if q.device != k.device:
            raise ValueError("q and k must be on the same device")


def _check_positions(q, table, positions):
    """The table's and the positions' part of the problem; positions as [B or 1, S]."""
    B, _, S, D = q.shape
    if table is None:
        if positions is not None:
            raise ValueError("positions without a table")
        return None
    if not isinstance(table, RotaryTable):
        raise TypeError("table must be a RotaryTable")
    if table.device != q.device:
        raise ValueError(f"the table is on {table.device} but q is on {q.device}")
    t = table.table
    if t.dtype != torch.float32 or not t.is_contiguous() or t.shape[1:] != (table.rotary_dim,):
        raise ValueError(f"the table's rows must be contiguous float32 [positions, {table.rotary_dim}]")
    if _grad(t):
        raise NotImplementedError("a rotary table has no gradient")
    if table.rotary_dim > D:
        raise ValueError(f"the table turns {table.rotary_dim} elements, the heads have {D}")
    if positions is None:
        if S > table.max_positions:
            raise ValueError(f"{S} tokens but the table has {table.max_positions} positions")
        return None
    if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
        raise TypeError("positions must be an int32 or int64 tensor")
    if positions.device != q.device:
        raise ValueError(f"positions are on {positions.device} but q is on {q.device}")
    if positions.dim() == 1:
        positions = positions[None]
    if positions.dim() != 2 or positions.shape[0] not in (1, B) or positions.shape[1] != S:
        raise ValueError(f"positions must be [S] or [B, S], got {tuple(positions.shape)}")
    return positions


def _problem(q, k, table, positions, norm: bool, weight_dtype, eps: float):
    B, Hq, S, D = q.shape
    turns = table is not None and table.rotary_dim > 0
    pos = positions if turns else None
    return _native.CraTurn(
        B, Hq, 0 if k is None else k.shape[1], S, D, table.rotary_dim if turns else 0,
        int(turns and table.interleaved), int(norm), _native.dtype_code(q.dtype),
        _native.dtype_code(weight_dtype), int(pos is not None and pos.dtype == torch.int64),
        float(eps), table.table.data_ptr() if turns else None,
        table.max_positions if turns else 0, None if pos is None else pos.data_ptr(),
        pos.stride(0) if pos is not None and pos.shape[0] > 1 else 0,
        pos.stride(1) if pos is not None else 0)


def _rows(t):
    return t if t is None or t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _grads(dys, like):
    """Upstream gradients in the rows' type, D contiguous; zeros for an output that got none."""
    return [None if x is None else torch.zeros_like(x) if d is None else _rows(d.to(x.dtype))
            for d, x in zip(dys, like)]


def _once(backward):
    """Gradients that are not differentiated again: under create_graph they carry a
    node that raises when they are."""
    @functools.wraps(backward)
    def wrapped(ctx, *grads):
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not torch.is_grad_enabled():
            return out
        error = torch._C._functions.DelayedError(
            f"{type(ctx).__name__} has no second derivative".encode(), len(out))
        return error(*(t if t is None else t.detach().requires_grad_() for t in out))
    return wrapped


class RotaryFunction(torch.autograd.Function):
    """Rotation of q and k; the backward turns the gradients back."""

    @staticmethod
    def forward(ctx, q, k, table, positions):
        ctx.table = table
        ctx.save_for_backward(table.table, positions)  # a change before the backward raises
        ctx.set_materialize_grads(False)
        q, k = _rows(q), _rows(k)
        ctx.dtype = q.dtype
        return _native.rotary(_problem(q, k, table, positions, False, q.dtype, 0.0), q, k, None, None)

    @staticmethod
    @_once
    def backward(ctx, dyq, dyk):
        one = [x for x in (dyq, dyk) if x is not None]
        if not one:
            return None, None, None, None
        one = [_rows(x.to(ctx.dtype)) for x in one]
        _, positions = ctx.saved_tensors
        y = _native.rotary(_problem(one[0], one[1] if len(one) > 1 else None, ctx.table,
                                    positions, False, ctx.dtype, 0.0),
                           one[0], one[1] if len(one) > 1 else None, None, None, transpose=True)
        if len(one) == 2:
            return y[0], y[1], None, None
        return (y[0], None, None, None) if dyq is not None else (None, y[0], None, None)


class NormRotaryFunction(torch.autograd.Function):
    """Norm of each head of q and k, then the rotation."""

    @staticmethod
    def forward(ctx, q, k, wq, wk, table, positions, eps):
        q, k = _rows(q), _rows(k)
        ctx.args = table, eps
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, wq, wk, None if table is None else table.table, positions)
        return _native.rotary(_problem(q, k, table, positions, True, _weight_dtype(q, wq, wk), eps),
                              q, k, wq, wk)

    @staticmethod
    @_once
    def backward(ctx, dyq, dyk):
        q, k, wq, wk, _, positions = ctx.saved_tensors
        table, eps = ctx.args
        if dyq is None and dyk is None:
            return (None,) * 7
        q, k = _rows(q), _rows(k)  # layouts that a saved-tensor hook changed
        dyq, dyk = _grads((dyq, dyk), (q, k))
        need = ctx.needs_input_grad
        dq, dk, dwq, dwk = _native.norm_rotary_backward(
            _problem(q, k, table, positions, True, _weight_dtype(q, wq, wk), eps), q, k, wq, wk,
            dyq, dyk, wq is not None and need[2], wk is not None and need[3])
        return dq, dk, dwq, dwk, None, None, None


def _weight_dtype(q, wq, wk):
    w = wq if wq is not None else wk
    return q.dtype if w is None else w.dtype


def _grad(*ts) -> bool:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        return True
    return _native.has_tangent(*ts)  # the Functions raise: forward mode is not built


@torch.compiler.disable
def rotary_embedding(q: torch.Tensor, k: Optional[torch.Tensor], table: RotaryTable,
                     positions: Optional[torch.Tensor] = None):
    """Turn the heads of q and k by their tokens' positions.

    Args:
        q: [B, H_q, S, D]; k: [B, H_kv, S, D] or None. D up to 256.
        table: the angles; the first ``table.rotary_dim`` elements of a head turn.
        positions: int32 or int64 [S] or [B, S] on the GPU; None: 0 .. S - 1. A
            position outside the table gives NaN in the elements that turn.

    Returns: (q, k) turned, in their dtype and layout; without k only q.
    """
    op = _native.fast_op("rotary") if type(table) is RotaryTable else None
    if op is not None:
        y = op(q, k, None, None, table.table, positions, table.interleaved, False, 0.0)
        if y:
            return y[0] if k is None else (y[0], y[1])
    # what the operator does not take (or nobody does: the checks say why)
    _check_rows(q, k)
    if table is None:
        raise TypeError("table must be a RotaryTable")
    positions = _check_positions(q, table, positions)
    if _grad(q, k):
        y = RotaryFunction.apply(q, k, table, positions)
    else:
        q, k = _rows(q), _rows(k)
        y = _native.rotary(_problem(q, k, table, positions, False, q.dtype, 0.0), q, k, None, None)
    return y[0] if k is None else y


@torch.compiler.disable
def qk_norm_rotary(q: torch.Tensor, k: Optional[torch.Tensor], q_weight: Optional[torch.Tensor],
                   k_weight: Optional[torch.Tensor], table: Optional[RotaryTable] = None,
                   positions: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """Divide each head of q and k by its root mean square, multiply by the
    weights, and turn it (:func:`rotary_embedding`), in one pass.

    Args:
        q_weight, k_weight: [D] in the rows' dtype or float32, one dtype for both;
            None: ones. Differentiable.
        table: None: the norm alone.

    Returns: (q, k) in their dtype and layout; without k only q.
    """
    op = _native.fast_op("rotary") if table is None or type(table) is RotaryTable else None
    if op is not None:
        y = op(q, k, q_weight, k_weight, None if table is None else table.table, positions,
               table is not None and table.interleaved, True, eps)
        if y:
            return y[0] if k is None else (y[0], y[1])
    _check_rows(q, k)
    positions = _check_positions(q, table, positions)
    D = q.shape[3]
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            continue
        if w.shape != (D,):
            raise ValueError(f"{name} must have shape [{D}], got {tuple(w.shape)}")
        if w.device != q.device:
            raise ValueError(f"{name} is on {w.device} but q is on {q.device}")
        if w.dtype not in (q.dtype, torch.float32):
            raise TypeError(f"{name} must be {q.dtype} or float32, got {w.dtype}")
    if k is None and k_weight is not None:
        raise ValueError("k_weight without k")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise TypeError("q_weight and k_weight dtypes differ")
    if not eps >= 0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    wq, wk = (w if w is None or w.is_contiguous() else w.contiguous() for w in (q_weight, k_weight))
    if _grad(q, k, wq, wk):
        y = NormRotaryFunction.apply(q, k, wq, wk, table, positions, float(eps))
    else:
        q, k = _rows(q), _rows(k)
        y = _native.rotary(_problem(q, k, table, positions, True, _weight_dtype(q, wq, wk), eps),
                           q, k, wq, wk)
    return y[0] if k is None else y
