"""Linear layers in 8-bit floating point, for serving.

The reference keeps its projections in 16 bits.  Here a weight is held as e4m3 codes
with a power-of-two scale for each block of 128 x 128 elements, half the memory a
decoding step reads, and the rows it meets are brought into the same form on the way,
with a scale for each row and 128 columns; the products run on the 8-bit matrix core,
which takes both scales itself (``csrc/cra_linear.hip``).  A power of two makes scaling
exact: what an element loses is the rounding to e4m3's 3 bits.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from . import _native

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
BLOCK = 128


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _exponents(k: int) -> int:
    """Exponent bytes of a row of k columns: its blocks, up to a multiple of four."""
    return (_blocks(k) + 3) // 4 * 4


def _check_gpu(name, t):
    if t.device.type != "cuda":
        raise RuntimeError(f"the 8-bit linear operators run on ROCm GPU tensors only ({name} is on {t.device})")


class E4M3Weight:
    """A weight [out_features, in_features] in 8 bits.

    ``codes``: float8_e4m3fn [out_features, in_features]; ``scales``: float32
    [ceil(out_features / 128), ceil(in_features / 128)], powers of two (the value of an
    element is its code times its block's scale).  Made by :meth:`from_dense` or
    :meth:`from_tensors`.
    """

    def __init__(self, out_features: int, in_features: int, codes: torch.Tensor, exponents: torch.Tensor):
        """Over the stored form: uint8 codes, rows a multiple of 128 long with zeros
        behind in_features, and exponent bytes, rows a multiple of four long."""
        N, K = int(out_features), int(in_features)
        if N < 1 or K < 1:
            raise ValueError(f"a weight needs at least one row and column, got [{N}, {K}]")
        for name, t, shape in (("codes", codes, (N, _blocks(K) * BLOCK)),
                               ("exponents", exponents, (_blocks(N), _exponents(K)))):
            if t.dtype != torch.uint8:
                raise TypeError(f"{name} must be uint8, got {t.dtype}")
            if tuple(t.shape) != shape or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous {list(shape)}, got {list(t.shape)}")
            _check_gpu(name, t)
        if codes.device != exponents.device:
            raise ValueError("codes and exponents must be on the same device")
        if codes.data_ptr() % 16 or exponents.data_ptr() % 4:
            raise ValueError("codes must lie on a 16-byte and exponents on a 4-byte address")
        self.out_features, self.in_features = N, K
        self._codes, self._exponents = codes, exponents

    @classmethod
    def from_dense(cls, weight: torch.Tensor) -> "E4M3Weight":
        """A weight of float16, bfloat16 or float32 elements, rounded to e4m3 (a block
        that holds an infinity or NaN becomes NaN)."""
        if weight.dim() != 2:
            raise ValueError(f"a weight is [out_features, in_features], got {list(weight.shape)}")
        if weight.dtype not in _DTYPES:
            raise TypeError(f"unsupported dtype {weight.dtype}; use float16, bfloat16 or float32")
        _check_gpu("the weight", weight)
        N, K = weight.shape
        if N < 1 or K < 1:
            raise ValueError(f"a weight needs at least one row and column, got [{N}, {K}]")
        w = weight.detach()
        w = w if w.stride(1) == 1 or K == 1 else w.contiguous()
        codes = torch.empty(N, _blocks(K) * BLOCK, dtype=torch.uint8, device=w.device)
        exponents = torch.zeros(_blocks(N), _exponents(K), dtype=torch.uint8, device=w.device)
        _native.e4m3_weight(w, codes, exponents)
        return cls(N, K, codes, exponents)

    @classmethod
    def from_tensors(cls, codes: torch.Tensor, scales: torch.Tensor) -> "E4M3Weight":
        """A weight that is in 8 bits already: codes float8_e4m3fn [out_features,
        in_features] and the scale of each block of 128 x 128, float32 powers of two from
        2^-126 to 2^127 or float8_e8m0fnu.  (Codes with other scales: multiply them out
        and take :meth:`from_dense`.)"""
        if codes.dim() != 2 or codes.dtype != torch.float8_e4m3fn:
            raise TypeError("codes must be float8_e4m3fn [out_features, in_features]")
        N, K = codes.shape
        if tuple(scales.shape) != (_blocks(N), _blocks(K)):
            raise ValueError(f"scales must be [{_blocks(N)}, {_blocks(K)}], got {list(scales.shape)}")
        if scales.device != codes.device:
            raise ValueError("codes and scales must be on the same device")
        if scales.dtype == torch.float8_e8m0fnu:
            e = scales.view(torch.uint8)
            good = (e > 0) & (e < 255)
        elif scales.dtype == torch.float32:
            bits = scales.contiguous().view(torch.int32)
            e = bits >> 23
            good = (bits & 0x7FFFFF == 0) & (e > 0) & (e < 255)
        else:
            raise TypeError(f"scales must be float32 or float8_e8m0fnu, got {scales.dtype}")
        if not bool(good.all()):
            raise ValueError("scales must be powers of two from 2^-126 to 2^127")
        held = torch.zeros(N, _blocks(K) * BLOCK, dtype=torch.uint8, device=codes.device)
        held[:, :K] = codes.view(torch.uint8)
        exponents = torch.zeros(_blocks(N), _exponents(K), dtype=torch.uint8, device=codes.device)
        exponents[:, :_blocks(K)] = e.to(torch.uint8)
        return cls(N, K, held, exponents)

    @property
    def codes(self) -> torch.Tensor:
        return self._codes[:, :self.in_features].view(torch.float8_e4m3fn)

    @property
    def scales(self) -> torch.Tensor:
        e = self._exponents[:, :_blocks(self.in_features)]
        return (e.to(torch.int32) << 23).view(torch.float32)

    @property
    def device(self) -> torch.device:
        return self._codes.device

    def dense(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values, rounded to ``dtype``."""
        s = self.scales.repeat_interleave(BLOCK, 0)[:self.out_features]
        s = s.repeat_interleave(BLOCK, 1)[:, :self.in_features]
        return (self.codes.float() * s).to(dtype)


def linear_e4m3(x: torch.Tensor, weight: E4M3Weight, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x times the weight's transpose (+ bias), both in 8 bits. No backward.

    Each row of x is brought into e4m3 with a power-of-two scale for each 128 columns
    (the smallest with which the largest element fits); products are summed in fp32
    and rounded once.  16-bit results take the 8-bit matrix core, whose sums are off by
    about 1.4e-5 of the result's norm (of the terms' where these cancel); fp32 ones the
    16-bit one, whose sums are fp32's.  A block of x that holds an infinity or NaN makes
    its row's results NaN.

    Args:
        x: [..., in_features] float16, bfloat16 or float32 on the GPU, any strides
            (columns apart, or rows that are not evenly spaced, are copied).
        bias: [out_features] in x's dtype.

    Returns: [..., out_features], contiguous, in x's dtype.
    """
    if not isinstance(weight, E4M3Weight):
        raise TypeError("weight must be an E4M3Weight")
    return _product(x, weight._codes, weight._exponents, weight.out_features, weight.in_features, bias)


@torch.compiler.disable
def _product(x, codes, exponents, N, K, bias):
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
        raise NotImplementedError("linear_e4m3 has no backward; call it under torch.no_grad()")
    op = _native.fast_op("linear_e4m3")
    if op is not None:
        y = op(x, codes, exponents, bias, N, K)
        if y:
            return y[0]
    # what the operator does not take (or nobody does: the checks say why)
    if _native.has_tangent(x, bias):
        raise NotImplementedError("linear_e4m3 has no forward-mode derivatives")
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError(f"x has shape {list(x.shape)}, the weight takes {K} columns")
    if x.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {x.dtype}; use float16, bfloat16 or float32")
    _check_gpu("x", x)
    if x.device != codes.device:
        raise ValueError(f"x is on {x.device} but the weight is on {codes.device}")
    if bias is not None:
        if bias.shape != (N,):
            raise ValueError(f"bias must have shape [{N}], got {list(bias.shape)}")
        if bias.dtype != x.dtype:
            raise TypeError(f"bias must be {x.dtype}, got {bias.dtype}")
        if bias.device != x.device:
            raise ValueError(f"bias is on {bias.device} but x is on {x.device}")
        bias = bias if bias.is_contiguous() else bias.contiguous()
    y = torch.empty(*x.shape[:-1], N, dtype=x.dtype, device=x.device)
    if y.numel():
        rows = x.reshape(-1, K)
        rows = rows if rows.stride(1) == 1 or K == 1 else rows.contiguous()
        _native.linear_e4m3(rows, codes, exponents, bias, y.view(-1, N))
    return y


class E4M3Linear(nn.Module):
    """nn.Linear with its weight in 8 bits (:func:`linear_e4m3`): no gradients. The
    weight's two parts are buffers (``codes``, ``exponents``, as :class:`E4M3Weight`
    stores them), the bias too."""

    def __init__(self, weight: E4M3Weight, bias: Optional[torch.Tensor] = None):
        super().__init__()
        self.out_features, self.in_features = weight.out_features, weight.in_features
        self.register_buffer("codes", weight._codes)
        self.register_buffer("exponents", weight._exponents)
        self.register_buffer("bias", None if bias is None else bias.detach().clone())

    @classmethod
    def from_linear(cls, *linears: nn.Linear) -> "E4M3Linear":
        """Of one linear layer, or of several over the same input, their outputs side by
        side (all with a bias, or none)."""
        weights, biases = [m.weight for m in linears], [m.bias for m in linears]
        if any((b is None) != (biases[0] is None) for b in biases):
            raise ValueError("layers with and without a bias")
        bias = None if biases[0] is None else torch.cat(list(biases))
        return cls(E4M3Weight.from_dense(torch.cat(list(weights))), bias)

    @property
    def weight(self) -> E4M3Weight:
        return E4M3Weight(self.out_features, self.in_features, self.codes, self.exponents)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return _product(x, self.codes, self.exponents, self.out_features, self.in_features, self.bias)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"bias={self.bias is not None}")
