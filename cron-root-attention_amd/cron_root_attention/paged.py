"""Serving: a paged key/value cache and the sqrt(N) attention of new tokens over it.

The reference attends whole sequences only.  Here the keys and values of many
sequences lie in the pages of one :class:`PagedKVCache` (per layer), in their
own type or in 8 bits with a scale for each row and head, and
:func:`cron_root_attention_paged` attends the new tokens of every sequence, one
or thousands each, to what the pattern of ``cron_root_attention`` gives them.

Lengths, page tables and token offsets are device tensors that the kernels read:
nothing synchronises with the host, and a call captured in a graph serves
whatever they hold when it is replayed.  The pattern depends on a sequence's
length through its window (ceil(sqrt(n))) and the relay switch (n > 2048): with
the defaults a step's rows are the last rows of ``cron_root_attention`` over the
sequence of the present length; a program that wants all its steps to agree with
one pass over the whole sequence passes the same ``window`` and ``relay`` to all of
them.  ``window`` at least the length is plain causal attention.  Relay rows count as
they are (there is no ``relay_log_scale`` here).
"""
from __future__ import annotations

import dataclasses
import math
from typing import Optional, Tuple

import torch
import torch.nn.functional as F

from . import _native

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
_STORES = {torch.float8_e4m3fn: _native.STORE_E4M3, torch.int8: _native.STORE_INT8}


def _width(head_dim: int) -> int:
    return (head_dim + 15) // 16 * 16


class PagedKVCache:
    """Pages of keys and values of one layer.

    ``k``, ``v``: [num_pages, n_kv_heads, page_size, width], width the head dim
    rounded up to 16 (columns behind the head dim are zero), of ``dtype`` or, with
    ``storage`` torch.float8_e4m3fn or torch.int8, 8-bit codes with fp32 scales
    ``k_scale``, ``v_scale`` [num_pages, n_kv_heads, page_size] (the value is code *
    scale; a row that held an infinity or NaN has scale NaN). ``k_norm`` of the same
    shape holds each key's sum of squares, by which relay rows are chosen.
    ``page_size``: a power of two from 16 to 1024. Which page belongs to which
    sequence is the caller's: see the ``page_table`` of :meth:`write`.
    """

    def __init__(self, num_pages: int, n_kv_heads: int, head_dim: int, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, storage: Optional[torch.dtype] = None,
                 device=None):
        if not 1 <= head_dim <= 256:
            raise NotImplementedError(f"head dim {head_dim} outside 1..256 is not built")
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        storage = dtype if storage is None else storage
        shape = (num_pages, n_kv_heads, page_size)
        k, v = (torch.zeros(*shape, _width(head_dim), dtype=storage, device=device) for _ in "kv")
        norm = torch.zeros(shape, dtype=torch.float32, device=device)
        scales = [None, None]
        if storage != dtype:
            scales = [torch.zeros(shape, dtype=torch.float32, device=device) for _ in "kv"]
        self._set(k, v, norm, *scales, dtype, head_dim)

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, k_norm: torch.Tensor,
                     k_scale: Optional[torch.Tensor] = None,
                     v_scale: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None,
                     head_dim: Optional[int] = None) -> "PagedKVCache":
        """A cache over the caller's own contiguous tensors (shapes as above; ``dtype``
        of the values where k and v hold 8-bit codes)."""
        self = object.__new__(cls)
        self._set(k, v, k_norm, k_scale, v_scale, k.dtype if dtype is None else dtype,
                  k.shape[-1] if head_dim is None else head_dim)
        return self

    def _set(self, k, v, k_norm, k_scale, v_scale, dtype, head_dim):
        if dtype not in _DTYPES:
            raise TypeError(f"unsupported dtype {dtype}; use float16, bfloat16 or float32")
        if k.dtype == dtype:
            store = _native.STORE_SAME
        elif k.dtype in _STORES:
            store = _STORES[k.dtype]
        else:
            raise TypeError(f"a cache of {dtype} cannot be stored as {k.dtype}; use its own dtype, "
                            "float8_e4m3fn or int8")
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v must be [num_pages, n_kv_heads, page_size, width], alike")
        P = k.shape[2]
        if P < 16 or P > 1024 or P & (P - 1):
            raise ValueError(f"page size must be a power of two from 16 to 1024, got {P}")
        if k.shape[0] < 1 or k.shape[1] < 1:
            raise ValueError("a cache needs at least one page and one head")
        if k.shape[0] * k.shape[1] * P >= 1 << 31:
            raise ValueError("the cache has 2^31 rows or more")
        if not 1 <= head_dim <= 256:
            raise NotImplementedError(f"head dim {head_dim} outside 1..256 is not built")
        if k.shape[3] != _width(head_dim):
            raise ValueError(f"rows of head dim {head_dim} take a width of {_width(head_dim)}, "
                             f"got {k.shape[3]}")
        rows = [k_norm] + ([] if store == _native.STORE_SAME else [k_scale, v_scale])
        for t in rows:
            if not isinstance(t, torch.Tensor) or t.shape != k.shape[:3] or t.dtype != torch.float32:
                raise ValueError("k_norm (and the scales of 8-bit storage) must be float32 "
                                 "[num_pages, n_kv_heads, page_size]")
        if store == _native.STORE_SAME and (k_scale is not None or v_scale is not None):
            raise ValueError("scales are for 8-bit storage")
        for t in [k, v] + rows:
            if t.device.type != "cuda" or t.device != k.device:
                raise RuntimeError(f"a paged cache lives on one ROCm GPU (got {t.device})")
            if not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError("the cache's tensors must be contiguous and 16-byte aligned")
            if t.requires_grad:
                raise ValueError("a cache has no gradients")
        self.k, self.v, self.k_norm, self.k_scale, self.v_scale = k, v, k_norm, k_scale, v_scale
        self.dtype, self.head_dim = dtype, int(head_dim)
        self._struct = _native.CraCache(
            k.data_ptr(), v.data_ptr(), k_norm.data_ptr(), _native._ptr(k_scale),
            _native._ptr(v_scale), k.shape[0], k.shape[1], P, k.shape[3],
            _native.dtype_code(dtype), store)

    @property
    def num_pages(self) -> int:
        return self.k.shape[0]

    @property
    def n_kv_heads(self) -> int:
        return self.k.shape[1]

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    @property
    def device(self) -> torch.device:
        return self.k.device

    @torch.compiler.disable
    def write(self, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
              seq_lens: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None) -> None:
        """Store the rows of new tokens, the last ones of their sequences.

        Args:
            k, v: [N, n_kv_heads, M, D], M new tokens of each of N sequences; or
                with ``cu_seqlens`` packed [1, n_kv_heads, T, D].
            page_table: int32 [N, pages]: row r of sequence b lies in page
                page_table[b, r // page_size]. Nothing is written to a page id
                outside the cache, nor behind the last page of a sequence's row.
            seq_lens: int32 [N], lengths with the new tokens.
            cu_seqlens: int32 [N + 1]: the new tokens of sequence b are
                cu_seqlens[b] .. cu_seqlens[b + 1] - 1 of T; tokens outside every
                sequence (padding) are passed over.

        All int32 tensors are on the GPU. No page may be written for two sequences
        in one call.
        """
        if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad):
            raise NotImplementedError("the cache has no backward; write under torch.no_grad()")
        op = _native.fast_op("cache_write")
        if op is not None and k.dtype == self.dtype and op(
                k, v, self.k, self.v, self.k_norm, self.k_scale, self.v_scale, page_table, seq_lens,
                cu_seqlens, self.head_dim):
            return
        # what the operator does not take (or nobody does: the checks say why)
        if _native.has_tangent(k, v):
            raise NotImplementedError("the cache has no forward-mode derivatives")
        batch = _batch(self, k, self.n_kv_heads, page_table, seq_lens, cu_seqlens, "k")
        if v.shape != k.shape:
            raise ValueError(f"v shape {tuple(v.shape)} does not match k {tuple(k.shape)}")
        if v.dtype != k.dtype or v.device != k.device:
            raise TypeError("k and v must have one dtype and device")
        if batch is None:
            return
        _native.cache_write(self._struct, batch, _ready(k), _ready(v))

    @torch.compiler.disable
    def read(self, page_table: torch.Tensor, seq_lens: torch.Tensor,
             length: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Rows 0 .. length - 1 of every sequence as contiguous k, v
        [N, n_kv_heads, length, D] in the cache's dtype (``length`` defaults to what
        a row of the table holds); rows behind a sequence's end are zeros, rows of
        a page outside the cache NaN."""
        _check_table(self, page_table, seq_lens)
        N = page_table.shape[0]
        length = page_table.shape[1] * self.page_size if length is None else int(length)
        if length < 0:
            raise ValueError(f"length must be >= 0, got {length}")
        k, v = (torch.empty(N, self.n_kv_heads, length, self.head_dim, dtype=self.dtype,
                            device=self.device) for _ in "kv")
        if k.numel():
            if page_table.shape[1] == 0:
                return k.zero_(), v.zero_()
            batch = _native.CraBatch(page_table.data_ptr(), page_table.stride(0),
                                     seq_lens.data_ptr(), None, N, page_table.shape[1], 0, 1)
            _native.cache_read(self._struct, batch, length, k, v)
        return k, v


def _check_table(cache, page_table, seq_lens):
    for name, t in (("page_table", page_table), ("seq_lens", seq_lens)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
            raise TypeError(f"{name} must be an int32 tensor")
        if t.device != cache.device:
            raise ValueError(f"{name} is on {t.device} but the cache is on {cache.device}")
    if page_table.dim() != 2 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError("page_table must be [sequences, pages] with contiguous rows")
    if seq_lens.shape != page_table.shape[:1] or not seq_lens.is_contiguous():
        raise ValueError("seq_lens must be contiguous [sequences]")


def _batch(cache, x, heads, page_table, seq_lens, cu_seqlens, name):
    """The batch of new tokens x [N or 1, heads, M or T, D]; None when it is empty."""
    _check_table(cache, page_table, seq_lens)
    N = page_table.shape[0]
    if x.dim() != 4:
        raise ValueError(f"{name} must be [sequences, heads, tokens, D]")
    if x.dtype != cache.dtype:
        raise TypeError(f"{name} is {x.dtype} but the cache holds {cache.dtype}")
    if x.device != cache.device:
        raise ValueError(f"{name} is on {x.device} but the cache is on {cache.device}")
    B, H, M, D = x.shape
    if heads is not None and H != heads:
        raise ValueError(f"{name} has {H} heads, the cache {heads}")
    if D != cache.head_dim:
        raise ValueError(f"{name} has head dim {D}, the cache {cache.head_dim}")
    if max(*x.shape, *page_table.shape) > 2**31 - 1:
        raise ValueError("a dimension of 2^31 or more")
    cu = None
    if cu_seqlens is not None:
        if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.dtype != torch.int32:
            raise TypeError("cu_seqlens must be an int32 tensor")
        if cu_seqlens.device != cache.device:
            raise ValueError(f"cu_seqlens is on {cu_seqlens.device} but the cache is on {cache.device}")
        if cu_seqlens.shape != (N + 1,) or not cu_seqlens.is_contiguous():
            raise ValueError(f"cu_seqlens must be contiguous [{N + 1}] for {N} sequences")
        if B != 1:
            raise ValueError(f"with cu_seqlens {name} must be packed [1, heads, tokens, D]")
        cu = cu_seqlens.data_ptr()
    elif B != N:
        raise ValueError(f"{name} has {B} sequences, the page table {N}")
    if N == 0 or M == 0:
        return None
    if page_table.shape[1] == 0:  # no pages: as a table of pages outside the cache
        page_table = page_table.new_full((N, 1), -1)
    batch = _native.CraBatch(page_table.data_ptr(), page_table.stride(0), seq_lens.data_ptr(), cu, N,
                             page_table.shape[1], M if cu is not None else 0, 0 if cu is not None else M)
    batch.table = page_table  # lives as long
    return batch


def _aligned(t: torch.Tensor) -> bool:
    vec = 16 // t.element_size()
    (sb, sh, ss, sd), shape = t.stride(), t.shape
    return (sd == 1 and t.data_ptr() % 16 == 0 and (shape[0] == 1 or sb % vec == 0)
            and (shape[1] == 1 or sh % vec == 0) and (shape[2] == 1 or ss % vec == 0))


def _ready(t: torch.Tensor) -> torch.Tensor:
    """Rows of a multiple of 8 elements, 16-byte aligned (a copy where they are not)."""
    if t.shape[3] % 8:
        t = F.pad(t, (0, -t.shape[3] % 8))
    return t if _aligned(t) else t.clone(memory_format=torch.contiguous_format)


@torch.compiler.disable
def cron_root_attention_paged(q: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor,
                              seq_lens: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None,
                              max_query_len: Optional[int] = None,
                              max_seqlen: Optional[int] = None, window: Optional[int] = None,
                              relay: Optional[bool] = None, relay_top_k: int = 2,
                              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the new tokens of every sequence over the cache, which holds
    their own rows already (:meth:`PagedKVCache.write` comes first). No backward.

    Args:
        q: [N, H_q, M, D], M new tokens of each of N sequences, or with
            ``cu_seqlens`` packed [1, H_q, T, D]; H_q a multiple of the cache's
            heads (query head h reads kv head h // (H_q / heads)).
        page_table, seq_lens, cu_seqlens: as in :meth:`PagedKVCache.write`.
        max_query_len: bound on a sequence's new tokens (with ``cu_seqlens``;
            default T). Where it times the query heads of a kv head is at most 16 the
            kernels for chunks are not launched; a sequence with more new tokens may
            give NaN.
        max_seqlen: bound on ``seq_lens`` (default: what a row of the table holds).
            A tighter bound makes for fewer, smaller pieces of work. A sequence
            longer than it gives NaN.
        window: None: ceil(sqrt(length)) of each sequence; else the window (and block
            size) of all, within their lengths.
        relay: None: relay rows for sequences of more than 2048 tokens; else on or off.
        relay_top_k: relay rows a block (1..4).
        out: where the result goes, shaped as q; rows of tokens outside every
            sequence are left as they were.

    Returns: like q (laid out as q). Rows of tokens outside every sequence are zeros; so
    is a query that sees no row (more new tokens than the sequence's length). A
    query that meets a page outside the cache gives NaN, and so may others of its sequence.
    """
    if torch.is_grad_enabled() and q.requires_grad:
        raise NotImplementedError("cron_root_attention_paged has no backward; call it under "
                                  "torch.no_grad() (training: cron_root_attention)")
    op = _native.fast_op("paged_attention")
    if (op is not None and out is None and q.dtype == cache.dtype and window != 0
            and max_query_len != 0 and max_seqlen != 0):
        y = op(q, cache.k, cache.v, cache.k_norm, cache.k_scale, cache.v_scale, page_table, seq_lens,
               cu_seqlens, cache.head_dim, max_query_len or 0, max_seqlen or 0, window or 0,
               -1 if relay is None else int(bool(relay)), relay_top_k)
        if y:
            return y[0]
    if _native.has_tangent(q):
        raise NotImplementedError("cron_root_attention_paged has no forward-mode derivatives")
    batch = _batch(cache, q, None, page_table, seq_lens, cu_seqlens, "q")
    Hq, D = q.shape[1], q.shape[3]
    if Hq < 1 or Hq % cache.n_kv_heads:
        raise ValueError(f"H_q={Hq} must be a multiple of the cache's {cache.n_kv_heads} heads")
    if window is not None and window < 1:
        raise ValueError(f"window must be >= 1, got {window}")
    if relay is not False and not 1 <= relay_top_k <= 4:
        raise ValueError(f"relay_top_k={relay_top_k} outside [1, 4]")
    held = max(1, page_table.shape[1]) * cache.page_size
    for name, x in (("max_query_len", max_query_len), ("max_seqlen", max_seqlen)):
        if x is not None and x < 1:
            raise ValueError(f"{name} must be >= 1, got {x}")
    if out is None:
        # rows outside every sequence are zeros in a fresh output
        o = torch.zeros_like(q) if batch is None else torch.empty_like(q)
    else:
        if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
            raise ValueError("out must have the shape, dtype and device of q")
        o = out
    if batch is None:
        return o
    plan = _native.CraPagedPlan(
        Hq, D + -D % 8, 0 if window is None else min(int(window), 2**31 - 1),
        -1 if relay is None else int(bool(relay)), int(relay_top_k),
        min(q.shape[2], max_query_len or q.shape[2]), min(held, max_seqlen or held, 2**31 - 1),
        int(out is None), 1.0 / math.sqrt(D))
    qr = _ready(q)
    if D % 8 == 0 and _aligned(o):
        _native.forward_paged(cache._struct, batch, plan, qr, o)
    else:  # through a buffer that the kernels can store to; o's other rows stay
        tmp = _ready(o) if cu_seqlens is not None else torch.empty_like(qr)
        _native.forward_paged(cache._struct, batch, plan, qr, tmp)
        o.copy_(tmp[..., :D])
    return o


@dataclasses.dataclass
class PagedBatch:
    """The sequences of one step of a layer over its cache: the arguments of
    :func:`cron_root_attention_paged` that are not the layer's own (two relay rows a
    block, as in its training path). A packed step should bound its new tokens
    (``max_query_len``, 1 for decoding): without a bound the kernels for chunks are
    launched too."""

    page_table: torch.Tensor
    seq_lens: torch.Tensor
    cu_seqlens: Optional[torch.Tensor] = None
    max_query_len: Optional[int] = None
    max_seqlen: Optional[int] = None
    window: Optional[int] = None
    relay: Optional[bool] = None

    def positions(self, tokens: int) -> torch.Tensor:
        """Position of each new token, int32 [N, tokens] or (packed) [1, tokens];
        tokens outside every sequence get 0."""
        t = torch.arange(tokens, dtype=torch.int32, device=self.seq_lens.device)
        if self.cu_seqlens is None:
            return (self.seq_lens - tokens)[:, None] + t
        cu = self.cu_seqlens
        b = (torch.searchsorted(cu, t, right=True) - 1).clamp_(0, self.seq_lens.shape[0] - 1)
        pos = self.seq_lens[b] - cu[b + 1] + t
        return torch.where((t >= cu[0]) & (t < cu[-1]), pos, 0).to(torch.int32)[None]
