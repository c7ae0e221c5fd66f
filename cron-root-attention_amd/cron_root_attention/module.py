"""nn.Module wrappers (reference module.py:1-247).

``CronRootAttention`` keeps the reference's constructor and forward
(module.py:20-126) and adds keyword arguments: ``hybrid`` (dispatch to
SDPA below the gfx950 crossover, as ``CronRootAttentionHybrid`` does) and
``threshold``; ``rotary`` (a :class:`RotaryTable`) and ``qk_norm`` (a norm of each
head of q and k, with weights of its own), which stand between the projections
and the attention (on the GPU: the plain layer's path for CPU tensors has neither);
``cache`` and ``batch`` of forward, which serve new tokens over a
:class:`PagedKVCache`; and ``to_e4m3``, which brings the projections into 8 bits for
serving.  Grouped kv heads go to the kernel natively
(``kv_groups``) instead of being expanded with ``repeat_interleave``
(module.py:111-113); query head h reads kv head h // kv_groups either way, so
the result is the same.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn
import torch.nn.functional as F

from .core import _layer_op
from .e4m3 import E4M3Linear
from .hybrid import dispatch_backend
from .paged import PagedBatch, PagedKVCache, cron_root_attention_paged
from .rotary import RotaryTable, qk_norm_rotary, rotary_embedding


class CronRootAttention(nn.Module):
    """sqrt(N) sparse attention layer with q/k/v/o projections."""

    def __init__(self, d_model: int, n_heads: int, n_kv_heads: Optional[int] = None,
                 dropout: float = 0.0, bias: bool = False, hybrid: bool = False,
                 threshold: Optional[int] = None, rotary: Optional[RotaryTable] = None,
                 qk_norm: bool = False, norm_eps: float = 1e-6):
        super().__init__()
        self.d_model = d_model
        self.n_heads = n_heads
        self.n_kv_heads = n_kv_heads or n_heads
        self.head_dim = d_model // n_heads
        self.dropout = dropout
        self.hybrid = hybrid
        self.threshold = threshold
        assert d_model % n_heads == 0, "d_model must be divisible by n_heads"
        assert n_heads % self.n_kv_heads == 0, "n_heads must be divisible by n_kv_heads"
        self.kv_groups = n_heads // self.n_kv_heads
        self.drop = nn.Dropout(dropout) if dropout > 0 else nn.Identity()
        self.q_proj = nn.Linear(d_model, d_model, bias=bias)
        self.k_proj = nn.Linear(d_model, self.n_kv_heads * self.head_dim, bias=bias)
        self.v_proj = nn.Linear(d_model, self.n_kv_heads * self.head_dim, bias=bias)
        self.o_proj = nn.Linear(d_model, d_model, bias=bias)
        self.qkv_proj = None  # the joint projection of to_e4m3
        self.rotary = rotary
        self.norm_eps = norm_eps
        self.q_norm = nn.Parameter(torch.ones(self.head_dim)) if qk_norm else None
        self.k_norm = nn.Parameter(torch.ones(self.head_dim)) if qk_norm else None
        self._reset_parameters()

    def __setstate__(self, state):
        super().__setstate__(state)
        if "qkv_proj" not in self._modules:  # a layer pickled before there was one
            self.__dict__.setdefault("qkv_proj", None)

    def _reset_parameters(self):
        for lin in (self.q_proj, self.k_proj, self.v_proj, self.o_proj):
            nn.init.xavier_uniform_(lin.weight)
            if lin.bias is not None:
                nn.init.zeros_(lin.bias)

    def to_e4m3(self) -> "CronRootAttention":
        """Bring the projections into 8 bits (:class:`E4M3Linear`), in place: q_proj,
        k_proj and v_proj become one product ``qkv_proj``, o_proj another. On the GPU;
        the layer has no gradients then."""
        if self.qkv_proj is not None:
            return self
        qkv = E4M3Linear.from_linear(self.q_proj, self.k_proj, self.v_proj)
        o = E4M3Linear.from_linear(self.o_proj)
        for name in ("q_proj", "k_proj", "v_proj", "o_proj"):
            delattr(self, name)
        self.qkv_proj, self.o_proj = qkv, o
        return self

    def _projected(self, x, kv):
        """q, k, v as [B, heads, S, head_dim]."""
        B, S, _ = x.shape
        if self.qkv_proj is None:
            return (p(y).view(B, S, h, self.head_dim).transpose(1, 2)
                    for p, y, h in ((self.q_proj, x, self.n_heads), (self.k_proj, kv, self.n_kv_heads),
                                    (self.v_proj, kv, self.n_kv_heads)))
        heads = (self.n_heads, self.n_kv_heads, self.n_kv_heads)
        y = self.qkv_proj(x).view(B, S, sum(heads), self.head_dim).transpose(1, 2)
        z = y if kv is x else self.qkv_proj(kv).view(B, S, sum(heads), self.head_dim).transpose(1, 2)
        return (y.split(heads, 1)[0], *z.split(heads, 1)[1:])

    def backend_for(self, x: torch.Tensor) -> str:
        """``"cron_root"`` or ``"sdpa"``: what forward(x) runs.  Without
        ``hybrid`` always the sqrt(N) op; with it the crossover of
        :func:`dispatch_backend` for this head dim, B*H and train/eval mode."""
        if not self.hybrid:
            return "cron_root"
        return dispatch_backend(x.shape[1], self.head_dim,
                                self.training and torch.is_grad_enabled(),
                                x.shape[0] * self.n_heads, self.threshold)

    def _table(self, device):
        if self.rotary is not None and self.rotary.device != device:
            self.rotary = self.rotary.to(device)
        return self.rotary

    def _appended(self, q, k, v, positions, cache, batch):
        """q normed and turned as the layer was made to; k, too, and stored with v."""
        args = batch.page_table, batch.seq_lens, batch.cu_seqlens
        if self.rotary is None and self.q_norm is None:
            cache.write(k, v, *args)
            return q
        return cache.append(q, k, v, *args, table=self._table(q.device), positions=positions,
                            norm=self.q_norm is not None, q_weight=self.q_norm, k_weight=self.k_norm,
                            eps=self.norm_eps)

    def _turned(self, q, k, positions):
        """q and k normed and turned, as the layer was made to."""
        self._table(q.device)
        if self.q_norm is not None:
            return qk_norm_rotary(q, k, self.q_norm, self.k_norm, self.rotary, positions,
                                  self.norm_eps)
        if self.rotary is not None:
            return rotary_embedding(q, k, self.rotary, positions)
        return q, k

    def forward(self, x: torch.Tensor, kv: Optional[torch.Tensor] = None,
                positions: Optional[torch.Tensor] = None, cache: Optional[PagedKVCache] = None,
                batch: Optional[PagedBatch] = None) -> torch.Tensor:
        """x [B, S, d_model] -> [B, S, d_model].

        ``positions`` (with ``rotary``): of the tokens, [S] or [B, S]; default 0 ..
        S - 1, or with a cache the tokens' places in their sequences. With ``cache``
        and ``batch`` x holds the new tokens of the batch's sequences, [N, S, d_model]
        or (``cu_seqlens``) packed [1, T, d_model]: their keys and values are stored and
        they attend to their sequences (no gradients)."""
        B, S, _ = x.shape
        if (cache is None) != (batch is None):
            raise ValueError("cache and batch belong together")
        if positions is not None and self.rotary is None:
            raise ValueError("positions without rotary: the layer has nothing to turn by")
        kv = kv if kv is not None else x
        q, k, v = self._projected(x, kv)
        if cache is not None:
            q = self._appended(q, k, v, positions, cache, batch)
            out = cron_root_attention_paged(q, cache, batch.page_table, batch.seq_lens,
                                            batch.cu_seqlens, batch.max_query_len, batch.max_seqlen,
                                            batch.window, batch.relay, prefix=batch.prefix)
        elif self.backend_for(x) == "sdpa":
            q, k = self._turned(q, k, positions)
            out = F.scaled_dot_product_attention(q, k, v, is_causal=True,
                                                 enable_gqa=self.kv_groups > 1)
        else:
            q, k = self._turned(q, k, positions)
            out = _layer_op(self.o_proj)(q, k, v, kv_groups=self.kv_groups)
        out = out.permute(0, 2, 1, 3).reshape(B, S, self.d_model)
        return self.drop(self.o_proj(out))


class CronRootMultiheadAttention(nn.Module):
    """nn.MultiheadAttention-shaped self-attention (reference module.py:129-247).

    As in the reference, attention is always causal sqrt(N) attention:
    ``key_padding_mask``, ``attn_mask`` and ``is_causal`` are ignored, no
    weights are returned, and query, key and value must be the same tensor.
    """

    def __init__(self, embed_dim: int, num_heads: int, dropout: float = 0.0, bias: bool = True,
                 batch_first: bool = True):
        super().__init__()
        self.embed_dim = embed_dim
        self.num_heads = num_heads
        self.head_dim = embed_dim // num_heads
        self.dropout = dropout
        self.batch_first = batch_first
        assert embed_dim % num_heads == 0, "embed_dim must be divisible by num_heads"
        self.in_proj_weight = nn.Parameter(torch.empty(3 * embed_dim, embed_dim))
        if bias:
            self.in_proj_bias = nn.Parameter(torch.empty(3 * embed_dim))
        else:
            self.register_parameter("in_proj_bias", None)
        self.out_proj = nn.Linear(embed_dim, embed_dim, bias=bias)
        self.drop = nn.Dropout(dropout) if dropout > 0 else nn.Identity()
        self._reset_parameters()

    def _reset_parameters(self):
        nn.init.xavier_uniform_(self.in_proj_weight)
        if self.in_proj_bias is not None:
            nn.init.zeros_(self.in_proj_bias)
        nn.init.xavier_uniform_(self.out_proj.weight)
        if self.out_proj.bias is not None:
            nn.init.zeros_(self.out_proj.bias)

    def forward(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                key_padding_mask: Optional[torch.Tensor] = None, need_weights: bool = False,
                attn_mask: Optional[torch.Tensor] = None, average_attn_weights: bool = True,
                is_causal: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        # self-attention only (reference module.py:223); checked before the
        # batch_first transpose, which makes three distinct views of one tensor
        assert query is key and key is value, "Cross-attention not yet supported"
        if not self.batch_first:
            query = query.transpose(0, 1)
        B, S, E = query.shape
        qkv = F.linear(query, self.in_proj_weight, self.in_proj_bias)
        qkv = qkv.view(B, S, 3, self.num_heads, self.head_dim).permute(2, 0, 3, 1, 4)
        out = _layer_op(self.out_proj)(*qkv.unbind(0))
        out = out.permute(0, 2, 1, 3).reshape(B, S, E)
        out = self.drop(self.out_proj(out))
        if not self.batch_first:
            out = out.transpose(0, 1)
        return out, None
