"""Oracle of the paged cache and of the attention over it, in 64 bits on the CPU."""
import math

import torch

STORES = {"same": None, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def quantise(x, storage):
    """Codes, scales and values (fp64) of rows x as the cache holds them."""
    if storage is None or storage == x.dtype:
        return x, None, x.double()
    f = x.float()
    most = f.abs().amax(-1)
    if storage == torch.float8_e4m3fn:
        part, power = torch.frexp(most.double() / 448.0)
        scale = torch.ldexp(torch.ones_like(part), (power - (part == 0.5).int()).clamp_min(-126)).float()
    else:
        scale = most * torch.tensor(1 / 127, dtype=torch.float32)
    scale = torch.where(most > 0, scale, torch.zeros_like(scale)).clamp_min(torch.finfo(torch.float32).tiny)
    scale = torch.where(most.isfinite(), scale, torch.full_like(scale, math.nan))
    y = f / scale[..., None]
    y = torch.where(y.isfinite(), y, torch.zeros_like(y))
    codes = y.to(storage) if storage == torch.float8_e4m3fn else y.round().to(torch.int8)
    return codes, scale, codes.double() * scale.double()[..., None]


def norm_sq(k):
    """Sum of squares in the library's order: 8 elements left to right by fused multiply-adds, then a butterfly."""
    x = k.float()
    if x.shape[-1] % 8:
        x = torch.nn.functional.pad(x, (0, -x.shape[-1] % 8))
    x = x.unflatten(-1, (-1, 8))
    s = torch.zeros(x.shape[:-1])
    for i in range(8):
        s = (s.double() + x[..., i].double() ** 2).float()
    lanes = 1
    while lanes < s.shape[-1]:
        lanes *= 2
    s = torch.nn.functional.pad(s, (0, lanes - s.shape[-1]))
    while s.shape[-1] > 1:
        h = s.shape[-1] // 2
        s = s[..., :h] + s[..., h:]
    return s[..., 0]


def plan(n, window=None, relay=None):
    W = min(n, window) if window else math.isqrt(n - 1) + 1
    return W, (n > 2048 if relay is None else relay)


def counts(n, i, W, relay, top_k, norm):
    """How often each of n rows is in the set of query i ([n] int64). norm: [n] squares."""
    c = torch.zeros(n, dtype=torch.int64)
    ls = max(0, i - W + 1)
    c[ls:i + 1] += 1
    for r in range(-(-ls // W)):
        c[r * W] += 1
    if relay:
        for r in range(ls // W):
            blk = norm[r * W:(r + 1) * W]
            key = torch.where(blk.isnan(), torch.full_like(blk, -1.0), blk)
            order = torch.sort(key, descending=True, stable=True).indices.tolist()
            order = [j for j in order if key[j] >= 0]
            for t in range(top_k):
                c[r * W + (order[t] if t < len(order) else 0)] += 1
    return c


def attend(q, k, v, norm, n, m, window=None, relay=None, top_k=2, scale=None):
    """Last m queries of one kv head's group: q [g, m, D], k, v [n, D] fp64, norm [n].
    Returns o [g, m, D], and the largest sum of |p v| weights (for tolerances)."""
    g, _, D = q.shape
    o = torch.zeros(g, m, D, dtype=torch.float64)
    mag = torch.zeros(g, m, D, dtype=torch.float64)
    W, rel = plan(n, window, relay) if n > 0 else (1, False)
    scale = scale or 1 / math.sqrt(D)
    for t in range(m):
        i = n - m + t
        if i < 0:
            continue
        c = counts(n, i, W, rel, top_k, norm)
        at = c.nonzero()[:, 0]
        w = c[at].double()
        s = q[:, t].double() @ k[at].t() * scale
        p = (s - s.amax(-1, keepdim=True)).exp() * w
        p = p / p.sum(-1, keepdim=True)
        o[:, t] = p @ v[at]
        mag[:, t] = p @ v[at].abs()
    return o, mag
