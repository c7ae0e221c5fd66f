"""Performance cases of the operators around the sqrt(N) attention on one GPU:
rotary positions, head norms with the rotation, the paged key/value cache and
the attention of new tokens over it.

A case is a dict of plain values; ``op`` names the operator:

    "rotary", "norm_rotary"   q [B, Hq, S, D] and k [B, Hkv, S, D]; train: the
          step's gradients too; layout "bhsd" contiguous, "bshd" views of
          [B, S, H, D] buffers, "fused" slices of one [B, S, Hq + 2 Hkv, D]
          projection; rot: leading elements of a head that turn; pairs are
          (2i, 2i+1) if interleaved, else (i, i + rot/2); scaling of the
          frequencies; start: positions count from here (random if < 0)
    "write", "write_read"   the last `new` tokens of every sequence are stored
          in a cache that holds sequences of `lens` tokens in pages of `page`
          rows, as `store` ("same" type, "e4m3" or "int8" with a scale for
          each row and head, a power of two for e4m3); write_read also reads all sequences back
    "paged"   attention of the last `new` tokens of every sequence over such a
          cache; window 0: the sqrt(N) rule for the present length, > 0: this
          window for every length (at least the length: dense causal attention)

``lens`` and ``new`` are comma-separated numbers, one for each sequence.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4}
_RELAY_FROM = 2048  # sequences longer than this have relay rows
_TOP_K = 2
_EPS = 1e-6


_package = None


def _cra():
    global _package
    if _package is None:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cron-root-attention_amd")
        if root not in sys.path:
            sys.path.insert(0, root)
        import cron_root_attention
        _package = cron_root_attention
    return _package


def _turn(name, op, train, B, Hq, Hkv, S, D, dtype, layout="bhsd", rot=0, interleaved=False, scaling="none", start=0):
    c = dict(op=op, train=train, B=B, Hq=Hq, Hkv=Hkv, S=S, D=D, dtype=dtype, layout=layout, rot=rot or D,
             interleaved=interleaved, scaling=scaling, start=start)
    return dict(c, name=name) if name else c


def _cached(name, op, Hq, Hkv, D, dtype, store, page, lens, new, window=0):
    c = dict(op=op, Hq=Hq, Hkv=Hkv, D=D, dtype=dtype, store=store, page=page, lens=",".join(map(str, lens)),
             new=",".join(map(str, new)), window=window)
    return dict(c, name=name) if name else c


# Lengths of requests in one serving batch: a few long, most of them short.
_SERVED = (32768, 30001, 20480, 17777, 16384, 12345, 9001, 8192, 8191, 6000, 5000, 4097, 4096, 4095, 3500, 3333,
           2900, 2500, 2222, 2049, 2048, 2047, 1800, 1600, 1500, 1400, 1300, 1200, 1100, 1025, 1024, 1023,
           1000, 900, 850, 800, 750, 700, 640, 600, 555, 512, 511, 480, 444, 400, 366, 333,
           300, 280, 257, 256, 255, 222, 200, 180, 150, 129, 128, 100, 64, 33, 17, 1)
_LONG = (131072, 131071, 120000, 100000, 90001, 77777, 65536, 65535, 50000, 40000, 30000, 20001, 10000, 5000, 2049, 700)
# Documents read in one pass: long, short, odd, one token.
_DOCS = (9001, 4096, 3333, 2049, 2048, 1500, 1023, 1000, 640, 511, 300, 257, 129, 64, 17, 1)


def listed():
    return [
        # positions of one new token of each of 64 requests: a call of launches and host time
        _turn("rotary_token", "rotary", False, 64, 32, 8, 1, 128, "bf16", layout="fused", start=-1),
        # training in full precision, half of each head turned, neighbouring pairs
        _turn("rotary_train_8k", "rotary", True, 1, 12, 12, 8191, 64, "f32", layout="bshd", rot=32, interleaved=True),
        # a short prompt of a small model
        _turn("norm_rotary_1k", "norm_rotary", False, 1, 12, 12, 1000, 64, "f16", layout="bshd"),
        # long-context training: grouped heads out of one projection, stretched positions
        _turn("norm_rotary_train_32k", "norm_rotary", True, 1, 16, 4, 32768, 128, "bf16", layout="fused", scaling="yarn"),
        # one new token of each of 64 requests into the cache
        _cached("write_token", "write", 32, 8, 128, "f16", "same", 16, [min(n, 2048) for n in _SERVED],
                [1] * len(_SERVED)),
        # prompts of many lengths into an 8-bit cache, and out again for another worker
        _cached("write_read_26k_e4m3", "write_read", 16, 4, 128, "bf16", "e4m3", 64, _DOCS, _DOCS),
        # the tail of one long prompt into an integer cache, the whole read back
        _cached("write_read_64k_int8", "write_read", 16, 16, 128, "f16", "int8", 128, [65536], [32768]),
        # one token of one request at the benchmark's context length
        _cached("decode_1_128k", "paged", 16, 16, 128, "f16", "same", 64, [131072], [1]),
        # a serving step of 64 requests, grouped heads
        _cached("decode_64", "paged", 32, 8, 128, "bf16", "same", 16, _SERVED, [1] * len(_SERVED)),
        # a serving step of long requests over an 8-bit cache
        _cached("decode_16_long_e4m3", "paged", 32, 8, 128, "bf16", "e4m3", 64, _LONG, [1] * len(_LONG)),
        # prefill of a long prompt in chunks: the last chunk of 8K tokens
        _cached("chunk_8k_128k", "paged", 16, 16, 128, "f16", "same", 64, [131072], [8192]),
        # a mixed step under dense causal attention: two prompts in chunks, the others a token or a few drafted ones
        _cached("mixed_dense_int8", "paged", 16, 4, 128, "bf16", "int8", 32,
                (16000, 8191, 20000, 12001, 9000, 5000, 4096, 3001, 2000, 1500, 1000, 700, 500, 100, 9, 1),
                (1000, 513, 1, 1, 1, 4, 1, 1, 5, 1, 1, 1, 1, 1, 9, 1), window=1 << 20),
    ]


# ---------------------------------------------------------------------------
# sizes
# ---------------------------------------------------------------------------
def _ints(text):
    return [int(x) for x in text.split(",")]


def _rule(n, window):
    """(window, relay) of a sequence of n tokens."""
    W = min(n, window) if window else math.isqrt(n - 1) + 1
    return W, n > _RELAY_FROM


def _prefixes(n, m, window):
    """Over the last m queries of n tokens: (query, key) pairs of one head, distinct rows read, rows whose norm is read."""
    W, relay = _rule(n, window)
    i = torch.arange(n - m, n, dtype=torch.int64)
    ls = (i - W + 1).clamp_min(0)
    strided, blocks = (ls + W - 1) // W, (ls // W) * int(relay)
    pairs = int(((i + 1).clamp_max(W) + strided + _TOP_K * blocks).sum())
    rows = n - int(ls[0]) + int(strided[-1]) + _TOP_K * int(blocks[-1])
    return pairs, min(n, rows), int(blocks[-1]) * W


def work(case):
    e, D, Hq, Hkv = _BYTES[case["dtype"]], case["D"], case["Hq"], case["Hkv"]
    if case["op"] in ("rotary", "norm_rotary"):
        tokens = case["B"] * case["S"]
        x = tokens * (Hq + Hkv) * D * e
        table = tokens * case["rot"] * 4
        norm = case["op"] == "norm_rotary"
        n = tokens * (Hq + Hkv)
        flops = n * (3 * case["rot"] + (4 * D if norm else 0))
        if not case["train"]:
            return {"bytes": 2 * x + table, "flops": flops}
        # a step: forward, then dy in and dx out (the norm's backward reads x again)
        return {"bytes": (5 if norm else 4) * x + table, "flops": 2 * flops + (n * 6 * D if norm else 0)}
    lens, new = _ints(case["lens"]), _ints(case["new"])
    row = D * (e if case["store"] == "same" else 1) + (0 if case["store"] == "same" else 4)
    if case["op"] != "paged":
        T, L = sum(new), sum(lens)
        b = 2 * T * Hkv * (D * e + row) + 4 * T * Hkv
        if case["op"] == "write_read":
            b += 2 * L * Hkv * (row + D * e)
        return {"bytes": b, "flops": 4 * T * Hkv * D + (2 * L * Hkv * D if case["op"] == "write_read" else 0)}
    pairs = rows = norms = 0
    for n, m in zip(lens, new):
        p, r, w = _prefixes(n, m, case["window"])
        pairs, rows, norms = pairs + p, rows + r, norms + w
    return {"bytes": 2 * sum(new) * Hq * D * e + Hkv * (2 * rows * row + 4 * norms), "flops": 4 * D * Hq * pairs}


_LARGEST = {}


def _fits(case):
    """Costs no more than the largest listed case of its kind: fp32 products weigh more, and the cache has to be made."""
    def cost(c):
        w = work(c)
        held = sum(_ints(c["lens"])) * c["Hkv"] * c["D"] * _BYTES[c["dtype"]] if "lens" in c else 0
        return w["flops"] * (8 if c["dtype"] == "f32" else 1), w["bytes"], held
    kind = "turn" if "B" in case else case["op"] == "paged"
    if kind not in _LARGEST:
        costs = [cost(c) for c in listed() if ("turn" if "B" in c else c["op"] == "paged") == kind]
        _LARGEST[kind] = [max(x) for x in zip(*costs)]
    return all(a <= b for a, b in zip(cost(case), _LARGEST[kind]))


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "norm_rotary", "norm_rotary", "write", "write_read", "paged", "paged", "paged", "paged"])
    D = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 256])
    dtype = rng.choice(["f16", "f16", "bf16", "bf16", "bf16", "f32"])
    Hkv = rng.choice([1, 2, 3, 4, 6, 8, 8, 12, 16])
    Hq = Hkv * rng.choice([g for g in (1, 1, 2, 4, 5, 8) if g * Hkv <= 64])
    if op in ("rotary", "norm_rotary"):
        rot = rng.choice([D, D, D, D // 2, D // 4])
        c = dict(layout=rng.choice(["bhsd", "bshd", "fused"]), rot=rot, interleaved=rng.random() < 0.4,
                 scaling=rng.choice(["none", "linear", "ntk", "yarn"]), start=rng.choice([0, -1, 1000, 100000]))
        B, S, train = rng.choice([1, 1, 2, 3, 16]), _log_int(rng, 1, 65536), rng.random() < 0.6
        while True:
            case = _turn(None, op, train, B, Hq, Hkv, S, D, dtype, **c)
            if _fits(case):
                return case
            S = max(1, int(S * 0.6))
            B = B if S > 1 else 1
    store = rng.choice(["same", "same", "e4m3", "int8"])
    page = rng.choice([16, 16, 32, 64, 128, 256])
    N = _log_int(rng, 1, 96)
    most = _log_int(rng, 64, 131072)
    lens = [_log_int(rng, 1, most) for _ in range(N)]
    style = rng.choice(["token", "token", "few", "chunk", "mixed"])
    new = [min(n, {"token": 1, "few": rng.randint(1, 8), "chunk": _log_int(rng, 1, 8192)}[
        style if style != "mixed" else rng.choice(["token", "token", "few", "chunk"])]) for n in lens]
    window = rng.choice([0, 0, 0, 0, 1 << 20, _log_int(rng, 1, 4096)])
    while True:
        case = _cached(None, op, Hq, Hkv, D, dtype, store, page, lens, new, window if op == "paged" else 0)
        if _fits(case):
            return case
        if len(lens) > 1:
            lens.pop(), new.pop()
        else:
            lens[0] = max(1, lens[0] // 2)
            new[0] = min(new[0], lens[0])


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


_SCALING = {"none": None, "linear": dict(type="linear", factor=4.0), "ntk": dict(type="ntk", factor=4.0),
            "yarn": dict(type="yarn", factor=8.0, original_positions=16384)}
_BASE = 10000.0


def _frequencies(rot, scaling):
    """Angle per position of each pair (64 bits), and the multiplier of cos and sin."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    s = _SCALING[scaling] or {"type": "none"}
    base = _BASE * (s["factor"] ** (rot / (rot - 2)) if s["type"] == "ntk" and rot > 2 else 1.0)
    f = base ** (-2 * i / rot)
    if s["type"] == "linear":
        f = f / s["factor"]
    if s["type"] != "yarn":
        return f, 1.0

    def pair_of(turns):  # the pair that makes this many turns over the original positions
        return rot * math.log(s["original_positions"] / (turns * 2 * math.pi)) / (2 * math.log(_BASE))
    lo, hi = max(0, math.floor(pair_of(32.0))), min(rot - 1, math.ceil(pair_of(1.0)))
    ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
    return f * (1 - ramp) + f / s["factor"] * ramp, 0.1 * math.log(s["factor"]) + 1


def _positions(case, gen):
    B, S = case["B"], case["S"]
    if case["start"] >= 0:
        return torch.arange(case["start"], case["start"] + S, device="cuda", dtype=torch.int32)
    return torch.randint(0, 131072, (B, S), generator=gen, device="cuda", dtype=torch.int32)


def _turn_inputs(case, seed):
    gen, dt = _gen(seed), _DTYPES[case["dtype"]]
    B, Hq, Hkv, S, D = (case[x] for x in ("B", "Hq", "Hkv", "S", "D"))

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    t = {"pos": _positions(case, gen)}
    if case["layout"] == "fused":
        x = (normal(B, S, Hq + 2 * Hkv, D) * 1.5).to(dt)
        t["q"], t["k"] = x[:, :, :Hq].transpose(1, 2), x[:, :, Hq:Hq + Hkv].transpose(1, 2)
    else:
        for n, H in (("q", Hq), ("k", Hkv)):
            x = (normal(B, S, H, D) * 1.5).to(dt)
            t[n] = x.transpose(1, 2) if case["layout"] == "bshd" else x.transpose(1, 2).contiguous()
    if case["op"] == "norm_rotary":
        t["wq"], t["wk"] = ((1 + 0.2 * normal(D)).to(dt) for _ in range(2))
    if case["train"]:
        t["dq"], t["dk"] = (normal(B, S, H, D).to(dt).transpose(1, 2) for H in (Hq, Hkv))
    return t


def _cached_inputs(case, seed):
    gen, dt = _gen(seed), _DTYPES[case["dtype"]]
    Hq, Hkv, D, P = (case[x] for x in ("Hq", "Hkv", "D", "page"))
    lens, new = _ints(case["lens"]), _ints(case["new"])
    N, T = len(lens), sum(new)
    need = [(n + P - 1) // P for n in lens]
    # pages of the sequences lie anywhere in a pool that holds a few others
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((N, max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, c in enumerate(need):
        table[b, :c] = order[at:at + c]
        at += c

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dt)

    t = {"table": table, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "pool": pool}
    cu = [0]
    for m in new:
        cu.append(cu[-1] + m)
    t["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    t["cu_host"] = cu
    t["k"], t["v"] = (normal(pool, Hkv, P, D) for _ in range(2))
    if case["op"] == "paged":
        t["q"] = normal(T, Hq, D) * 1.5
    else:
        t["new_k"], t["new_v"] = (normal(T, Hkv, D) for _ in range(2))
    return t


def _store(case, x):
    """Pages of `x` as they are stored, and the scale of each row (or None)."""
    if case["store"] == "same":
        return x, None
    f = x.float()
    most = f.abs().amax(-1)
    if case["store"] == "e4m3":  # the smallest power of two that brings the row within 448
        part, power = torch.frexp(most / 448.0)
        scale = torch.ldexp(torch.ones_like(most), power - (part == 0.5).int())
    else:
        scale = most / 127.0
    scale = torch.where(most > 0, scale, 0.0).clamp_min(torch.finfo(torch.float32).tiny)
    f = f / scale[..., None]
    return (f.to(torch.float8_e4m3fn) if case["store"] == "e4m3" else f.round().to(torch.int8)), scale


def prepare(case, seed):
    if case["op"] in ("rotary", "norm_rotary"):
        t = _turn_inputs(case, seed)
        leaves = [t[n] for n in ("q", "k", "wq", "wk") if n in t]
        top = int(max(131072, case["start"] + case["S"]))
        st = {"case": case, "t": t, "leaves": leaves}
        if own:
            st["table"] = _cra().RotaryTable(case["rot"], top, base=_BASE, scaling=_SCALING[case["scaling"]],
                                             interleaved=case["interleaved"], device="cuda")
            for x in leaves:
                x.requires_grad_(case["train"])
        else:
            f, m = _frequencies(case["rot"], case["scaling"])
            a = torch.arange(top, dtype=torch.float64, device="cuda")[:, None] * f.cuda()
            st["cos"], st["sin"] = ((g(a) * m).float() for g in (torch.cos, torch.sin))
        return st
    t = _cached_inputs(case, seed)
    k, ks = _store(case, t["k"])
    v, vs = _store(case, t["v"])
    norm = t["k"].float().square().sum(-1)
    st = {"case": case, "table": t["table"], "lens": t["lens"], "cu": t["cu"], "cu_host": t["cu_host"],
          "lens_host": _ints(case["lens"]), "new_host": _ints(case["new"])}
    for n in ("q", "new_k", "new_v"):
        if n in t:
            # tokens of all sequences behind each other, as a projection leaves them: [1, H, T, D]
            st[n] = t[n][None].transpose(1, 2)
    if all(m == 1 for m in st["new_host"]) and "q" in st:
        st["q"] = t["q"][:, :, None]  # one token each: [N, H, 1, D]
    if own:
        st["cache"] = _cra().PagedKVCache.from_tensors(k, v, norm, ks, vs, dtype=_DTYPES[case["dtype"]],
                                                       head_dim=case["D"])
    else:
        st |= {"k": k, "v": v, "ks": ks, "vs": vs, "norm": norm}
    return st


# ---------------------------------------------------------------------------
# the pass
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if case["op"] in ("rotary", "norm_rotary"):
        return _run_turn_own(state) if own else _run_turn(state)
    if case["op"] == "paged":
        return _run_paged_own(state) if own else _run_paged(state)
    return _run_write_own(state) if own else _run_write(state)


def _run_turn_own(state):
    case, t, cra = state["case"], state["t"], _cra()

    def call():
        if case["op"] == "rotary":
            return cra.rotary_embedding(t["q"], t["k"], state["table"], t["pos"])
        return cra.qk_norm_rotary(t["q"], t["k"], t["wq"], t["wk"], state["table"], t["pos"], eps=_EPS)
    if not case["train"]:
        with torch.no_grad():
            return call()
    y = call()
    return [x.detach() for x in y] + list(torch.autograd.grad(y, state["leaves"], [t["dq"], t["dk"]]))


def _run_write_own(state):
    case, cache = state["case"], state["cache"]
    cache.write(state["new_k"], state["new_v"], state["table"], state["lens"], cu_seqlens=state["cu"])
    if case["op"] == "write":
        return _cache_values(case, cache.k, cache.v, cache.k_scale, cache.v_scale, cache.k_norm)
    return [*cache.read(state["table"], state["lens"], max(state["lens_host"])), cache.k_norm]


def _cache_values(case, k, v, ks, vs, norm):
    """What the cache holds: its own buffers, 8-bit ones as the values they stand for."""
    if ks is None:
        return [k, v, norm]
    return [k.float() * ks[..., None], v.float() * vs[..., None], norm]


def _run_paged_own(state):
    case = state["case"]
    ragged = state["q"].shape[0] != len(state["lens_host"]) or state["q"].shape[2] != 1
    return _cra().cron_root_attention_paged(
        state["q"], state["cache"], state["table"], state["lens"], cu_seqlens=state["cu"] if ragged else None,
        max_query_len=max(state["new_host"]), max_seqlen=max(state["lens_host"]), window=case["window"] or None)


# ---- the plain form --------------------------------------------------------
def _turn_plain(x, cos, sin, case, back=False):
    """x fp32 [B, H, S, D], cos and sin [.., S, rot/2]; back: the transpose."""
    rot = case["rot"]
    if case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    s = -sin if back else sin
    ya, yb = a * cos - b * s, b * cos + a * s
    y = torch.stack([ya, yb], -1).flatten(-2) if case["interleaved"] else torch.cat([ya, yb], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _run_turn(state):
    case, t = state["case"], state["t"]
    dt = _DTYPES[case["dtype"]]
    pos = t["pos"].long()
    cos, sin = state["cos"][pos], state["sin"][pos]
    if pos.dim() == 2:
        cos, sin = cos[:, None], sin[:, None]
    norm = case["op"] == "norm_rotary"
    out, grads, dws = [], [], []
    for n in "qk":
        x = t[n].float()
        if norm:
            w = t["w" + n].float()
            r = (x.square().mean(-1, keepdim=True) + _EPS).rsqrt()
            hat = x * r
            z = hat * w
        else:
            z = x
        out.append(_turn_plain(z, cos, sin, case).to(dt))
        if case["train"]:
            dz = _turn_plain(t["d" + n].float(), cos, sin, case, back=True)
            if norm:
                dws.append((dz * hat).sum((0, 1, 2)).to(dt))
                g = dz * w
                dz = r * (g - hat * (g * hat).mean(-1, keepdim=True))
            grads.append(dz.to(dt))
    return out + grads + dws


def _rows(pages, scale, table_row, heads, rows, P):
    """fp32 rows of one sequence: rows [L] or [Hkv, L] -> [Hkv, L, D]."""
    page, off = table_row[rows // P].long(), rows % P
    x = pages[page, heads[:, None], off].float()
    return x if scale is None else x * scale[page, heads[:, None], off][..., None]


def _run_write(state):
    case, P = state["case"], state["case"]["page"]
    table, cu = state["table"].long(), state["cu_host"]
    dt, dev = _DTYPES[case["dtype"]], table.device
    seq = torch.cat([torch.full((m,), b, device=dev) for b, m in enumerate(state["new_host"])])
    row = torch.cat([torch.arange(n - m, n, device=dev) for n, m in zip(state["lens_host"], state["new_host"])])
    page, off = table[seq, row // P], row % P
    for n in "kv":
        x = state["new_" + n][0].transpose(0, 1)  # [T, Hkv, D]
        codes, scale = _store(case, x)
        state[n][page, :, off] = codes
        if scale is not None:
            state[n + "s"][page, :, off] = scale
        if n == "k":
            state["norm"][page, :, off] = x.float().square().sum(-1)
    if case["op"] == "write":
        return _cache_values(case, state["k"], state["v"], state["ks"], state["vs"], state["norm"])
    heads = torch.arange(case["Hkv"], device=dev)
    outs = []
    for n in "kv":
        y = torch.zeros(len(state["lens_host"]), case["Hkv"], max(state["lens_host"]), case["D"], dtype=dt, device=dev)
        for b, L in enumerate(state["lens_host"]):
            y[b, :, :L] = _rows(state[n], state[n + "s"], table[b], heads, torch.arange(L, device=dev), P).to(dt)
        outs.append(y)
    return [*outs, state["norm"]]


def _run_paged(state):
    case, P = state["case"], state["case"]["page"]
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    table, q, cu = state["table"], state["q"], state["cu_host"]
    single = q.shape[0] == len(state["lens_host"]) and q.shape[2] == 1
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    heads = torch.arange(Hkv, device=q.device)
    for b, (n, m) in enumerate(zip(state["lens_host"], state["new_host"])):
        W, relay = _rule(n, case["window"])
        at = (lambda x: x[b]) if single else (lambda x: x[0, :, cu[b]:cu[b + 1]])
        qb, ob = at(q), at(out)  # [Hq, m, D]
        blocks = max(0, n - W) // W  # whole blocks before the last query's window
        per = 1 + _TOP_K if relay else 1
        nb = (max(0, n - W) + W - 1) // W
        G = torch.arange(nb, device=q.device) * W
        G = G[None, :, None].expand(Hkv, nb, per).clone()
        if relay and blocks:
            r = torch.arange(blocks * W, device=q.device)
            norm = state["norm"][table[b][r // P].long(), :, r % P].t().view(Hkv, blocks, W)
            best = norm.sort(dim=-1, descending=True, stable=True).indices[..., :_TOP_K]
            if W == 1:
                best = best.expand(Hkv, blocks, _TOP_K)
            G[:, :blocks, 1:] = best + (torch.arange(blocks, device=q.device) * W)[:, None]
        G = G.reshape(Hkv, -1)
        gk, gv = (_rows(state[x], state[x + "s"], table[b], heads, G, P) for x in "kv")
        C = max(16, min(m, (1 << 28) // (Hq * (G.shape[1] + min(n, W + m)))))
        for m0 in range(0, m, C):
            m1 = min(m, m0 + C)
            i = torch.arange(n - m + m0, n - m + m1, device=q.device)
            ls = (i - W + 1).clamp_min(0)
            lo, hi = max(0, n - m + m0 - W + 1), n - m + m1
            j = torch.arange(lo, hi, device=q.device)
            kk = torch.cat([gk, _rows(state["k"], state["ks"], table[b], heads, j[None], P)], 1)
            vv = torch.cat([gv, _rows(state["v"], state["vs"], table[b], heads, j[None], P)], 1)
            pre = per * (ls // W) + (ls % W != 0).long()
            see = torch.cat([torch.arange(G.shape[1], device=q.device)[None] < pre[:, None],
                             (j[None] <= i[:, None]) & (j[None] >= ls[:, None])], 1)
            qc = qb[:, m0:m1].float().reshape(Hkv, -1, D)
            s = torch.bmm(qc, kk.transpose(1, 2).contiguous()).view(Hkv, Hq // Hkv, m1 - m0, -1) / math.sqrt(D)
            s = s.masked_fill_(~see, -math.inf)
            p = (s - s.amax(-1, keepdim=True)).exp_()
            p = p / p.sum(-1, keepdim=True)
            ob[:, m0:m1] = torch.bmm(p.view(Hkv, -1, p.shape[-1]), vv).view(Hq, m1 - m0, D).to(q.dtype)
    return out


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] in ("rotary", "norm_rotary"):
        return _exact_turn(case, seed)
    with torch.no_grad():
        return _exact_paged(case, seed) if case["op"] == "paged" else _exact_write(case, seed)


def _exact_turn(case, seed):
    """Pairs as complex numbers times exp(i p f); the gradients by differentiation."""
    t = _turn_inputs(case, seed)
    f, m = _frequencies(case["rot"], case["scaling"])
    angle = t["pos"].double()[..., None] * f.cuda()
    if angle.dim() == 3:
        angle = angle[:, None]
    spin = torch.polar(torch.full_like(angle, m), angle)
    rot, outs, grads = case["rot"], [], []
    for n in "qk":
        x = t[n].double().requires_grad_(case["train"])
        w = t["w" + n].double().requires_grad_(case["train"]) if "w" + n in t else None
        z = x if w is None else x / (x.pow(2).sum(-1, keepdim=True) / case["D"] + _EPS).sqrt() * w
        h = z[..., :rot].unflatten(-1, (-1, 2) if case["interleaved"] else (2, -1))
        h = h if case["interleaved"] else h.transpose(-1, -2)
        h = torch.view_as_real(torch.view_as_complex(h.contiguous()) * spin)
        h = h if case["interleaved"] else h.transpose(-1, -2)
        y = torch.cat([h.flatten(-2), z[..., rot:]], -1)
        outs.append(y.detach())
        if case["train"]:
            grads.append(torch.autograd.grad(y, [x] if w is None else [x, w], t["d" + n].double()))
    return outs + [g[i] for i in range(len(grads[0]) if grads else 0) for g in grads]


def _exact_stored(case, x):
    """The values that the cache holds for rows x. A scale is stored as a 32-bit number."""
    if case["store"] == "same":
        return x.double()
    d = x.double()
    most = d.abs().amax(-1, keepdim=True)
    tiny = torch.finfo(torch.float32).tiny
    if case["store"] == "int8":
        scale = (most / 127).float().clamp_min(tiny).double()
        return (d / scale).round() * scale
    scale = torch.exp2(torch.floor(torch.log2(most.clamp_min(tiny) / 448)) - 1)
    for _ in range(3):  # up to the first power of two that holds the row
        scale = torch.where(448 * scale < most, 2 * scale, scale)
    scale = scale.clamp_min(tiny)
    y = d / scale
    # 3 bits behind the leading one, in steps of 2^-9 at least
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return (y / step).round() * step * scale


def _exact_write(case, seed):
    t = _cached_inputs(case, seed)
    P, lens, new = case["page"], _ints(case["lens"]), _ints(case["new"])
    norm = t["k"].double().square().sum(-1)
    k, v = (_exact_stored(case, t[x]) for x in "kv")
    nk, nv = (_exact_stored(case, t["new_" + x]) for x in "kv")
    at = 0
    for b, (n, m) in enumerate(zip(lens, new)):
        for p in range((n - m) // P, (n - 1) // P + 1):  # page by page
            lo, hi = max(n - m, p * P), min(n, (p + 1) * P)
            page, src = int(t["table"][b, p]), slice(at + lo - (n - m), at + hi - (n - m))
            k[page, :, lo - p * P:hi - p * P] = nk[src].transpose(0, 1)
            v[page, :, lo - p * P:hi - p * P] = nv[src].transpose(0, 1)
            norm[page, :, lo - p * P:hi - p * P] = t["new_k"][src].double().square().sum(-1).t()
        at += m
    if case["op"] == "write":
        return [k, v, norm]
    outs = []
    for x in (k, v):
        y = torch.zeros(len(lens), case["Hkv"], max(lens), case["D"], dtype=torch.float64, device="cuda")
        for b, n in enumerate(lens):
            whole = x[t["table"][b, :(n + P - 1) // P].long()]
            y[b, :, :n] = whole.transpose(0, 1).flatten(1, 2)[:, :n]
        outs.append(y)
    return [*outs, norm]


def _exact_paged(case, seed):
    """Every key of the sequence against every query, each counted as often as the query's set holds it."""
    Hq, Hkv, D, P = (case[x] for x in ("Hq", "Hkv", "D", "page"))
    lens, new = _ints(case["lens"]), _ints(case["new"])
    grp = Hq // Hkv
    if 4.0 * D * Hq * sum(n * m for n, m in zip(lens, new)) > 2e13 or Hkv * sum(new) * max(lens) > 1e11:
        return None
    t = _cached_inputs(case, seed)
    norm = t["k"].float().square().sum(-1)  # the norms that the cache is given
    (k, ks), (v, vs) = (_store(case, t[x]) for x in "kv")
    dev = t["q"].device
    out = torch.empty(Hq, sum(new), D, dtype=torch.float64, device=dev)
    at = 0
    for b, (n, m) in enumerate(zip(lens, new)):
        W, relay = _rule(n, case["window"])
        pages = t["table"][b, :(n + P - 1) // P].long()
        j = torch.arange(n, device=dev)
        nb = (n + W - 1) // W
        for h in range(Hkv):
            def whole(x, s):
                y = x[pages, h].double()
                return (y if s is None else y * s[pages, h][..., None].double()).reshape(-1, D)[:n]
            kk, vv = whole(k, ks), whole(v, vs)
            times = torch.zeros(n, dtype=torch.int64, device=dev)  # how often a row is a relay row of its block
            if relay:
                rank = torch.full((nb * W,), -1.0, dtype=torch.float64, device=dev)
                rank[:n] = norm[pages, h].reshape(-1)[:n].double()
                rank = rank.view(nb, W)
                for pick in range(_TOP_K):
                    top = rank.argmax(-1)
                    top = (rank == rank.gather(1, top[:, None])).to(torch.int8).argmax(-1)  # the first of equals
                    got = rank.gather(1, top[:, None])[:, 0] >= 0
                    first = torch.arange(nb, device=dev) * W
                    r = torch.where(got, first + top, first)  # nothing left: the block's first row
                    times.scatter_add_(0, r.clamp_max(n - 1), torch.ones_like(r))
                    rank.scatter_(1, top[:, None], -1.0)
            C = max(1, (1 << 27) // (n * grp))
            for m0 in range(0, m, C):
                m1 = min(m, m0 + C)
                i = torch.arange(n - m + m0, n - m + m1, device=dev)[:, None]
                ls = (i - W + 1).clamp_min(0)
                count = ((j <= i) & (j >= ls)).double()
                count += (j % W == 0) & (j < ls)
                count += times * ((j // W + 1) * W <= ls)
                qc = t["q"][at + m0:at + m1, h * grp:(h + 1) * grp].double().transpose(0, 1).reshape(-1, D)
                s = (qc @ kk.t().contiguous()).view(grp, m1 - m0, n) / math.sqrt(D)
                s = s - s.masked_fill(count == 0, -math.inf).amax(-1, keepdim=True)
                p = torch.where(count > 0, s, torch.full_like(s, -math.inf)).exp() * count
                o = (p.view(-1, n) @ vv) / p.sum(-1).view(-1, 1)
                out[h * grp:(h + 1) * grp, at + m0:at + m1] = o.view(grp, m1 - m0, D)
        at += m
    if all(m == 1 for m in new):
        return out.transpose(0, 1)[:, :, None]
    return out[None]
