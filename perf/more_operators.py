"""Performance cases of one serving step on one GPU: the projections as products in
8-bit floating point, new tokens appended to the paged cache with the norm and the
rotation applied on the way, and the attention of a batch whose sequences share a
long prefix.

A case is a dict of plain values; ``op`` names the operator:

    "linear"   y = x w^T (+ bias), x [M, K] in `dtype` and w [N, K]: both in e4m3 with
          a power-of-two scale, x for each row and 128 columns, w for each block of
          128 x 128; x comes as it is and is brought into 8 bits in the pass
    "append"   the last `new` tokens of every sequence: q and k normed (`norm`) and
          turned by their tokens' places in the sequences, k and v stored in a cache
          that holds sequences of `lens` tokens in pages of `page` rows, as `store`
          ("same" type, "e4m3" or "int8" with a scale for each row and head); 8-bit
          caches are read back
    "shared"   attention of M new tokens of every sequence over such a cache, whose
          sequences begin with the same `prefix` tokens in the same pages, and have
          `own` tokens behind them; window: that of the sqrt(N) pattern for every
          length (at least the length: dense causal attention)

``lens``, ``new`` and ``own`` are comma-separated numbers, one for each sequence.
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
_BASE = 10000.0
_BLOCK = 128


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


def _named(name, c):
    return dict(c, name=name) if name else c


def _linear(name, M, N, K, dtype, bias=False):
    return _named(name, dict(op="linear", M=M, N=N, K=K, dtype=dtype, bias=bias))


def _append(name, Hq, Hkv, D, dtype, store, page, lens, new, norm=True, rot=0, interleaved=False, scaling="none"):
    return _named(name, dict(op="append", Hq=Hq, Hkv=Hkv, D=D, dtype=dtype, store=store, page=page,
                             lens=",".join(map(str, lens)), new=",".join(map(str, new)), norm=norm, rot=rot or D,
                             interleaved=interleaved, scaling=scaling))


def _shared(name, Hq, Hkv, D, dtype, store, page, prefix, behind, M, window):
    return _named(name, dict(op="shared", Hq=Hq, Hkv=Hkv, D=D, dtype=dtype, store=store, page=page, prefix=prefix,
                             own=",".join(map(str, behind)), M=M, window=window))


_DENSE = 1 << 20
# Lengths of requests in one serving batch: a few long, most of them short.
_SERVED = (32768, 30001, 20480, 17777, 16384, 12345, 9001, 8192, 8191, 6000, 5000, 4097, 4096, 4095, 3500, 3333,
           2900, 2500, 2222, 2049, 2048, 2047, 1800, 1600, 1500, 1400, 1300, 1200, 1100, 1025, 1024, 1023,
           1000, 900, 850, 800, 750, 700, 640, 600, 555, 512, 511, 480, 444, 400, 366, 333,
           300, 280, 257, 256, 255, 222, 200, 180, 150, 129, 128, 100, 64, 33, 17, 1)
# Documents read in one pass: long, short, odd, one token.
_DOCS = (9001, 4096, 3333, 2049, 2048, 1500, 1023, 1000, 640, 511, 300, 257, 129, 64, 17, 1)


def _spread(n, lo, hi):
    """n lengths from lo to hi, evenly over their logarithm."""
    return [int(round(lo * (hi / lo) ** (i / max(1, n - 1)))) for i in range(n)]


def listed():
    return [
        # one token of one request through the joint projection of 32/8 heads: the weights are read once
        _linear("linear_token", 1, 6144, 4096, "bf16"),
        # a decoding step of 64 requests through an output projection
        _linear("linear_64", 64, 4096, 4096, "f16"),
        # a prompt of odd length through the joint projection of a small model, with bias, in full precision around it
        _linear("linear_1001", 1001, 2304, 768, "f32", bias=True),
        # prompts of a whole batch
        _linear("linear_16k", 16384, 6144, 4096, "bf16"),
        # one new token of each of 64 requests: launches and host time
        _append("append_token", 32, 8, 128, "bf16", "same", 16, _SERVED, [1] * len(_SERVED)),
        # a few drafted tokens of 16 requests into an integer cache, half of each head turned, no norm
        _append("append_drafts_int8", 16, 16, 64, "f16", "int8", 32, _SERVED[-16:], [min(5, n) for n in _SERVED[-16:]],
                norm=False, rot=32, interleaved=True),
        # prompts of many lengths into an 8-bit cache, stretched positions
        _append("append_26k_e4m3", 16, 4, 128, "bf16", "e4m3", 64, _DOCS, _DOCS, scaling="yarn"),
        # the tail of one long prompt
        _append("append_32k", 16, 16, 128, "f16", "same", 64, [65536], [32768]),
        # eight answers sampled to one prompt of a small model
        _shared("shared_8", 12, 12, 64, "f16", "same", 16, 2000, _spread(8, 1, 300), 1, _DENSE),
        # 64 requests behind one long system prompt, grouped heads, dense attention
        _shared("shared_64_32k", 32, 8, 128, "bf16", "same", 64, 32768, _spread(64, 1, 1000), 1, _DENSE),
        # the same over an 8-bit cache, a few drafted tokens each, a prefix that ends within a page
        _shared("shared_100_e4m3", 32, 8, 128, "bf16", "e4m3", 32, 15001, _spread(100, 2, 500), 2, _DENSE),
        # 48 requests about one document of the benchmark's length, in the sqrt(N) pattern the layer was trained with
        _shared("shared_48_128k", 16, 16, 128, "f16", "same", 64, 131072, _spread(48, 1, 2000), 1, 363),
    ]


# ---------------------------------------------------------------------------
# sizes
# ---------------------------------------------------------------------------
def _ints(text):
    return [int(x) for x in text.split(",")]


def _up(n, m):
    return (n + m - 1) // m


def _relay(n):
    return n > _RELAY_FROM


def _shared_sizes(case):
    """(query, key) pairs of one head, rows of the prefix and of all sequences' own that are seen, norms looked at."""
    P, M = case["prefix"], case["M"]
    pairs = prefix_rows = rows = norms = 0
    for x in _ints(case["own"]):
        n = P + x
        W, per = min(n, case["window"]), 1 + _TOP_K * int(_relay(n))
        for i in range(n - M, n):
            ls = max(0, i - W + 1)
            pairs += min(i + 1, W) + _up(ls, W) + (per - 1) * (ls // W)
        first, last = max(0, n - M - W + 1), max(0, n - W)
        in_prefix = _up(min(P, last), W) + (per - 1) * (min(P, last) // W)
        prefix_rows = max(prefix_rows, min(P, in_prefix + max(0, P - first)))
        seen = _up(last, W) + (per - 1) * (last // W) - in_prefix
        rows += min(x, n - max(P, first) + max(0, seen))
        norms = max(norms, min(P, last) // W * W if per > 1 else 0)
    return pairs, prefix_rows, rows, norms


def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": M * K * e + N * K + _up(N, _BLOCK) * _up(K, _BLOCK) + M * N * e + (N * e if case["bias"] else 0),
                "flops": 2 * M * N * K}
    D, Hq, Hkv = case["D"], case["Hq"], case["Hkv"]
    row = D * (e if case["store"] == "same" else 1) + (0 if case["store"] == "same" else 4)
    if case["op"] == "append":
        T, L = sum(_ints(case["new"])), sum(_ints(case["lens"]))
        b = T * (2 * Hq * D * e + Hkv * (2 * D * e + 2 * row + 4) + case["rot"] * 4)
        if case["store"] != "same":
            b += 2 * L * Hkv * (row + D * e)
        return {"bytes": b, "flops": T * (Hq + Hkv) * (3 * case["rot"] + (4 * D if case["norm"] else 0)) + 2 * T * Hkv * D}
    pairs, prefix_rows, rows, norms = _shared_sizes(case)
    T = case["M"] * len(_ints(case["own"]))
    return {"bytes": 2 * T * Hq * D * e + Hkv * (2 * (prefix_rows + rows) * row + 4 * norms), "flops": 4 * D * Hq * pairs}


def _held(case):
    """Bytes of what prepare() makes and the plain form holds."""
    e = _BYTES[case["dtype"]]
    if case["op"] == "linear":
        return case["N"] * case["K"]
    if case["op"] == "append":
        return sum(_ints(case["lens"])) * case["Hkv"] * case["D"] * e
    x = _ints(case["own"])
    return (case["prefix"] + len(x) * max(x)) * case["Hkv"] * case["D"] * e


_LARGEST = {}


def _fits(case):
    """Costs no more than the largest listed case of its kind: fp32 attention weighs more."""
    def cost(c):
        w = work(c)
        heavy = 8 if c["dtype"] == "f32" and c["op"] != "linear" else 1
        seqs = len(_ints(c["own"])) * c["M"] * c["Hq"] * (c["prefix"] if c["window"] >= _DENSE else 1) if "own" in c else 0
        return w["flops"] * heavy, w["bytes"], _held(c), seqs
    if case["op"] not in _LARGEST:
        _LARGEST[case["op"]] = [max(x) for x in zip(*(cost(c) for c in listed() if c["op"] == case["op"]))]
    return all(a <= b for a, b in zip(cost(case), _LARGEST[case["op"]]))


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "append", "append", "shared", "shared", "shared"])
    dtype = rng.choice(["f16", "f16", "bf16", "bf16", "bf16", "f32"])
    if op == "linear":
        while True:
            M = rng.choice([1, 1, _log_int(rng, 2, 16), _log_int(rng, 17, 256), _log_int(rng, 257, 16384)])
            N, K = _log_int(rng, 64, 16384), _log_int(rng, 64, 16384)
            if rng.random() < 0.6:  # sizes of heads
                N, K = 64 * _up(N, 64), 64 * _up(K, 64)
            else:
                K = 8 * _up(K, 8)
            case = _linear(None, M, N, K, dtype, rng.random() < 0.3)
            if _fits(case):
                return case
    D = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 256])
    Hkv = rng.choice([1, 2, 3, 4, 6, 8, 8, 12, 16])
    Hq = Hkv * rng.choice([g for g in (1, 1, 2, 4, 5, 8) if g * Hkv <= 64])
    store = rng.choice(["same", "same", "e4m3", "int8"])
    page = rng.choice([16, 16, 32, 64, 128, 256])
    if op == "append":
        store = "same" if dtype == "f32" else store
        N, most = _log_int(rng, 1, 96), _log_int(rng, 64, 65536)
        lens = [_log_int(rng, 1, most) for _ in range(N)]
        style = rng.choice(["token", "token", "few", "chunk", "mixed"])
        new = [min(n, {"token": 1, "few": rng.randint(1, 8), "chunk": _log_int(rng, 1, 8192)}[
            style if style != "mixed" else rng.choice(["token", "token", "few", "chunk"])]) for n in lens]
        more = dict(norm=rng.random() < 0.6, rot=rng.choice([D, D, D // 2, D // 4]), interleaved=rng.random() < 0.4,
                    scaling=rng.choice(["none", "linear", "ntk", "yarn"]))
        while True:
            case = _append(None, Hq, Hkv, D, dtype, store, page, lens, new, **more)
            if _fits(case):
                return case
            if len(lens) > 1:
                lens.pop(), new.pop()
            else:
                lens[0] = max(1, lens[0] // 2)
                new[0] = min(new[0], lens[0])
    M = rng.choice([1, 1, 1, 2, 3])
    N = _log_int(rng, 2, 128)
    prefix = _log_int(rng, 256, 131072)
    most = _log_int(rng, M, 2000)
    behind = [_log_int(rng, M, most) for _ in range(N)]
    window = rng.choice([_DENSE, _DENSE, math.isqrt(prefix) + 1, _log_int(rng, 64, 1024)])
    while True:
        case = _shared(None, Hq, Hkv, D, dtype, store, page, prefix, behind, M, window)
        if _fits(case):
            return case
        if len(behind) > 2:
            behind.pop()
        elif prefix > 256:
            prefix = max(256, prefix // 2)
        else:
            Hq, Hkv = Hq // Hkv, 1


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


_SCALING = {"none": None, "linear": dict(type="linear", factor=4.0), "ntk": dict(type="ntk", factor=4.0),
            "yarn": dict(type="yarn", factor=8.0, original_positions=16384)}
_POSITIONS = 131072


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


def _linear_inputs(case, seed):
    """Rows as a norm leaves them, a few columns much larger; weights of small, uneven scale."""
    gen, dt = _gen(seed), _DTYPES[case["dtype"]]
    M, N, K = case["M"], case["N"], case["K"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    column = torch.where(torch.rand(K, generator=gen, device="cuda") < 0.01, 20.0, 1.0)
    t = {"x": (normal(M, K) * column).to(dt)}
    t["w"] = (normal(N, K) * (0.5 + torch.rand(N, 1, generator=gen, device="cuda")) / math.sqrt(K)).to(torch.bfloat16)
    t["bias"] = normal(N).to(dt) if case["bias"] else None
    return t


def _pages(lens, page, gen):
    """Pages of sequences, anywhere in a pool that holds a few others: table [N, most], and the pool's size."""
    need = [_up(n, page) for n in lens]
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, c in enumerate(need):
        table[b, :c] = order[at:at + c]
        at += c
    return table, pool


def _append_inputs(case, seed):
    gen, dt = _gen(seed), _DTYPES[case["dtype"]]
    Hq, Hkv, D, P = (case[x] for x in ("Hq", "Hkv", "D", "page"))
    lens, new = _ints(case["lens"]), _ints(case["new"])
    table, pool = _pages(lens, P, gen)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    cu = [0]
    for m in new:
        cu.append(cu[-1] + m)
    t = {"table": table, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
         "cu": torch.tensor(cu, dtype=torch.int32, device="cuda"),
         "k": normal(pool, Hkv, P, D).to(dt), "v": normal(pool, Hkv, P, D).to(dt)}
    # tokens of all sequences behind each other, as one projection leaves them: [1, T, heads, D]
    x = (normal(1, cu[-1], Hq + 2 * Hkv, D) * 1.5).to(dt).transpose(1, 2)
    t["q"], t["new_k"], t["new_v"] = x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]
    if case["norm"]:
        t["wq"], t["wk"] = ((1 + 0.2 * normal(D)).to(dt) for _ in range(2))
    return t


def _shared_inputs(case, seed):
    gen, dt = _gen(seed), _DTYPES[case["dtype"]]
    Hq, Hkv, D, page, P, M = (case[x] for x in ("Hq", "Hkv", "D", "page", "prefix", "M"))
    behind = _ints(case["own"])
    N, whole = len(behind), P // page
    table, pool = _pages([whole * page] + [P % page + x for x in behind], page, gen)
    prefix, mine = table[0, :whole], table[1:, :_up(max(P % page + x for x in behind), page)]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dt)

    t = {"k": normal(pool, Hkv, page, D), "v": normal(pool, Hkv, page, D), "q": normal(N, Hq, M, D) * 1.5}
    if P % page:  # a page that the prefix ends in: each sequence has its own copy of those rows
        for x in (t["k"], t["v"]):
            x[mine[:, 0].long(), :, :P % page] = x[mine[0, 0].long(), :, :P % page]
    t["table"] = torch.cat([prefix.expand(N, -1), mine], 1).contiguous()
    t["lens"] = torch.tensor([P + x for x in behind], dtype=torch.int32, device="cuda")
    t["prefix_table"] = t["table"][0, :_up(P, page)].clone()
    t["prefix_len"] = torch.tensor([P], dtype=torch.int32, device="cuda")
    return t


def _power_scale(most):
    """The smallest power of two s with most <= 448 s, at least 2^-126."""
    part, power = torch.frexp(most / 448.0)
    scale = torch.ldexp(torch.ones_like(most), power - (part == 0.5).int())
    return torch.where(most > 0, scale, 0.0).clamp_min(torch.finfo(torch.float32).tiny)


def _store(store, x):
    """Rows `x` as they are stored, and the scale of each row (or None)."""
    if store == "same":
        return x, None
    f = x.float()
    most = f.abs().amax(-1)
    scale = _power_scale(most) if store == "e4m3" else (most / 127.0).clamp_min(torch.finfo(torch.float32).tiny)
    f = f / scale[..., None]
    return (f.to(torch.float8_e4m3fn) if store == "e4m3" else f.round().to(torch.int8)), scale


def _blocks(x, rows):
    """Codes of x [R, C] and the scale of each block of `rows` x 128 ([R / rows, C / 128], rounded up)."""
    R, C = x.shape
    f = torch.nn.functional.pad(x.float(), (0, -C % _BLOCK, 0, -R % rows))
    f = f.view(_up(R, rows), rows, _up(C, _BLOCK), _BLOCK)
    scale = _power_scale(f.abs().amax((1, 3)))
    codes = (f / scale[:, None, :, None]).to(torch.float8_e4m3fn)
    return codes.flatten(2).flatten(0, 1)[:R, :C], scale


def prepare(case, seed):
    st = {"case": case}
    if case["op"] == "linear":
        t = _linear_inputs(case, seed)
        st |= {"x": t["x"], "bias": t["bias"]}
        if own:
            st["w"] = _cra().E4M3Weight.from_dense(t["w"])
        else:
            st["codes"], st["scales"] = _blocks(t["w"], _BLOCK)
        return st
    append = case["op"] == "append"
    t = (_append_inputs if append else _shared_inputs)(case, seed)
    (k, ks), (v, vs) = (_store(case["store"], t.pop(x)) if x in t else None for x in ("k", "v"))
    norm = k.float() if ks is None else k.float() * ks[..., None]
    norm = norm.square().sum(-1)
    st |= t
    if append:
        st |= {"lens_host": _ints(case["lens"]), "new_host": _ints(case["new"])}
        if own:
            st["turns"] = _cra().RotaryTable(case["rot"], _POSITIONS, base=_BASE, scaling=_SCALING[case["scaling"]],
                                             interleaved=case["interleaved"], device="cuda")
        else:
            f, m = _frequencies(case["rot"], case["scaling"])
            a = torch.arange(_POSITIONS, dtype=torch.float64, device="cuda")[:, None] * f.cuda()
            st["cos"], st["sin"] = ((g(a) * m).float() for g in (torch.cos, torch.sin))
    else:
        st["own_host"] = _ints(case["own"])
    if own:
        st["cache"] = _cra().PagedKVCache.from_tensors(k, v, norm, ks, vs, dtype=_DTYPES[case["dtype"]], head_dim=case["D"])
    else:
        st |= {"k": k, "v": v, "ks": ks, "vs": vs, "norm": norm}
    return st


# ---------------------------------------------------------------------------
# the pass
# ---------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if op == "linear":
        return _run_linear_own(state) if own else _run_linear(state)
    if op == "append":
        return _run_append_own(state) if own else _run_append(state)
    return _run_shared_own(state) if own else _run_shared(state)


def _run_linear_own(state):
    return _cra().linear_e4m3(state["x"], state["w"], state["bias"])


def _run_append_own(state):
    case, cache = state["case"], state["cache"]
    q = cache.append(state["q"], state["new_k"], state["new_v"], state["table"], state["lens"], state["cu"],
                     table=state["turns"], norm=case["norm"], q_weight=state.get("wq"), k_weight=state.get("wk"), eps=_EPS)
    if case["store"] == "same":
        return _appended(case, q, cache.k, cache.v, cache.k_norm)
    return _appended(case, q, *cache.read(state["table"], state["lens"], max(state["lens_host"])), cache.k_norm)


def _appended(case, q, k, v, norm):
    """Keys that lie next to a border between two numbers of a 16-bit type round either way, and their
    sums of squares (fp32) follow by more than fp32's last bits: those come in the rows' type."""
    return [q, k, v, norm.to(_DTYPES[case["dtype"]])]


def _run_shared_own(state):
    cra, case = _cra(), state["case"]
    return cra.cron_root_attention_paged(
        state["q"], state["cache"], state["table"], state["lens"], window=case["window"],
        max_seqlen=case["prefix"] + max(state["own_host"]),
        prefix=cra.SharedPrefix(state["prefix_table"], state["prefix_len"]))


# ---- the plain form --------------------------------------------------------
def _run_linear(state):
    case, x = state["case"], state["x"]
    M, N, K = case["M"], case["N"], case["K"]
    codes, scale = _blocks(x, 1)
    f = codes.float() * scale.repeat_interleave(_BLOCK, 1)[:, :K]
    wide = state["scales"].repeat_interleave(_BLOCK, 0)[:N].repeat_interleave(_BLOCK, 1)[:, :K]
    y = f @ (state["codes"].float() * wide).t()
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(x.dtype)


def _turn_plain(x, cos, sin, case):
    """x fp32 [.., D], cos and sin [.., rot/2]."""
    rot = case["rot"]
    if case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    ya, yb = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([ya, yb], -1).flatten(-2) if case["interleaved"] else torch.cat([ya, yb], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _places(state):
    """Sequence and row of each new token."""
    cu, lens = state["cu"].long(), state["lens"].long()
    t = torch.arange(sum(state["new_host"]), device=cu.device)
    seq = torch.searchsorted(cu, t, right=True) - 1
    return seq, lens[seq] - cu[seq + 1] + t


def _run_append(state):
    case, P = state["case"], state["case"]["page"]
    dt, table = _DTYPES[case["dtype"]], state["table"].long()
    seq, row = _places(state)
    cos, sin = state["cos"][row], state["sin"][row]

    def turned(x, w):
        f = x.float()
        if w is not None:
            f = f * (f.square().mean(-1, keepdim=True) + _EPS).rsqrt() * w.float()
        return _turn_plain(f, cos, sin, case).to(dt)

    q, k = turned(state["q"], state.get("wq")), turned(state["new_k"], state.get("wk"))
    page, off = table[seq, row // P], row % P
    state["norm"][page, :, off] = k[0].float().square().sum(-1).t()
    for n, x in (("k", k), ("v", state["new_v"])):
        codes, scale = _store(case["store"], x[0].transpose(0, 1))
        state[n][page, :, off] = codes
        if scale is not None:
            state[n + "s"][page, :, off] = scale
    if case["store"] == "same":
        return _appended(case, q, state["k"], state["v"], state["norm"])
    j = torch.arange(max(state["lens_host"]), device=table.device)
    there = (j < state["lens"][:, None])[:, None, :, None]
    page, off = table[:, j // P].clamp_min(0), (j % P).expand(table.shape[0], -1)
    k, v = (torch.where(there, (state[n][page, :, off].float() * state[n + "s"][page, :, off][..., None]).transpose(1, 2),
                        0.0).to(dt) for n in "kv")
    return _appended(case, q, k, v, state["norm"])


def _rows_at(state, n, page, off, heads):
    """fp32 rows of k or v; page, off and heads broadcast together: [.., D]."""
    x = state[n][page, heads, off].float()
    return x if state[n + "s"] is None else x * state[n + "s"][page, heads, off][..., None]


def _best_rows(norm, blocks, W):
    """The _TOP_K rows of largest norm of each block [.., blocks, W] (as rows of the block)."""
    best = norm.view(*norm.shape[:-1], blocks, W).sort(dim=-1, descending=True, stable=True).indices[..., :_TOP_K]
    return best if W > 1 else best.expand(*best.shape[:-1], _TOP_K)


def _run_shared(state):
    """The scores of all queries against the prefix's rows (global rows, and its last window), and of
    each sequence's queries against its own, which begin with the block that the prefix ends in."""
    case = state["case"]
    Hq, Hkv, D, page, P, M = (case[x] for x in ("Hq", "Hkv", "D", "page", "prefix", "M"))
    q, dev = state["q"], state["q"].device
    N, g, most = q.shape[0], Hq // Hkv, P + max(state["own_host"])
    W, dense = min(case["window"], most), case["window"] >= most
    table, lens = state["table"].long(), state["lens"].long()
    relay, some = _relay(lens)[:, None, None], not dense and _relay(most)
    heads = torch.arange(Hkv, device=dev)
    i = lens[:, None] - M + torch.arange(M, device=dev)  # [N, M]
    ls = (i - W + 1).clamp_min(0)
    blocks = P // W
    # rows of the prefix: the first of every block, the best ones of whole blocks, the last window
    row = (torch.arange(_up(P, W), device=dev) * W).expand(Hkv, -1)
    seen = row[0] < ls[..., None]  # [N, M, rows]
    if some and blocks:
        j = torch.arange(blocks * W, device=dev)
        best = _best_rows(state["norm"][table[0, j // page], :, j % page].t(), blocks, W)
        best = best + (torch.arange(blocks, device=dev) * W)[:, None]
        row = torch.cat([row, best.flatten(1)], 1)
        end = ((torch.arange(blocks, device=dev) + 1) * W).repeat_interleave(_TOP_K)
        seen = torch.cat([seen, (end <= ls[..., None]) & relay], -1)
    j = torch.arange(max(0, P - W), P, device=dev)
    row = torch.cat([row, j.expand(Hkv, -1)], 1)
    seen = torch.cat([seen, j >= ls[..., None]], -1)
    pk, pv = (_rows_at(state, n, table[0][row // page], row % page, heads[:, None]) for n in "kv")  # [Hkv, R, D]
    x = q.float().view(N, Hkv, g, M, D)
    s = torch.bmm(x.transpose(0, 1).reshape(Hkv, -1, D), pk.transpose(1, 2).contiguous()).view(Hkv, N, g, M, -1)
    s = (s / math.sqrt(D)).masked_fill_(~seen[None, :, None], -math.inf)
    # each sequence's own rows, and how often a query's set holds them
    first, L = (P, most - P) if dense else (blocks * W, _up(most - blocks * W, W) * W)
    j = first + torch.arange(L, device=dev)
    at = j.clamp_max(table.shape[1] * page - 1)
    pages, off = table[:, at // page].clamp_min(0), (at % page).expand(N, -1)
    i, ls = i[:, None, :, None], ls[:, None, :, None]  # [N, 1, M, 1]
    count = ((j >= P) & (j <= i) & (j >= ls)).int() + ((j >= P) & (j % W == 0) & (j < ls)).int()
    if some:
        norm = state["norm"][pages, :, off].transpose(1, 2).masked_fill(j >= lens[:, None, None], -1.0)
        best = _best_rows(norm, L // W, W) + (torch.arange(L // W, device=dev) * W)[:, None]
        times = torch.zeros(N, Hkv, L, dtype=torch.int32, device=dev)
        times.scatter_add_(2, best.flatten(2), torch.ones_like(best.flatten(2), dtype=torch.int32))
        count = count + times[:, :, None] * (((j // W + 1) * W <= ls) & relay[..., None]).int()
    ok, ov = (_rows_at(state, n, pages[:, None], off[:, None], heads[:, None]) for n in "kv")  # [N, Hkv, L, D]
    t = torch.bmm(x.reshape(N * Hkv, g * M, D), ok.flatten(0, 1).transpose(1, 2).contiguous()) / math.sqrt(D)
    t = t.view(N, Hkv, g, M, L) + count.expand(N, Hkv, M, L).float().log()[:, :, None]
    # one softmax over both
    top = torch.maximum(s.amax(-1).transpose(0, 1), t.amax(-1))[..., None]  # [N, Hkv, g, M, 1]
    p, r = (s - top.transpose(0, 1)).exp_(), (t - top).exp_()
    total = p.sum(-1, keepdim=True).transpose(0, 1) + r.sum(-1, keepdim=True)
    o = torch.bmm(p.view(Hkv, N * g * M, -1), pv).view(Hkv, N, g, M, D).transpose(0, 1)
    o = o + torch.bmm(r.view(N * Hkv, g * M, L), ov.flatten(0, 1)).view(N, Hkv, g, M, D)
    return (o / total).reshape(N, Hq, M, D).to(q.dtype)


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def exact(case, seed):
    with torch.no_grad():
        return {"linear": _exact_linear, "append": _exact_append, "shared": _exact_shared}[case["op"]](case, seed)


def _round_e4m3(y):
    """To 3 bits behind the leading one, in steps of 2^-9 at least."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return (y / step).round() * step


def _exact_scale(most):
    """The smallest power of two s with most <= 448 s, found step by step."""
    tiny = torch.finfo(torch.float32).tiny
    scale = torch.exp2(torch.floor(torch.log2(most.clamp_min(tiny) / 448)) - 1)
    for _ in range(3):
        scale = torch.where(448 * scale < most, 2 * scale, scale)
    return scale.clamp_min(tiny)


def _exact_linear(case, seed):
    t = _linear_inputs(case, seed)
    x, w = t["x"].double(), t["w"].double()
    y = torch.zeros(case["M"], case["N"], dtype=torch.float64, device="cuda")
    for c in range(0, case["K"], _BLOCK):  # block by block
        a, b = x[:, c:c + _BLOCK], w[:, c:c + _BLOCK]
        s = _exact_scale(a.abs().amax(1, keepdim=True))
        qa = _round_e4m3(a / s) * s
        qb = torch.empty_like(b)
        for r in range(0, case["N"], _BLOCK):
            part = b[r:r + _BLOCK]
            s = _exact_scale(part.abs().max())
            qb[r:r + _BLOCK] = _round_e4m3(part / s) * s
        y += qa @ qb.t().contiguous()
    return y if t["bias"] is None else y + t["bias"].double()


def _exact_stored(store, x):
    """The values that the cache holds for rows x. A scale is stored as a 32-bit number."""
    if store == "same":
        return x.double()
    d = x.double()
    most = d.abs().amax(-1, keepdim=True)
    if store == "int8":
        scale = (most / 127).float().clamp_min(torch.finfo(torch.float32).tiny).double()
        return (d / scale).round() * scale
    scale = _exact_scale(most)
    return _round_e4m3(d / scale) * scale


def _exact_append(case, seed):
    """Pairs as complex numbers times exp(i p f). A key is a number of the rows' type before it is stored."""
    t = _append_inputs(case, seed)
    P, rot, dt = case["page"], case["rot"], _DTYPES[case["dtype"]]
    lens, new = _ints(case["lens"]), _ints(case["new"])
    f, m = _frequencies(rot, case["scaling"])
    place = torch.cat([torch.arange(n - c, n) for n, c in zip(lens, new)]).double().cuda()
    angle = place[:, None] * f.cuda()
    spin = torch.polar(torch.full_like(angle, m), angle)

    def turned(x, w):
        z = x.double()
        if w is not None:
            z = z / (z.pow(2).sum(-1, keepdim=True) / case["D"] + _EPS).sqrt() * w.double()
        h = z[..., :rot].unflatten(-1, (-1, 2) if case["interleaved"] else (2, -1))
        h = h if case["interleaved"] else h.transpose(-1, -2)
        h = torch.view_as_real(torch.view_as_complex(h.contiguous()) * spin)
        h = h if case["interleaved"] else h.transpose(-1, -2)
        return torch.cat([h.flatten(-2), z[..., rot:]], -1)

    q, k = turned(t["q"], t.get("wq")), turned(t["new_k"], t.get("wk")).to(dt)[0].transpose(0, 1)
    held, fresh = {}, {"k": k, "v": t["new_v"][0].transpose(0, 1)}
    norm = _exact_stored(case["store"], t["k"]).square().sum(-1)
    for n in "kv":
        x, y = _exact_stored(case["store"], t[n]), _exact_stored(case["store"], fresh[n])
        at = 0
        for b, (length, count) in enumerate(zip(lens, new)):
            for p in range((length - count) // P, (length - 1) // P + 1):  # page by page
                lo, hi = max(length - count, p * P), min(length, (p + 1) * P)
                page, src = int(t["table"][b, p]), slice(at + lo - (length - count), at + hi - (length - count))
                x[page, :, lo - p * P:hi - p * P] = y[src].transpose(0, 1)
                if n == "k":
                    norm[page, :, lo - p * P:hi - p * P] = k[src].double().square().sum(-1).t()
            at += count
        if case["store"] != "same":
            whole = torch.zeros(len(lens), case["Hkv"], max(lens), case["D"], dtype=torch.float64, device="cuda")
            for b, length in enumerate(lens):
                pages = x[t["table"][b, :_up(length, P)].long()]
                whole[b, :, :length] = pages.transpose(0, 1).flatten(1, 2)[:, :length]
            x = whole
        held[n] = x
    return [q, held["k"], held["v"], norm]


def _exact_shared(case, seed):
    """Every key of a sequence against its queries, each counted as often as the query's set holds it."""
    Hq, Hkv, D, page, P, M = (case[x] for x in ("Hq", "Hkv", "D", "page", "prefix", "M"))
    behind, g = _ints(case["own"]), Hq // Hkv
    if len(behind) * Hkv > 4000:
        return None
    t = _shared_inputs(case, seed)
    (k, ks), (v, vs) = (_store(case["store"], t[x]) for x in "kv")
    norm = (k.float() if ks is None else k.float() * ks[..., None]).square().sum(-1)  # as the cache is given them
    dev = t["q"].device
    out = torch.empty(len(behind), Hq, M, D, dtype=torch.float64, device=dev)
    for b, x in enumerate(behind):
        n = P + x
        W = min(n, case["window"])
        pages = t["table"][b, :_up(n, page)].long()
        j, nb = torch.arange(n, device=dev), _up(n, W)
        for h in range(Hkv):
            def whole(z, s):
                y = z[pages, h].double()
                return (y if s is None else y * s[pages, h][..., None].double()).reshape(-1, D)[:n]
            kk, vv = whole(k, ks), whole(v, vs)
            times = torch.zeros(n, dtype=torch.int64, device=dev)  # how often a row is a relay row of its block
            if _relay(n):
                rank = torch.full((nb * W,), -1.0, dtype=torch.float64, device=dev)
                rank[:n] = norm[pages, h].reshape(-1)[:n].double()
                rank = rank.view(nb, W)
                for pick in range(_TOP_K):
                    top = rank.argmax(-1)
                    top = (rank == rank.gather(1, top[:, None])).to(torch.int8).argmax(-1)  # the first of equals
                    got = rank.gather(1, top[:, None])[:, 0] >= 0
                    r = torch.arange(nb, device=dev) * W
                    r = torch.where(got, r + top, r)  # nothing left: the block's first row
                    times.scatter_add_(0, r.clamp_max(n - 1), torch.ones_like(r))
                    rank.scatter_(1, top[:, None], -1.0)
            i = torch.arange(n - M, n, device=dev)[:, None]
            ls = (i - W + 1).clamp_min(0)
            count = ((j <= i) & (j >= ls)).double()
            count += (j % W == 0) & (j < ls)
            count += times * ((j // W + 1) * W <= ls)
            z = t["q"][b, h * g:(h + 1) * g].double().reshape(-1, D)
            s = (z @ kk.t().contiguous()).view(g, M, n) / math.sqrt(D)
            s = s - s.masked_fill(count == 0, -math.inf).amax(-1, keepdim=True)
            p = torch.where(count > 0, s, torch.full_like(s, -math.inf)).exp() * count
            o = (p.view(-1, n) @ vv) / p.sum(-1).view(-1, 1)
            out[b, h * g:(h + 1) * g] = o.view(g, M, D)
    return out
