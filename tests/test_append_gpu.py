"""New tokens appended to the paged cache with the norm and the rotation applied on the
way, on the GPU.

Appending is the norm and rotation and then the write, which have 64-bit oracles of their
own: the write of what append itself gives as a turned row is what it stores, bit for
bit, and a turned row is within the errors of both ways of the rotary operators'.
Against 64 bits here, errors counted: the table and each of two
products and a sum are rounded to fp32 (2^-24 each of |a| + |b|, with the multiplier of
cos and sin), the root mean square is off by at most (D + 4) 2^-24 of itself (a sum of D
squares, a mean, a root, two products), and the result is rounded once (eps / 2 of it).
"""
import math

import pytest
import torch

import cron_root_attention as cra
from paged_util import STORES, quantise

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def make(lens, new, Hq, Hkv, D, dtype, store="same", page=16, seed=0, pad=(0, 0), fused=True, garbage=True):
    """A cache, packed new tokens (with `pad` of padding before and behind), and their batch."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pool = sum(need) + 2
    order = torch.randperm(pool, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for b, c in enumerate(need):
        table[b, :c] = order[at:at + c]
        at += c
    cache = cra.PagedKVCache(pool, Hkv, D, page, dtype, STORES[store], device=DEV)
    if garbage:
        cache.k_norm.fill_(7.0)
        for t in (cache.k_scale, cache.v_scale):
            if t is not None:
                t.fill_(3.0)
        for t in (cache.k, cache.v):
            t.view(torch.uint8).fill_(0x39)
    cu = [pad[0]]
    for m in new:
        cu.append(cu[-1] + m)
    T = cu[-1] + pad[1]
    if fused:
        x = (torch.randn(1, T, Hq + 2 * Hkv, D, generator=g) * 1.5).to(dtype).to(DEV).transpose(1, 2)
        q, k, v = x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]
    else:
        q, k, v = ((torch.randn(1, H, T, D, generator=g) * 1.5).to(dtype).to(DEV) for H in (Hq, Hkv, Hkv))
    return cache, q, k, v, table.to(DEV), ints(lens), ints(cu)


def copy_of(c):
    own = [t if t is None else t.clone() for t in (c.k, c.v, c.k_norm, c.k_scale, c.v_scale)]
    return cra.PagedKVCache.from_tensors(*own, dtype=c.dtype, head_dim=c.head_dim)


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def apart(cache, q, k, v, pages, lens, cu, table=None, norm=False, q_weight=None, k_weight=None, eps=1e-6,
          positions=None):
    """The operators one after the other; padding is zeros."""
    if positions is None and table is not None:
        positions = cra.PagedBatch(pages, lens, cu).positions(q.shape[2])
    if norm:
        q, k = cra.qk_norm_rotary(q, k, q_weight, k_weight, table, positions, eps)
    else:
        q, k = cra.rotary_embedding(q, k, table, positions)
    cache.write(k, v, pages, lens, cu)
    if cu is not None:
        t = torch.arange(q.shape[2], device=DEV)
        q = torch.where(((t >= cu[0]) & (t < cu[-1]))[:, None], q, torch.zeros_like(q))
    return q


def close(got, want):
    """As near as two ways of turning a row are: (D + 8) 2^-24 of a pair's magnitudes each (at most
    2.9 times the row's largest), and a rounding that falls to the other side."""
    assert torch.equal(got.isnan(), want.isnan())
    x, y = got.double().nan_to_num(), want.double().nan_to_num()
    most = y.abs().amax(-1, keepdim=True)
    off = 2 * (y.shape[-1] + 8) * 2.0 ** -24 * 2.9 * most + 1.01 * torch.finfo(want.dtype).eps * y.abs()
    assert bool(((x - y).abs() <= off).all())


def agree(cache, q, k, v, pages, lens, cu, **kw):
    other, third = copy_of(cache), copy_of(cache)
    with torch.no_grad():
        want = apart(other, q, k, v, pages, lens, cu, **kw)
        got = cache.append(q, k, v, pages, lens, cu, **kw)
        # k as q: the same arithmetic, and its rows come back
        turned = copy_of(third).append(k, k, v, pages, lens, cu, **kw | {"q_weight": kw.get("k_weight")})
        third.write(turned, v, pages, lens, cu)
    assert got.dtype == q.dtype and got.shape == q.shape
    close(got, want)
    for n in ("k", "v", "k_norm", "k_scale", "v_scale"):
        x, y = getattr(cache, n), getattr(third, n)
        assert x is None or same_bits(x, y), n
    if cache.k.dtype == cache.dtype:
        close(cache.k, other.k)
        assert same_bits(cache.v, other.v)
    return got


LENS, NEW = [1, 16, 17, 300, 2049, 40, 9], [1, 5, 17, 1, 33, 0, 9]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("store", ["same", "e4m3", "int8"])
@pytest.mark.parametrize("D,rot,interleaved", [(64, 64, False), (128, 64, True), (80, 80, False), (256, 256, True),
                                               (128, 128, False), (96, 24, False), (16, 8, True), (80, 20, False),
                                               (8, 8, False), (256, 4, False), (32, 0, False)])
def test_same_as_the_operators_apart(dtype, store, D, rot, interleaved):
    table = cra.RotaryTable(rot, 4096, interleaved=interleaved, device=DEV) if rot else None
    w = [(1 + 0.3 * torch.randn(D, generator=torch.Generator().manual_seed(i))).to(DEV) for i in (1, 2)]
    for norm in (True, False):
        if not norm and not rot:
            continue
        args = make(LENS, NEW, 6, 2, D, dtype, store, seed=D + rot, pad=(2, 3))
        wq, wk = ([x.to(dtype) for x in w] if D % 32 else w) if norm else (None, None)
        agree(*args, table=table, norm=norm, q_weight=wq, k_weight=wk)


@pytest.mark.parametrize("H", [(1, 1), (40, 8), (3, 3), (16, 1)])
@pytest.mark.parametrize("new", [[1] * 70, [3, 0, 1, 0, 0, 200, 1, 2]])
def test_heads_and_many_sequences(H, new):
    lens = [m + 37 * i % 500 for i, m in enumerate(new)]
    table = cra.RotaryTable(64, 1024, device=DEV)
    agree(*make(lens, new, *H, 64, BF16, "same", seed=1), table=table, norm=True)


@pytest.mark.parametrize("H,fused", [((6, 2), True), ((6, 2), False), ((5, 1), True)])
@pytest.mark.parametrize("dtype,D,rot,interleaved", [(BF16, 128, 128, False), (F32, 80, 40, True), (F16, 16, 8, False)])
def test_many_rows(H, fused, dtype, D, rot, interleaved):
    new = [2001, 7, 0, 1, 1300, 31, 64, 65]
    lens = [m + 90 * i for i, m in enumerate(new)]
    table = cra.RotaryTable(rot, 4096, interleaved=interleaved, device=DEV)
    args = make(lens, new, *H, D, dtype, "same", seed=D, pad=(3, 70), fused=fused)
    w = [(1 + 0.3 * torch.randn(D, generator=torch.Generator().manual_seed(i))).to(DEV) for i in (1, 2)]
    agree(*args, table=table, norm=True, q_weight=w[0], k_weight=w[1])


@pytest.mark.parametrize("n", [1, 2, 62, 63, 64, 65, 200])
def test_numbers_of_sequences(n):
    new = [(7 * i + 3) % 5 for i in range(n)]
    new[-1] += n == 2
    lens = [m + 11 * i % 200 for i, m in enumerate(new)]
    table = cra.RotaryTable(64, 512, device=DEV)
    agree(*make(lens, new, 4, 2, 64, F16, "int8", seed=n, pad=(1, 2)), table=table, norm=True)


@pytest.mark.parametrize("fused", [True, False])
def test_layouts_and_single_tokens_without_offsets(fused):
    lens, D = [5, 77, 130], 64
    cache, q, k, v, pages, n, _ = make(lens, [1, 1, 1], 4, 2, D, F16, "e4m3", fused=fused)
    rows = [x.transpose(0, 2).contiguous() for x in (q, k, v)]  # [3, H, 1, D]
    table = cra.RotaryTable(D, 256, device=DEV)
    got = agree(cache, *rows, pages, n, None, table=table)
    assert got.stride() == rows[0].stride()
    # rows that do not lie between 16-byte addresses, and columns apart
    wide = torch.zeros(1, 4, 3, D + 1, dtype=F16, device=DEV)
    wide[..., 1:] = q
    agree(cache, wide[..., 1:], k, v, pages, n, ints([0, 1, 2, 3]), table=table)
    far = q.transpose(2, 3).contiguous().transpose(2, 3)
    agree(cache, far, k, v, pages, n, ints([0, 1, 2, 3]), table=table, norm=True)


@pytest.mark.parametrize("dtype,store", [(BF16, "same"), (F16, "int8"), (F32, "e4m3")])
def test_against_64_bits(dtype, store):
    D, Hq, Hkv, rot = 64, 4, 2, 32
    lens, new = [3000, 1, 700], [5, 1, 20]
    scaling = dict(type="yarn", factor=4.0, original_positions=1024)
    table = cra.RotaryTable(rot, 4096, scaling=scaling, interleaved=True, device=DEV)
    cache, q, k, v, pages, n, cu = make(lens, new, Hq, Hkv, D, dtype, store, seed=4)
    w = [(1 + 0.3 * torch.randn(D)).to(dtype).to(DEV) for _ in "qk"]
    with torch.no_grad():
        got = cache.append(q, k, v, pages, n, cu, table=table, norm=True, q_weight=w[0], k_weight=w[1])
        rk, rv = cache.read(pages, n)
    from cron_root_attention.rotary import rotary_frequencies
    f, mul = rotary_frequencies(rot, 10000.0, scaling)
    place = torch.cat([torch.arange(a - m, a) for a, m in zip(lens, new)]).double()
    spin = torch.polar(torch.full((len(place), rot // 2), mul, dtype=torch.float64), place[:, None] * f)

    def turned(x, w):
        z = x.double().cpu()
        z = z / (z.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double().cpu()
        h = torch.view_as_complex(z[..., :rot].unflatten(-1, (-1, 2)).contiguous()) * spin
        y = torch.cat([torch.view_as_real(h).flatten(-2), z[..., rot:]], -1)
        pair = z[..., :rot].abs().unflatten(-1, (-1, 2)).sum(-1).repeat_interleave(2, -1) * mul
        return y, torch.cat([pair, z[..., rot:].abs()], -1)

    eps = torch.finfo(dtype).eps
    y, mag = turned(q, w[0])
    assert bool(((got.double().cpu() - y).abs() <= (D + 8) * 2.0 ** -24 * mag + eps / 2 * y.abs()).all())
    # a stored key: what a row off by so much may be stored as; a code is off by half a step, the scale of a row by
    # what its largest element is
    y, mag = turned(k, w[1])
    off = (D + 8) * 2.0 ** -24 * mag + eps / 2 * y.abs()
    most = (y.abs() + off).amax(-1, keepdim=True)
    if store == "int8":
        off = off + most / 127 * 0.51 + off.amax(-1, keepdim=True) + eps / 2 * y.abs() * 1.1
    elif store == "e4m3":
        off = off * 1.1 + 2.0 ** -4 * y.abs() * 1.01 + most / 448 * 2.0 ** -9 + eps / 2 * y.abs() * 1.1
    held = torch.cat([rk[b, :, a - m:a] for b, (a, m) in enumerate(zip(lens, new))], 1)
    assert bool(((held.double().cpu() - y[0]).abs() <= off[0]).all())
    values = quantise(v[0].cpu(), STORES[store])[2]
    held = torch.cat([rv[b, :, a - m:a] for b, (a, m) in enumerate(zip(lens, new))], 1)
    assert bool(((held.double().cpu() - values).abs() <= eps / 2 * values.abs()).all())


def test_given_positions_and_ones_outside_the_table():
    table = cra.RotaryTable(64, 100, device=DEV)
    args = make([20, 90, 130], [3, 2, 4], 4, 2, 64, BF16, "same")
    for dtype in (torch.int32, torch.int64):
        pos = torch.tensor([0, 99, 5, 100, -1, 7, 7, 2 ** 30, 1], device=DEV, dtype=dtype)
        got = agree(*args, table=table, positions=pos)
        bad = got[0].isnan().all(0).all(-1)
        assert bad.tolist() == [False, False, False, True, True, False, False, True, False]
        agree(*args, table=table, positions=pos[None].expand(1, -1), norm=True)
    got = agree(*args, table=table)  # places 126 .. 129
    assert got[0].isnan().any(-1).any(0).tolist() == [False] * 5 + [True] * 4


def test_sequences_that_their_table_cannot_hold_or_shorter_than_their_new_tokens():
    table = cra.RotaryTable(64, 4096, device=DEV)
    cache, q, k, v, pages, n, cu = make([40, 40, 3], [4, 4, 3], 4, 2, 64, BF16, "same")
    n[0], n[2] = 50, 1  # 48 rows are held; two of three new tokens lie before the first row
    pages[1, 2] = 10 ** 6  # rows 36 .. 39 of sequence 1 lie outside the cache
    agree(cache, q, k, v, pages, n, cu, table=table)


def test_nothing_to_append():
    table = cra.RotaryTable(64, 64, device=DEV)
    cache, q, k, v, pages, n, cu = make([4, 5], [0, 0], 4, 2, 64, BF16, "same", pad=(0, 3))
    before = cache.k.clone()
    assert cache.append(q, k, v, pages, n, cu, table=table).abs().max() == 0
    assert same_bits(cache.k, before)
    empty = [x[:, :, :0] for x in (q, k, v)]
    assert cache.append(*empty, pages, n, ints([0, 0, 0]), table=table).shape == (1, 4, 0, 64)


def test_captured_and_replayed_on_another_stream():
    table = cra.RotaryTable(64, 4096, device=DEV)
    cache, q, k, v, pages, n, cu = make([5, 600], [1, 1], 4, 2, 64, BF16, "e4m3")
    other = copy_of(cache)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(stream):
        cache.append(q, k, v, pages, n, cu, table=table)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y = cache.append(q, k, v, pages, n, cu, table=table)
    torch.cuda.current_stream().wait_stream(stream)
    with torch.no_grad():
        other.append(q, k, v, pages, n, cu, table=table)
        for i in range(3):
            n += 1
            n.clamp_max_(608)
            q.copy_(torch.randn_like(q)), k.copy_(torch.randn_like(k))
            graph.replay()
            want = other.append(q, k, v, pages, n, cu, table=table)
            torch.cuda.synchronize()
            assert same_bits(y, want) and same_bits(cache.k, other.k) and same_bits(cache.k_norm, other.k_norm)


def test_refusals():
    table = cra.RotaryTable(64, 64, device=DEV)
    cache, q, k, v, pages, n, cu = make([4, 5], [1, 2], 4, 2, 64, BF16, "same")
    w = torch.ones(64, device=DEV)

    def no(error, *a, **kw):
        with pytest.raises(error):
            cache.append(*a, **kw)
    no(ValueError, q, k, v, pages, n, cu)
    no(ValueError, q, k, v, pages, n, cu, table=table, q_weight=w)
    no(ValueError, q[:, :, :2], k, v, pages, n, cu, table=table)
    no(ValueError, q, k, v[:, :, :2], pages, n, cu, table=table)
    no(ValueError, q, k[:, :1], v[:, :1], pages, n, cu, table=table)
    no(ValueError, q, k, v, pages, n, cu, table=cra.RotaryTable(128, 64, device=DEV))
    no(ValueError, q, k, v, pages, n, cu, table=cra.RotaryTable(64, 64, device="cpu"))
    no(ValueError, q, k, v, pages, n, cu, table=table, norm=True, q_weight=w[:32])
    no(ValueError, q, k, v, pages, n, cu, table=table, norm=True, eps=-1.0)
    no(ValueError, q, k, v, pages, n, cu, norm=True, positions=n)
    no(TypeError, q, k, v, pages, n, cu, table=w)
    no(TypeError, q.float(), k, v, pages, n, cu, table=table)
    no(TypeError, q, k, v, pages.long(), n, cu, table=table)
    no(TypeError, q, k, v, pages, n, cu, table=table, positions=n.float())
    no(NotImplementedError, q.detach().requires_grad_(), k, v, pages, n, cu, table=table)
    no(NotImplementedError, q, k, v, pages, n, cu, table=table, norm=True, k_weight=w.clone().requires_grad_())
    import torch.autograd.forward_ad as ad
    with ad.dual_level(), torch.no_grad():
        no(NotImplementedError, ad.make_dual(q, q), k, v, pages, n, cu, table=table)
    assert math.isfinite(float(cache.k.float().sum()))


@pytest.mark.parametrize("dtype,store", [(F16, "same"), (BF16, "e4m3"), (F32, "int8"), (F32, "same")])
@pytest.mark.parametrize("D,width,rot", [(64, 256, 0), (64, 128, 64), (32, 128, 32), (16, 64, 16), (8, 256, 0), (40, 256, 8),
                                         (24, 32, 24)])
def test_heads_narrower_than_the_rows_of_the_cache(dtype, store, D, width, rot):
    """Through the C ABI, which takes any head up to the cache's row: every token's row is stored,
    as the write stores the turned rows."""
    from cron_root_attention import _native as N
    lib, B, H, S, page = N.load_library(), 3, 2, 150, 16
    g = torch.Generator().manual_seed(D + width)
    k, v = (torch.randn(B, H, S, D, generator=g).to(dtype).to(DEV) for _ in "kv")
    wk = (1 + 0.3 * torch.randn(D, generator=g)).to(dtype).to(DEV)
    table = cra.RotaryTable(rot, 256, device=DEV) if rot else None
    pages = torch.randperm(40, generator=g)[:30].view(B, 10).to(torch.int32).to(DEV)
    lens = ints([150, 153, 160])
    batch = N.CraBatch(pages.data_ptr(), 10, lens.data_ptr(), None, B, 10, 0, S)

    def cache():
        own = [torch.full((40, H, page, n), 3.0, device=DEV).to(t or dtype)
               for n, t in ((width, STORES[store]),) * 2 + ((1, F32),) * 3]
        scales = [t.data_ptr() if store != "same" else None for t in own[3:]]
        return own, N.CraCache(*(t.data_ptr() for t in own[:3]), *scales, 40, H, page, width, N.dtype_code(dtype),
                               list(STORES).index(store))
    turn = N.CraTurn(B, H, H, S, D, rot, 0, 1, N.dtype_code(dtype), N.dtype_code(dtype), 0, 1e-6,
                     table.table.data_ptr() if rot else None, 256 if rot else 0, None, 0, 0)
    (a, ca), (b, cb), y = cache(), cache(), torch.empty_like(k)
    stream = torch.cuda.current_stream().cuda_stream
    ref = [N.ctypes.byref(x) for x in (ca, batch, turn, cb)]
    w = wk.data_ptr()
    assert lib.cra_cache_append(ref[0], ref[1], ref[2], N.row_arg(k), N.row_arg(k), N.row_arg(v), w, w, N.row_arg(y), stream) == 0
    assert lib.cra_cache_write(ref[3], ref[1], N.row_arg(y), N.row_arg(v), D, stream) == 0
    for s, t in zip(a, b):
        assert same_bits(s, t)


def test_tangents_of_the_norm_weights_are_refused():
    import torch.autograd.forward_ad as ad
    table = cra.RotaryTable(64, 64, device=DEV)
    cache, q, k, v, pages, n, cu = make([4, 5], [1, 2], 4, 2, 64, BF16, "same")
    w = torch.ones(64, device=DEV)
    for name in ("q_weight", "k_weight"):
        with ad.dual_level(), torch.no_grad(), pytest.raises(NotImplementedError):
            cache.append(q, k, v, pages, n, cu, table=table, norm=True, **{name: ad.make_dual(w, w)})
