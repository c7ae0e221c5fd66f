"""The paged cache and the attention over it on the GPU against 64-bit oracles.

Cache: what is written is exact (codes and scales bit for bit), what is read is
rounded once. Attention, errors counted: scores in fp32 leave exp off by at most
about 2^-15 (D products of |q k| up to 40 in units of 2^-24, times the largest
score); P is rounded to the type (eps/2 of each weight), V of an 8-bit cache once
more (eps/2), the result once (eps/2 of the value). So |o - ref| <= (eps + 2^-14)
sum p |v| + eps/2 |ref|, in fp32 with its own eps and 2^-17 for the scores.
"""
import math
import random

import pytest
import torch

import cron_root_attention as cra
from paged_util import STORES, attend, norm_sq, quantise

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


class Setup:
    """A cache filled through write(), and the oracle's own copy of the sequences."""

    def __init__(self, lens, Hkv, D, dtype, store="same", page=16, seed=0, spare=3, table_extra=0):
        self.lens, self.Hkv, self.D, self.dtype = list(lens), Hkv, D, dtype
        g = torch.Generator().manual_seed(seed)
        self.g = g
        need = [-(-n // page) for n in lens]
        pool = sum(need) + spare
        order = torch.randperm(pool, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max(need + [1]) + table_extra), -1, dtype=torch.int32)
        at = 0
        for b, c in enumerate(need):
            self.table[b, :c] = order[at:at + c]
            at += c
        self.cache = cra.PagedKVCache(pool, Hkv, D, page, dtype, STORES[store], device=DEV)
        # garbage where nothing is written: NaN must not come out of it
        self.cache.k_norm.fill_(math.nan)
        if store == "same":
            self.cache.k.fill_(math.nan), self.cache.v.fill_(math.nan)
        else:
            self.cache.k_scale.fill_(math.nan), self.cache.v_scale.fill_(math.nan)
        T = sum(lens)
        self.k, self.v = (torch.randn(T, Hkv, D, generator=g).to(dtype) for _ in "kv")
        self.cu = [0]
        for n in lens:
            self.cu.append(self.cu[-1] + n)
        self.dtable = self.table.to(DEV)
        if T:
            self.write(self.k, self.v, self.lens, self.cu)

    def ints(self, x):
        return torch.tensor(x, dtype=torch.int32, device=DEV)

    def write(self, k, v, lens, cu):
        self.cache.write(k.to(DEV)[None].transpose(1, 2), v.to(DEV)[None].transpose(1, 2), self.dtable,
                         self.ints(lens), cu_seqlens=self.ints(cu))

    def held(self, b, h):
        """Values (fp64) and norms of a sequence's head as the cache must hold them."""
        sl = slice(self.cu[b], self.cu[b + 1])
        k, v = self.k[sl, h], self.v[sl, h]
        st = None if self.cache.k.dtype == self.dtype else self.cache.k.dtype
        return quantise(k, st)[2], quantise(v, st)[2], norm_sq(k)

    def expect(self, q, new, **kw):
        """Oracle of packed q [T, Hq, D]."""
        T, Hq, D = q.shape
        g = Hq // self.Hkv
        o, mag = (torch.zeros(T, Hq, D, dtype=torch.float64) for _ in "om")
        at = 0
        for b, (n, m) in enumerate(zip(self.lens, new)):
            for h in range(self.Hkv if m else 0):
                k, v, norm = self.held(b, h)
                qq = q[at:at + m, h * g:(h + 1) * g].transpose(0, 1)
                x, y = attend(qq, k, v, norm, n, m, **kw)
                o[at:at + m, h * g:(h + 1) * g], mag[at:at + m, h * g:(h + 1) * g] = x.transpose(0, 1), y.transpose(0, 1)
            at += m
        return o, mag


def check(got, o, mag, dtype):
    eps = torch.finfo(dtype).eps
    tol = (eps + (2.0 ** -17 if dtype == F32 else 2.0 ** -14)) * mag + eps / 2 * o.abs() + torch.finfo(dtype).tiny
    off = (got.double().cpu() - o).abs() - tol
    assert bool((off <= 0).all()), f"{int((~(off <= 0)).sum())} elements off, worst by {float(off.max()):.3e}"


def run(s, q, new, **kw):
    """Packed q [T, Hq, D] through the public call."""
    cu = [0]
    for m in new:
        cu.append(cu[-1] + m)
    with torch.no_grad():
        o = cra.cron_root_attention_paged(q.to(DEV)[None].transpose(1, 2), s.cache, s.dtable, s.ints(s.lens),
                                          cu_seqlens=s.ints(cu), **kw)
    assert o.shape == (1, q.shape[1], q.shape[0], q.shape[2])
    return o[0].transpose(0, 1)


# ------------------------------------------------------------------ cache
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("store", ["same", "e4m3", "int8"])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 64), (80, 32), (33, 16), (256, 16), (7, 1024)])
def test_write_and_read(dtype, store, D, page):
    s = Setup([1, 16, 17, 63, 130, 5], 3, D, dtype, store, page, seed=D)
    W = (D + 15) // 16 * 16
    assert s.cache.k.shape[-1] == W
    for b, n in enumerate(s.lens):
        pages = s.table[b, :-(-n // page)].long()
        for name in "kv":
            x = getattr(s, name)[s.cu[b]:s.cu[b + 1]].transpose(0, 1)  # [Hkv, n, D]
            codes, scale, _ = quantise(x, STORES[store])
            got = getattr(s.cache, name).cpu()[pages].transpose(0, 1).flatten(1, 2)[:, :n]
            if store == "e4m3":
                got, codes = got.view(torch.int8), codes.view(torch.int8)
            assert torch.equal(got[..., :D], codes), (b, name)
            assert not got[..., D:].float().any()
            if scale is not None:
                sc = getattr(s.cache, name + "_scale").cpu()[pages].transpose(0, 1).flatten(1, 2)[:, :n]
                assert torch.equal(sc, scale)
        norm = s.cache.k_norm.cpu()[pages].transpose(0, 1).flatten(1, 2)[:, :n]
        assert torch.equal(norm, norm_sq(s.k[s.cu[b]:s.cu[b + 1]].transpose(0, 1)))
    k, v = s.cache.read(s.dtable, s.ints(s.lens), 131)
    assert k.shape == v.shape == (6, 3, 131, D) and k.dtype == dtype
    for b, n in enumerate(s.lens):
        for h in range(3):
            wk, wv, _ = s.held(b, h)
            # the stored value, rounded once: codes times scales are exact in fp32
            assert torch.equal(k[b, h, :n].cpu(), wk.float().to(dtype)), (b, h)
            assert torch.equal(v[b, h, :n].cpu(), wv.float().to(dtype))
        assert not k[b, :, n:].any() and not v[b, :, n:].any()


@pytest.mark.parametrize("store", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_scales_of_special_rows(store, dtype):
    """Zeros, the type's extremes, values at the codes' ties and borders, infinities and NaN."""
    D = 32
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    rows = torch.zeros(12, D)
    rows[1] = big
    rows[2] = -tiny
    rows[3] = tiny * torch.finfo(dtype).eps  # the smallest subnormal
    rows[4] = torch.linspace(-448, 448, D)
    rows[5] = torch.arange(D) * 8.0 + 200
    rows[6, 0], rows[6, 1:] = 448, 17.0  # ties of e4m3 between 16 and 18
    rows[7, 0], rows[7, 1:] = 127, torch.arange(1, D) - 0.5  # ties of int8
    rows[8, 5] = math.inf
    rows[9, 7] = math.nan
    rows[10, 0], rows[10, 3] = -math.inf, math.nan
    rows[11, 0] = 449
    x = rows.to(dtype)
    s = Setup([12], 1, D, dtype, store)
    s.k = s.v = x[:, None]
    s.write(s.k, s.v, [12], [0, 12])
    codes, scale, value = quantise(x, STORES[store])
    page = int(s.table[0, 0])
    assert torch.equal(s.cache.k_scale[page, 0, :12].cpu().nan_to_num(-1), scale.nan_to_num(-1))
    got = s.cache.k[page, 0, :12].cpu()
    fine = scale.isfinite()
    assert torch.equal(got[fine].view(torch.int8), codes[fine].view(torch.int8))
    k, _ = s.cache.read(s.dtable, s.ints([12]), 12)
    k = k[0, 0].cpu()
    assert k[8:11].isnan().all() and torch.equal(k[fine], value[fine].float().to(dtype))


def test_write_passes_over_padding_bad_pages_and_rows_before_the_start():
    s = Setup([20, 30], 2, 64, F16, page=16, spare=4)
    before = [t.clone() for t in (s.cache.k, s.cache.v, s.cache.k_norm)]
    k = torch.randn(1, 2, 12, 64, device=DEV).half()
    # tokens 0 and 1 before, 10 and 11 behind the sequences; page ids outside the cache
    table = s.dtable.clone()
    table[0, 1] = 1 << 30
    table[1, 1] = -7
    s.cache.write(k, k, table, s.ints([20, 30]), cu_seqlens=s.ints([2, 6, 10]))
    for a, b in zip(before, (s.cache.k, s.cache.v, s.cache.k_norm)):
        assert torch.equal(a.nan_to_num(-9), b.nan_to_num(-9))
    # more new tokens than the sequence is long: the last 3 of 5 are its rows
    table = s.dtable
    s.cache.write(k[:, :, :5], k[:, :, :5], table[:1], s.ints([3]), cu_seqlens=s.ints([0, 5]))
    got, _ = s.cache.read(table[:1], s.ints([3]), 4)
    assert torch.equal(got[0, :, :3], k[0, :, 2:5]) and not got[0, :, 3].any()
    # a length beyond what the table's row holds is held within it
    kk, _ = s.cache.read(table[:, :1], s.ints([1 << 30, -5]), 40)
    assert not kk[0, :, 16:].any() and not kk[1].any()
    kk, _ = s.cache.read(torch.full((1, 2), 99, dtype=torch.int32, device=DEV), s.ints([20]), 32)
    assert kk[0, :, :20].isnan().all() and not kk[0, :, 20:].any()


def test_write_layouts_and_batch_forms():
    """[N, H, M, D] batches, strided rows, an odd head dim in an unaligned slice."""
    N_, H, M, D = 3, 2, 4, 20
    cache = cra.PagedKVCache(6, H, D, 16, BF16, device=DEV)
    table = torch.tensor([[0, 3], [1, 4], [2, 5]], dtype=torch.int32, device=DEV)
    x = torch.randn(N_, M, H, D + 1, device=DEV).bfloat16()[..., 1:].transpose(1, 2)
    y = torch.randn(N_, H, M, D, device=DEV).bfloat16()
    lens = torch.tensor([4, 17, 32], dtype=torch.int32, device=DEV)
    cache.write(x, y, table, lens)
    k, v = cache.read(table, lens)
    for b, n in enumerate([4, 17, 32]):
        assert torch.equal(k[b, :, n - M:n], x[b]) and torch.equal(v[b, :, n - M:n], y[b])
    assert k.shape[2] == 32


# ------------------------------------------------------------------ attention
CASES = [
    # lens, new, Hq, Hkv, D, page, kw
    ([1], [1], 1, 1, 64, 16, {}),
    ([1, 2, 3, 31, 32, 33, 64, 65, 100], [1] * 9, 2, 2, 64, 16, {}),
    ([5, 300, 17], [2, 3, 17], 4, 4, 128, 32, {}),
    ([2047, 2048, 2049, 2500], [1, 1, 1, 1], 8, 2, 128, 64, {}),            # relay from 2049 on
    ([2600, 40], [20, 40], 6, 2, 64, 16, {}),                               # chunks, three heads a kv head
    ([2100], [70], 10, 2, 32, 128, {}),
    ([400, 1000], [133, 64], 4, 2, 256, 16, {}),
    ([300, 5, 900], [64, 1, 100], 3, 3, 80, 64, dict(window=1 << 30)),      # dense causal
    ([1500], [1], 16, 1, 96, 16, dict(window=1 << 30)),
    ([700, 650], [40, 1], 2, 1, 64, 16, dict(window=7, relay=True)),        # many small blocks
    ([130], [130], 2, 2, 128, 16, dict(window=1, relay=True, relay_top_k=4)),  # blocks smaller than top_k
    ([900, 901], [30, 2], 4, 2, 64, 32, dict(window=64, relay=True, relay_top_k=1)),
    ([900, 2300], [1, 35], 4, 2, 33, 16, dict(relay=False)),
    ([0, 10, 0, 50], [0, 3, 0, 20], 2, 1, 64, 16, {}),                      # empty sequences
    ([4, 7], [6, 40], 2, 1, 64, 16, {}),                                    # more new tokens than rows
    ([64, 128, 192], [32, 64, 128], 2, 1, 64, 16, dict(window=64)),         # everything on tile borders
    ([0, 0, 5, 40], [1, 20, 9, 2], 2, 1, 64, 16, {}),                       # new tokens of empty sequences
    ([2500, 40, 3000], [1, 3, 1], 40, 1, 64, 16, {}),                       # one kv head for many query heads
    ([2500, 40, 3001], [1, 3, 1], 160, 1, 32, 16, dict(window=1 << 30)),
    ([2300, 1700], [1, 30], 2, 2, 64, 32, dict(window=600, relay=True, relay_top_k=3)),  # wide blocks
    ([1100, 2040], [20, 1], 2, 2, 64, 16, dict(window=506, relay=True)),
    ([1100, 2040], [1, 20], 2, 2, 64, 16, dict(window=505, relay=True, relay_top_k=4)),
    ([1000, 777], [1, 3], 2, 2, 64, 16, dict(window=121, relay=True, relay_top_k=4)),  # blocks of 16, 32, 64 lanes
    ([1000, 777], [1, 3], 2, 2, 64, 16, dict(window=122, relay=True, relay_top_k=4)),
    ([1000, 1777], [1, 3], 2, 2, 64, 64, dict(window=249, relay=True, relay_top_k=3)),
    ([1000, 1777], [1, 30], 2, 2, 64, 64, dict(window=250, relay=True)),
]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("dtype,store", [(F16, "same"), (BF16, "same"), (F32, "same"), (F16, "e4m3"), (BF16, "e4m3"),
                                         (F16, "int8"), (BF16, "int8"), (F32, "int8"), (F32, "e4m3")])
def test_attention(case, dtype, store):
    lens, new, Hq, Hkv, D, page, kw = CASES[case]
    s = Setup(lens, Hkv, D, dtype, store, page, seed=case)
    q = (1.5 * torch.randn(sum(new), Hq, D, generator=s.g)).to(dtype)
    got = run(s, q, new, max_query_len=max(new), max_seqlen=max(lens), **kw)
    okw = dict(window=kw.get("window"), relay=kw.get("relay"), top_k=kw.get("relay_top_k", 2))
    check(got, *s.expect(q, new, **okw), dtype)
    # bounds left to their defaults: other pieces of work, results within the same bounds
    check(run(s, q, new, **kw), *s.expect(q, new, **okw), dtype)


@pytest.mark.parametrize("dtype,store", [(BF16, "same"), (F16, "e4m3"), (F32, "same")])
def test_batch_form_equals_packed_form(dtype, store):
    s = Setup([300, 90, 2200], 2, 64, dtype, store)
    for m in (1, 4, 20):
        q = torch.randn(3 * m, 4, 64, generator=s.g).to(dtype)
        packed = run(s, q, [m] * 3, max_query_len=m)
        qb = q.to(DEV).view(3, m, 4, 64).transpose(1, 2)
        with torch.no_grad():
            o = cra.cron_root_attention_paged(qb, s.cache, s.dtable, s.ints(s.lens))
        assert torch.equal(o.transpose(1, 2).reshape(3 * m, 4, 64), packed)


def test_chunk_equals_rows_of_the_whole_sequence():
    """A chunk over the cache against cron_root_attention over the sequence: the same pattern, chosen rows included."""
    for S, m, D in ((5000, 700, 128), (3001, 64, 64), (1000, 1000, 64)):
        g = torch.Generator().manual_seed(S)
        q, k, v = (torch.randn(1, H, S, D, generator=g).half().to(DEV) for H in (8, 2, 2))
        want = cra.cron_root_attention(q, k, v, kv_groups=4)[:, :, S - m:]
        cache = cra.PagedKVCache(S // 64 + 1, 2, D, 64, F16, device=DEV)
        table = torch.randperm(S // 64 + 1, device=DEV).int()[None]
        lens = torch.tensor([S], dtype=torch.int32, device=DEV)
        cache.write(k, v, table, lens)
        got = cra.cron_root_attention_paged(q[:, :, S - m:], cache, table, lens)
        # both within their bounds of the exact result: 2 x (eps + 2^-14) sum p|v|, |v| averages below 1
        assert float((got.float() - want.float()).abs().max()) <= 2 * (2 ** -10 + 2 ** -14) * 1.5


def test_steps_with_one_plan_equal_one_pass():
    """Chunks and single tokens with a fixed window and relay give the rows of the pass over the whole sequence."""
    S, D, W = 2400, 64, 49
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(1, H, S, D, generator=g).bfloat16().to(DEV) for H in (4, 2, 2))
    from cron_root_attention.core import _attention_with_plan
    want = _attention_with_plan(q, k, v, W, True, kv_groups=2)
    cache = cra.PagedKVCache(40, 2, D, 64, BF16, device=DEV)
    table = torch.randperm(40, device=DEV).int()[None, :38]
    got, at = [], 0
    for m in (1000, 1, 1, 700, 13, 680, 1, 4):
        lens = torch.tensor([at + m], dtype=torch.int32, device=DEV)
        sl = slice(at, at + m)
        cache.write(k[:, :, sl], v[:, :, sl], table, lens)
        got.append(cra.cron_root_attention_paged(q[:, :, sl], cache, table, lens, window=W, relay=True))
        at += m
    assert at == S
    assert float((torch.cat(got, 2).float() - want.float()).abs().max()) <= 2 * (2 ** -7 + 2 ** -14) * 1.5


@pytest.mark.parametrize("dtype,store", [(F16, "same"), (BF16, "same"), (F32, "same"), (BF16, "e4m3"), (F16, "int8")])
@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
def test_rows_that_a_query_does_not_see_do_not_reach_it(dtype, store, poison):
    """Later tokens of the chunk hold NaN or infinities in v, then in k: the queries before them are as without, those
    that see them get what they hold."""
    for Hq, new in ((2, 60), (2, 8), (1, 16)):
        s = Setup([200], 1, 64, dtype, store, seed=9)
        q = torch.randn(new, Hq, 64, generator=s.g).to(dtype)
        o, mag = s.expect(q, [new], window=1000)
        row, seen = 200 - new // 2, new // 2  # queries from `seen` on see the row
        s.v[row, 0, 3] = poison
        s.write(s.k, s.v, [200], [0, 200])
        got = run(s, q, [new], window=1000)
        check(got[:seen], o[:seen], mag[:seen], dtype)
        hit = got[seen:].float()
        if store == "same":
            assert (hit[..., 3].isnan() if math.isnan(poison) else hit[..., 3] == poison).all()
            keep = [c for c in range(64) if c != 3]
            check(got[seen:][..., keep], o[seen:][..., keep], mag[seen:][..., keep], dtype)
        else:
            assert hit.isnan().all()  # the row's scale is NaN
        s.k[row, 0, 5] = poison
        s.write(s.k, s.v, [200], [0, 200])
        check(run(s, q, [new], window=1000)[:seen], o[:seen], mag[:seen], dtype)


@pytest.mark.parametrize("store", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new", [1, 5, 40])
def test_rows_of_very_different_scales(dtype, store, new):
    """A v row of the largest fp16 values among ordinary ones, not seen, seen, and seen with a small weight."""
    for row, key in ((130, 0.0), (100, 0.0), (100, -9.0)):
        s = Setup([200], 1, 64, dtype, store, seed=new)
        q = torch.randn(new, 2, 64, generator=s.g).to(dtype)
        s.k[row, 0] = key * q[0, 0] / 4
        s.v[row, 0] = 60000 * torch.sign(s.v[row, 0].float()).to(dtype)
        s.write(s.k, s.v, [200], [0, 200])
        # below the window its multiples are seen: of 50 row 100 is one, of 64 row 130 is none
        window = 64 if row == 130 else 50
        check(run(s, q, [new], window=window), *s.expect(q, [new], window=window), dtype)


def test_lowest_values_and_large_scores():
    """Keys whose scores are the type's largest: the softmax stays finite."""
    s = Setup([100], 1, 64, BF16)
    s.k[:, 0] = 0
    s.k[40, 0, 0], s.k[60, 0, 0] = 1e4, -3e38
    s.write(s.k, s.v, [100], [0, 100])
    q = torch.zeros(4, 2, 64)
    q[:, :, 0] = 50.0
    got = run(s, q.bfloat16(), [4], window=1000)
    assert torch.equal(got.cpu(), s.v[40].expand(4, 2, 64))


def test_padding_rows_and_out():
    s = Setup([50, 60], 2, 64, F16)
    q = torch.randn(1, 4, 12, 64, device=DEV).half()
    cu = s.ints([2, 6, 9])  # two rows before, three behind the sequences
    out = torch.full_like(q, 7.0)
    got = cra.cron_root_attention_paged(q, s.cache, s.dtable, s.ints(s.lens), cu_seqlens=cu, out=out)
    assert got is out
    assert (out[:, :, :2] == 7).all() and (out[:, :, 9:] == 7).all() and out[:, :, 2:9].isfinite().all()
    fresh = cra.cron_root_attention_paged(q, s.cache, s.dtable, s.ints(s.lens), cu_seqlens=cu)
    assert torch.equal(fresh[:, :, 2:9], out[:, :, 2:9])
    assert not fresh[:, :, :2].any() and not fresh[:, :, 9:].any()
    # an out that the kernels cannot store to, and an odd head dim
    wide = torch.full((1, 4, 12, 65), 7.0, device=DEV).half()[..., 1:]
    cra.cron_root_attention_paged(q, s.cache, s.dtable, s.ints(s.lens), cu_seqlens=cu, out=wide)
    assert torch.equal(wide, out)
    o = Setup([50, 60], 2, 33, F16)
    q = torch.randn(1, 4, 12, 33, device=DEV).half()
    out = torch.full_like(q, 7.0)
    cra.cron_root_attention_paged(q, o.cache, o.dtable, o.ints(o.lens), cu_seqlens=cu, out=out)
    assert (out[:, :, :2] == 7).all() and (out[:, :, 9:] == 7).all() and out[:, :, 2:9].isfinite().all()


@pytest.mark.parametrize("dtype,store", [(F16, "same"), (BF16, "int8"), (F32, "same")])
def test_bad_pages_and_bounds_give_nan(dtype, store):
    for new in (1, 30):
        s = Setup([100, 2300, 120], 2, 64, dtype, store)
        q = torch.randn(3 * new, 4, 64, generator=s.g).to(dtype)
        good = run(s, q, [new] * 3)
        for entry in (-1, 1 << 30, s.cache.num_pages):
            s.dtable[1, 100] = entry  # rows 1600..1615: seen as strided or relay rows
            got = run(s, q, [new] * 3)
            assert got[new:2 * new].isnan().all()
            assert torch.equal(got[:new], good[:new]) and torch.equal(got[2 * new:], good[2 * new:])
        s.dtable.copy_(s.table)
        got = run(s, q, [new] * 3, max_seqlen=2299)
        assert got[new:2 * new].isnan().all() and torch.equal(got[:new], good[:new])
    # more new tokens than the bound says
    got = run(s, q, [new] * 3, max_query_len=2)
    assert got.isnan().all()


@pytest.mark.parametrize("dtype,store", [(BF16, "same"), (F32, "same"), (F16, "int8")])
def test_many_sequences(dtype, store):
    """More sequences than a wave's lanes: single tokens, chunks, and both with empty sequences between them."""
    g = random.Random(3)
    lens = [g.choice([0, 1, 5, 33, 130, 300]) for _ in range(150)]
    lens[77] = lens[130] = 2400
    for kind in ("single", "mixed"):
        new = [min(n, 1 if kind == "single" or b % 7 else g.randint(0, 30)) for b, n in enumerate(lens)]
        s = Setup(lens, 2, 32, dtype, store, seed=5)
        q = torch.randn(sum(new), 4, 32, generator=s.g).to(dtype)
        check(run(s, q, new, max_query_len=max(new)), *s.expect(q, new), dtype)


@pytest.mark.parametrize("dtype,store", [(F16, "same"), (BF16, "same"), (F32, "same"), (BF16, "e4m3"), (F16, "int8"),
                                         (F32, "int8")])
@pytest.mark.parametrize("D", [64, 256])
def test_chunks_behind_long_wide_contexts(dtype, store, D):
    """Few row tiles over thousands of keys each: their key ranges are cut into pieces and joined."""
    s = Setup([3000, 70, 2000], 2, D, dtype, store, seed=D)
    new = [40, 1, 90]
    q = (1.5 * torch.randn(sum(new), 4, D, generator=s.g)).to(dtype)
    for kw in (dict(window=1 << 30), dict(window=1900, relay=True), dict(window=3, relay=True, relay_top_k=4)):
        okw = dict(window=kw["window"], relay=kw.get("relay"), top_k=kw.get("relay_top_k", 2))
        good = run(s, q, new, max_seqlen=3000, **kw)
        check(good, *s.expect(q, new, **okw), dtype)
        assert torch.equal(run(s, q, new, max_seqlen=3000, **kw), good)
    # a page outside the cache among the first piece's keys
    s.dtable[0, 3] = -1
    got = run(s, q, new, window=1 << 30)
    assert got[:40].isnan().all() and not got[40:].isnan().any()


@pytest.mark.parametrize("dtype,store", [(F16, "same"), (BF16, "e4m3"), (F32, "same")])
@pytest.mark.parametrize("poison", [math.nan, math.inf])
def test_unseen_rows_of_cut_chunks(dtype, store, poison):
    """As above, with values that are not finite in rows that leave the window inside the chunk, and in the chunk."""
    n, m, W = 3000, 40, 2000
    s = Setup([n], 1, 64, dtype, store, seed=2)
    q = torch.randn(m, 2, 64, generator=s.g).to(dtype)
    o, mag = s.expect(q, [m], window=W, relay=False)
    first, last = n - m - W + 1, n - 10  # seen by the first query alone; by the last ten
    s.v[first, 0, 7] = s.v[last, 0, 7] = poison
    s.k[last, 0, 9] = poison
    s.write(s.k, s.v, [n], [0, n])
    got = run(s, q, [m], window=W, relay=False)
    mine = slice(1, m - 10)
    check(got[mine], o[mine], mag[mine], dtype)
    assert not got[0, :, 7].isfinite().any() and not got[m - 10:, :, 7].isfinite().any()


@pytest.mark.parametrize("dtype,store", [(BF16, "same"), (F32, "e4m3")])
def test_single_tokens_behind_long_wide_contexts(dtype, store):
    s = Setup([5000, 3, 2500], 2, 64, dtype, store, seed=8)
    q = torch.randn(3, 8, 64, generator=s.g).to(dtype)
    for kw in (dict(window=1 << 30), dict(window=2, relay=True, relay_top_k=1)):
        okw = dict(window=kw["window"], relay=kw.get("relay"), top_k=kw.get("relay_top_k", 2))
        check(run(s, q, [1] * 3, max_query_len=1, **kw), *s.expect(q, [1] * 3, **okw), dtype)


def test_repeated_pages():
    """Sequences that share their first pages, and a table that names one page twice."""
    s = Setup([64, 64], 1, 64, BF16)
    s.dtable[1, :2] = s.dtable[0, :2]
    s.k[64:96], s.v[64:96] = s.k[:32], s.v[:32]
    q = torch.randn(2, 2, 64, generator=s.g).bfloat16()
    check(run(s, q, [1, 1], window=64), *s.expect(q, [1, 1], window=64), BF16)
    s.dtable[1, 1] = s.dtable[1, 0]
    s.k[80:96], s.v[80:96] = s.k[64:80], s.v[64:80]
    check(run(s, q, [1, 1], window=64), *s.expect(q, [1, 1], window=64), BF16)


@pytest.mark.parametrize("window,top_k", [(None, 2), (46, 4), (600, 2), (600, 4), (150, 3), (300, 4)])
def test_equal_norms_take_the_earlier_row(window, top_k):
    s = Setup([2100], 1, 64, F16)
    s.k[:] = s.k.sign() * 0.5  # every row has the same norm, but for a few pairs
    s.k[50:52] *= 2
    s.k[700:703] *= 2
    s.k[1300], s.k[1350] = s.k[1300] * 4, s.k[1350] * 4
    s.write(s.k, s.v, [2100], [0, 2100])
    q = (8 * torch.randn(1, 1, 64, generator=s.g)).half()
    check(run(s, q, [1], window=window, relay=True, relay_top_k=top_k),
          *s.expect(q, [1], window=window, relay=True, top_k=top_k), F16)


def test_nan_norms_are_not_chosen():
    s = Setup([2100], 1, 64, F16)
    s.k[47:93] = math.nan  # one whole block of W = 46 and a row
    s.k[46] = 0.1
    s.write(s.k, s.v, [2100], [0, 2100])
    q = torch.randn(1, 1, 64, generator=s.g).half()
    # block 1 is rows 46..91: its first row is the only number; block 2 starts at row 92, which is NaN and strided
    got = run(s, q, [1])
    assert got.isnan().all()
    s.k[92] = 0.2
    s.write(s.k, s.v, [2100], [0, 2100])
    o, mag = s.expect(q, [1])
    assert o.isfinite().all()
    check(run(s, q, [1]), o, mag, F16)


@pytest.mark.parametrize("store", ["same", "e4m3"])
def test_a_cache_beyond_32_bits_of_bytes(store):
    """Rows whose byte offsets pass 2^32: pages at the end of a cache of 6 GB and more."""
    D, H, P = 128, 8, 64
    pages = 50000 if store == "same" else 100000
    cache = cra.PagedKVCache(pages, H, D, P, BF16, STORES[store], device=DEV)
    assert cache.k.numel() * cache.k.element_size() > 1 << 32
    s = Setup([300, 2100], 2, D, BF16, store, P)
    far = torch.arange(pages - s.table.shape[1] * 2, pages, device=DEV).int().view(2, -1)
    k = torch.randn(1, H, 2400, D, device=DEV).bfloat16()
    v = torch.randn(1, H, 2400, D, device=DEV).bfloat16()
    lens, cu = s.ints([300, 2100]), s.ints([0, 300, 2400])
    cache.write(k, v, far, lens, cu_seqlens=cu)
    near = cra.PagedKVCache(far.numel(), H, D, P, BF16, STORES[store], device=DEV)
    table = (far - far[0, 0]).contiguous()
    near.write(k, v, table, lens, cu_seqlens=cu)
    assert all(torch.equal(a, b) for a, b in zip(cache.read(far, lens), near.read(table, lens)))
    for m in (1, 40):
        q = torch.randn(2, 16, m, D, device=DEV).bfloat16()
        assert torch.equal(cra.cron_root_attention_paged(q, cache, far, lens),
                           cra.cron_root_attention_paged(q, near, table, lens))


def test_drawn_cases():
    """Sizes of no particular choice."""
    rng = random.Random(5)
    for i in range(24):
        D = rng.choice([16, 32, 40, 64, 72, 112, 128, 200, 256])
        Hkv = rng.choice([1, 2, 3])
        Hq = Hkv * rng.choice([1, 2, 5, 8, 17])
        dtype, store = rng.choice([F16, BF16, F32]), rng.choice(["same", "e4m3", "int8"])
        lens = [rng.choice([rng.randint(1, 80), rng.randint(1, 2600)]) for _ in range(rng.randint(1, 5))]
        new = [rng.choice([1, 1, min(n, rng.randint(1, 40)), min(n, rng.randint(1, 300))]) for n in lens]
        new = [m if m * Hq < 3000 else 1 for m in new]
        kw = rng.choice([{}, {}, dict(window=rng.randint(1, 300)), dict(window=5000),
                         dict(window=rng.randint(1, 300), relay=True)])
        s = Setup(lens, Hkv, D, dtype, store, rng.choice([16, 32, 256]), seed=i, table_extra=rng.randint(0, 3))
        q = (1.5 * torch.randn(sum(new), Hq, D, generator=s.g)).to(dtype)
        print("case", i, lens, new, Hq, Hkv, D, dtype, store, kw, flush=True)
        got = run(s, q, new, max_query_len=max(new), **kw)
        check(got, *s.expect(q, new, **kw), dtype)


def test_same_results_every_time_and_on_other_streams():
    s = Setup([3000, 500, 2222], 2, 128, BF16, "e4m3", seed=3)
    q = torch.randn(90, 8, 128, generator=s.g).bfloat16()
    for new in ([1, 1, 1], [30, 30, 30]):
        first = run(s, q[:sum(new)], new)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        others = []
        with torch.cuda.stream(side):
            for _ in range(3):
                others.append(run(s, q[:sum(new)], new))
        main = [run(s, q[:sum(new)], new) for _ in range(3)]  # at the same time
        torch.cuda.synchronize()
        assert all(torch.equal(first, x) for x in others + main)


def test_captured_step_serves_growing_sequences():
    """One captured decoding step (write + attention): replays read lengths, tables and tokens anew."""
    D, H, Hq, N_ = 64, 2, 8, 3
    start = [2046, 100, 31]
    s = Setup(start, H, D, F16, page=16, spare=12, table_extra=2)
    free = sorted(set(range(s.cache.num_pages)) - set(s.table.flatten().tolist()))
    table = s.table.clone()
    for b, n in enumerate(start):  # room for the tokens to come
        for j in range(-(-n // 16), -(-(n + 6) // 16)):
            table[b, j] = free.pop()
    table = table.to(DEV)
    lens = s.ints(start)
    k, v, q = (torch.zeros(N_, h, 1, D, device=DEV).half() for h in (H, H, Hq))

    def step(cache):
        cache.write(k, v, table, lens)
        return cra.cron_root_attention_paged(q, cache, table, lens)
    twin = cra.PagedKVCache.from_tensors(s.cache.k.clone(), s.cache.v.clone(), s.cache.k_norm.clone())
    warm = cra.PagedKVCache.from_tensors(s.cache.k.clone(), s.cache.v.clone(), s.cache.k_norm.clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step(s.cache)
    for i in range(5):
        lens.add_(1)
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        got = o.clone()
        assert torch.equal(got, step(twin)), i
        assert torch.equal(s.cache.k.nan_to_num(-9), twin.k.nan_to_num(-9)), i


def test_empty_calls():
    cache = cra.PagedKVCache(4, 2, 64, 16, F16, device=DEV)
    none = torch.zeros(0, 4, dtype=torch.int32, device=DEV)
    lens = torch.zeros(0, dtype=torch.int32, device=DEV)
    q = torch.zeros(0, 4, 1, 64, device=DEV).half()
    assert cra.cron_root_attention_paged(q, cache, none, lens).shape == q.shape
    k = torch.zeros(0, 2, 1, 64, device=DEV).half()
    cache.write(k, k, none, lens)
    assert cache.read(none, lens)[0].shape == (0, 2, 64, 64)
    one, l1 = torch.zeros(1, 4, dtype=torch.int32, device=DEV), torch.tensor([3], dtype=torch.int32, device=DEV)
    q = torch.zeros(1, 4, 0, 64, device=DEV).half()
    assert cra.cron_root_attention_paged(q, cache, one, l1).shape == q.shape
    assert cache.read(one, l1, 0)[0].shape == (1, 2, 0, 64)
    # a sequence of length 0 with a new token: its query sees nothing
    q = torch.ones(1, 4, 1, 64, device=DEV).half()
    assert not cra.cron_root_attention_paged(q, cache, one, l1 * 0).any()


def test_refusals_on_the_gpu():
    cache = cra.PagedKVCache(4, 2, 64, 16, F16, device=DEV)
    table = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    lens = torch.ones(2, dtype=torch.int32, device=DEV)
    q = torch.zeros(2, 4, 1, 64, device=DEV).half()
    f = cra.cron_root_attention_paged
    for bad in (lambda: f(q[:1], cache, table, lens), lambda: f(q[:, :3], cache, table, lens),
                lambda: f(q[..., :32], cache, table, lens), lambda: f(q[0], cache, table, lens),
                lambda: f(q, cache, table.cpu(), lens), lambda: f(q, cache, table, lens[:1]),
                lambda: f(q, cache, table.t().contiguous().t(), lens),
                lambda: f(q, cache, table, lens, window=0), lambda: f(q, cache, table, lens, relay_top_k=5),
                lambda: f(q, cache, table, lens, max_seqlen=0), lambda: f(q, cache, table, lens, max_query_len=0),
                lambda: f(q, cache, table, lens, cu_seqlens=lens), lambda: f(q, cache, table, lens, out=q[:, :, :, :32]),
                lambda: f(q, cache, table, lens, cu_seqlens=torch.zeros(3, dtype=torch.int32, device=DEV)),
                lambda: cache.write(q, q, table, lens), lambda: cache.write(q[:, :2], q[:, :1], table, lens),
                lambda: cache.read(table, lens, -1)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: f(q.float(), cache, table, lens), lambda: f(q, cache, table.long(), lens),
                lambda: f(q, cache, table, lens.long()), lambda: f(q, cache, table, lens, cu_seqlens=lens.float()),
                lambda: cache.write(q[:, :2], q[:, :2].float(), table, lens)):
        with pytest.raises(TypeError):
            bad()
    r = q.clone().requires_grad_(True)
    with pytest.raises(NotImplementedError):
        f(r, cache, table, lens)
    with pytest.raises(NotImplementedError):
        cache.write(r[:, :2], r[:, :2], table, lens)
    with torch.no_grad():
        f(r, cache, table, lens)
    half = torch.zeros(4, 2, 16, 64, device=DEV).half()
    norm = torch.zeros(4, 2, 16, device=DEV)
    with pytest.raises(ValueError, match="contiguous"):
        cra.PagedKVCache.from_tensors(half.transpose(0, 2).contiguous().transpose(0, 2), half, norm)
    with pytest.raises(RuntimeError):
        cra.PagedKVCache.from_tensors(half, half, norm.cpu())


@pytest.mark.parametrize("path", ["op", "function"])
def test_tangents_are_refused(path, monkeypatch):
    """Nothing of the paged path has derivatives: dual tensors raise, as those that require a gradient do."""
    from torch.autograd import forward_ad
    if path == "function":
        monkeypatch.setattr(cra.paged._native, "fast_op", lambda name: None)
    s = Setup([20], 2, 64, F16)
    q, k = (torch.randn(1, H, 1, 64, device=DEV).half() for H in (4, 2))
    lens = s.ints(s.lens)
    before = s.cache.k.clone()
    with forward_ad.dual_level(), torch.no_grad():
        dq, dk = (forward_ad.make_dual(x, torch.ones_like(x)) for x in (q, k))
        with pytest.raises(NotImplementedError):
            cra.cron_root_attention_paged(dq, s.cache, s.dtable, lens)
        for kk, vv in ((dk, k), (k, dk)):
            with pytest.raises(NotImplementedError):
                s.cache.write(kk, vv, s.dtable, lens)
        cra.cron_root_attention_paged(q, s.cache, s.dtable, lens)  # without a tangent
    assert torch.equal(s.cache.k.nan_to_num(-9), before.nan_to_num(-9))


@pytest.mark.parametrize("store", ["same", "e4m3", "int8"])
def test_write_of_sequences_that_outgrew_their_table(store):
    """Tokens behind what a row of the table holds are passed over; those before them go to their own rows."""
    D, H, room = 64, 2, 64
    s = Setup([room, room], H, D, F16, store, page=16)
    tensors = [t for t in (s.cache.k, s.cache.v, s.cache.k_norm, s.cache.k_scale, s.cache.v_scale) if t is not None]
    before = [t.clone() for t in tensors]
    x = torch.randn(2, H, 6, D, device=DEV).half()
    packed = x.transpose(0, 1).reshape(1, H, 12, D)

    def same():
        return all(torch.equal(a.float().nan_to_num(-9), b.float().nan_to_num(-9)) for a, b in zip(before, tensors))
    # every new token behind the table's last row
    for lens in ([room + 6, room + 1000], [2**31 - 1, room + 6]):
        s.cache.write(x, x, s.dtable, s.ints(lens))
        s.cache.write(packed, packed, s.dtable, s.ints(lens), cu_seqlens=s.ints([0, 6, 12]))
        assert same(), lens
    # rows 60 .. 63 are the first four of six new tokens; the other sequence's are its last six
    twin = Setup([room, room], H, D, F16, store, page=16)
    want = torch.zeros(1, H, 10, D, device=DEV).half()
    want[0, :, :4], want[0, :, 4:] = x[0, :, :4], x[1]
    twin.cache.write(want, want, twin.dtable, s.ints([room, room]), cu_seqlens=s.ints([0, 4, 10]))
    s.cache.write(x, x, s.dtable, s.ints([room + 2, room]))
    for a, b in zip(s.cache.read(s.dtable, s.ints([room, room])), twin.cache.read(twin.dtable, s.ints([room, room]))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,store", [(F16, "same"), (BF16, "same"), (F32, "same"), (F16, "e4m3"), (BF16, "int8"),
                                         (F32, "int8")])
@pytest.mark.parametrize("poison,D", [(math.inf, 64), (-math.inf, 64), (math.nan, 64), (math.inf, 256), (math.inf, 40),
                                      (math.nan, 128)])
def test_values_that_are_not_finite_in_rows_that_are_seen(dtype, store, poison, D):
    """What a seen row of v holds reaches the query, its weight however small: in the last row of a tile cut short
    (n = 200: 200 keys, or 15 of the window and 13 strided ones), in whole tiles, for one new token and for more."""
    for n, new, window, row, low in ((200, 1, 1000, 199, False), (200, 1, 1000, 40, True), (224, 1, 1000, 223, False),
                                     (200, 1, None, 199, False), (200, 1, None, 180, False), (200, 4, 1000, 40, True),
                                     (200, 40, 1000, 40, True), (3000, 1, 3000, 2999, False), (3000, 1, 3000, 500, True)):
        s = Setup([n], 1, D, dtype, store, seed=n + new)
        q = torch.randn(new, 1, D, generator=s.g).to(dtype)
        q[:] = q[0]
        if low:  # a weight of about exp(-30): nothing of it is left in fp16
            s.k[row, 0] = (-30 * math.sqrt(D) * q[0, 0].double() / q[0, 0].double().square().sum()).to(dtype)
        o, mag = s.expect(q, [new], window=window)
        s.v[row, 0, 3] = poison
        s.write(s.k, s.v, [n], [0, n])
        got = run(s, q, [new], window=window)
        if store == "same":
            hit = got[..., 3].float()
            assert (hit.isnan() if math.isnan(poison) else hit == poison).all(), (n, new, window, row)
            keep = [c for c in range(D) if c != 3]
            check(got[..., keep], o[..., keep], mag[..., keep], dtype)
        else:
            assert got.isnan().all()  # the row's scale is NaN


@pytest.mark.parametrize("packed", [False, True])
def test_contiguous_rows_at_odd_addresses(packed):
    """q, k, v and out that are contiguous but start between 16-byte addresses are copied, not refused."""
    def odd(x):
        y = torch.zeros(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape)
        y.copy_(x)
        assert y.is_contiguous() and y.data_ptr() % 16
        return y
    s = Setup([40], 2, 64, F16)
    lens, cu = s.ints([40]), s.ints([0, 3]) if packed else None
    q, k, v = (torch.randn(1, H, 3, 64, device=DEV).half() for H in (4, 2, 2))
    s.cache.write(odd(k), odd(v), s.dtable, lens, cu_seqlens=cu)
    for x, y in zip(s.cache.read(s.dtable, lens, 40), (k, v)):
        assert torch.equal(x[:, :, 37:], y)
    want = cra.cron_root_attention_paged(q, s.cache, s.dtable, lens, cu_seqlens=cu)
    assert torch.equal(cra.cron_root_attention_paged(odd(q), s.cache, s.dtable, lens, cu_seqlens=cu), want)
    out = odd(torch.zeros_like(q))
    cra.cron_root_attention_paged(q, s.cache, s.dtable, lens, cu_seqlens=cu, out=out)
    assert torch.equal(out, want)


def test_table_without_pages():
    """Pages of no sequence: an empty one gives zeros, one with rows is longer than its table (NaN); rows of out outside
    every sequence stay; nothing is written."""
    cache = cra.PagedKVCache(4, 2, 64, 16, F16, device=DEV)
    none = torch.zeros(2, 0, dtype=torch.int32, device=DEV)
    lens = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
    q = torch.ones(2, 4, 2, 64, device=DEV).half()
    o = cra.cron_root_attention_paged(q, cache, none, lens)
    assert not o[0].any() and o[1].isnan().all()
    out = torch.full((1, 4, 6, 64), 7.0, device=DEV).half()
    cu = torch.tensor([1, 3, 5], dtype=torch.int32, device=DEV)
    cra.cron_root_attention_paged(out.clone(), cache, none, lens, cu_seqlens=cu, out=out)
    assert (out[:, :, [0, 5]] == 7).all() and not out[:, :, 1:3].any() and out[:, :, 3:5].isnan().all()
    cache.write(q[:, :2], q[:, :2], none, lens)
    assert not cache.k.any() and not cache.k_norm.any()
    assert cache.read(none, lens)[0].shape == (2, 2, 0, 64) and not cache.read(none, lens, 5)[0].any()


@pytest.mark.parametrize("dtype,store", [(F16, "same"), (BF16, "int8"), (F32, "same")])
def test_captured_mixed_step_replays_over_other_batches(dtype, store):
    """One captured packed step (write + attention): replays take chunks, single tokens, empty sequences and padding
    from the offsets, lengths and tables that are there then."""
    D, H, Hq, T, N_ = 64, 2, 4, 200, 4
    caches = [cra.PagedKVCache(4 * 160, H, D, 16, dtype, STORES[store], device=DEV) for _ in range(2)]
    table = torch.randperm(4 * 160, device=DEV).int().view(N_, 160)
    lens, cu = torch.zeros(N_, dtype=torch.int32, device=DEV), torch.zeros(N_ + 1, dtype=torch.int32, device=DEV)
    k, v, q = (torch.zeros(1, h, T, D, device=DEV, dtype=dtype) for h in (H, H, Hq))
    g = torch.Generator(device=DEV).manual_seed(4)
    for c in caches:  # the same old rows in both
        x = torch.randn(N_, H, 2500, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(dtype)
        c.write(x, x.flip(1), table, lens + 2500)

    def step(cache):
        cache.write(k, v, table, lens, cu_seqlens=cu)
        return cra.cron_root_attention_paged(q, cache, table, lens, cu_seqlens=cu)
    warm = cra.PagedKVCache(4 * 160, H, D, 16, dtype, STORES[store], device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step(caches[0])
    for offsets, lengths in (([0, 1, 2, 3, 4], [2500, 1, 2049, 17]), ([0, 100, 100, 190, 200], [2400, 0, 90, 2048]),
                             ([5, 30, 31, 31, 150], [2501, 40, 7, 119]), ([200, 200, 200, 200, 200], [9, 9, 9, 9]),
                             ([0, 0, 0, 0, 200], [1, 2, 3, 2300]), ([0, 1, 2, 3, 4], [2500, 1, 2049, 17])):
        cu.copy_(torch.tensor(offsets)), lens.copy_(torch.tensor(lengths))
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, device=DEV, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = o.clone()
        want = step(caches[1])
        assert want[:, :, offsets[0]:offsets[-1]].isfinite().all() and torch.equal(got, want), offsets
