"""Attention of sequences that share a prefix, on the GPU: against the 64-bit oracle of the
attention over whole sequences, with its tolerance (the same roundings; a sequence's two
parts are joined in fp32, which adds a few units of 2^-24 to sums of |p v|).
"""
import math

import pytest
import torch

import cron_root_attention as cra
from paged_util import STORES, attend, norm_sq, quantise

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
DENSE = 1 << 20


class Shared:
    """Sequences of P common rows and own[b] behind them, in a cache that is filled through write()."""

    def __init__(self, P, own, Hkv, D, dtype, store="same", page=16, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.g, self.P, self.own, self.Hkv, self.D, self.dtype, self.store = g, P, list(own), Hkv, D, dtype, store
        self.lens = [P + n for n in own]
        whole, most = P // page, -(-(P % page + max(own + [0])) // page)
        pool = whole + most * len(own) + 3
        order = torch.randperm(pool, generator=g).to(torch.int32)
        table = torch.empty(len(own), whole + most, dtype=torch.int32)
        table[:, :whole] = order[:whole]
        table[:, whole:] = order[whole:whole + most * len(own)].view(len(own), most)
        self.cache = cra.PagedKVCache(pool, Hkv, D, page, dtype, STORES[store], device=DEV)
        self.cache.k_norm.fill_(math.nan)
        if store == "same":
            self.cache.k.fill_(math.nan), self.cache.v.fill_(math.nan)
        else:
            self.cache.k_scale.fill_(math.nan), self.cache.v_scale.fill_(math.nan)
        self.k, self.v = ([torch.randn(P, Hkv, D, generator=g).to(dtype)] +
                          [torch.randn(n, Hkv, D, generator=g).to(dtype) for n in own] for _ in "kv")
        self.table = table.to(DEV)
        self.write()

    def write(self):
        for b in range(len(self.own)):  # the prefix's rows are written again, the same
            k, v = (torch.cat([x[0], x[1 + b]]).to(DEV).transpose(0, 1)[None] for x in (self.k, self.v))
            if k.shape[2]:
                self.cache.write(k, v, self.table[b:b + 1], self.ints([self.lens[b]]), self.ints([0, self.lens[b]]))

    @staticmethod
    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=DEV)

    def prefix(self, P=None):
        P = self.P if P is None else P
        return cra.SharedPrefix(self.table[0, :-(-P // self.cache.page_size)].contiguous(), self.ints([P]))

    def expect(self, q, new, window, relay=None, top_k=2):
        T, Hq, D = q.shape
        g = Hq // self.Hkv
        o, mag = (torch.zeros(T, Hq, D, dtype=torch.float64) for _ in "om")
        st, at = STORES[self.store], 0
        for b, (n, m) in enumerate(zip(self.lens, new)):
            for h in range(self.Hkv if m else 0):
                k, v = (torch.cat([x[0], x[1 + b]])[:, h] for x in (self.k, self.v))
                qq = q[at:at + m, h * g:(h + 1) * g].transpose(0, 1)
                x, y = attend(qq, quantise(k, st)[2], quantise(v, st)[2], norm_sq(k), n, m, window, relay, top_k)
                o[at:at + m, h * g:(h + 1) * g] = x.transpose(0, 1)
                mag[at:at + m, h * g:(h + 1) * g] = y.transpose(0, 1)
            at += m
        return o, mag

    def run(self, q, new, packed=True, prefix=None, **kw):
        cu = [0]
        for m in new:
            cu.append(cu[-1] + m)
        with torch.no_grad():
            if not packed:
                y = cra.cron_root_attention_paged(q.to(DEV).view(len(new), new[0], *q.shape[1:]).transpose(1, 2), self.cache,
                                                  self.table, self.ints(self.lens), prefix=prefix or self.prefix(), **kw)
                return y.transpose(1, 2).flatten(0, 1)
            y = cra.cron_root_attention_paged(q.to(DEV)[None].transpose(1, 2), self.cache, self.table, self.ints(self.lens),
                                              self.ints(cu), prefix=prefix or self.prefix(), **kw)
        return y[0].transpose(0, 1)

    def q(self, new, Hq):
        return (torch.randn(sum(new), Hq, self.D, generator=self.g) * 1.5).to(self.dtype)


def check(got, o, mag, dtype):
    eps = torch.finfo(dtype).eps
    tol = (eps + (2.0 ** -17 if dtype == F32 else 2.0 ** -14)) * mag + eps / 2 * o.abs() + torch.finfo(dtype).tiny
    off = (got.double().cpu() - o).abs() - tol
    assert bool((off <= 0).all()), f"{int((~(off <= 0)).sum())} elements off, worst by {float(off.max()):.3e}"


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("store", ["same", "e4m3", "int8"])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 64), (80, 32), (256, 16), (32, 128)])
@pytest.mark.parametrize("window", [DENSE, 40])
def test_types_stores_and_widths(dtype, store, D, page, window):
    s = Shared(16 * page if page < 100 else 400, [1, 7, 64, 100, 3], 2, D, dtype, store, page, seed=D)
    new = [1] * 5
    q = s.q(new, 6)
    check(s.run(q, new, window=window, relay=True), *s.expect(q, new, window, True), dtype)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (8, 8), (16, 1), (10, 2), (32, 1), (40, 8)])
@pytest.mark.parametrize("M", [1, 2, 5])
def test_heads_and_drafted_tokens(Hq, Hkv, M):
    """Up to 16 rows a kv head share; above, the sequences attend by themselves."""
    s = Shared(300, [M, M + 9, 33, 70], Hkv, 64, BF16, "same", 16, seed=Hq + M)
    new = [M] * 4
    q = s.q(new, Hq)
    for window in (DENSE, 50):
        o = s.expect(q, new, window)
        check(s.run(q, new, window=window), *o, BF16)
        check(s.run(q, new, packed=False, window=window), *o, BF16)


@pytest.mark.parametrize("P", [1, 15, 16, 17, 63, 64, 65, 500, 2049, 2500])
@pytest.mark.parametrize("window", [DENSE, 1, 7, 64, 600])
def test_lengths_and_windows(P, window):
    s = Shared(P, [1, 2, 40, 90, 700], 2, 64, F16, "same", 16, seed=P)
    new = [1, 2, 1, 3, 1]
    q = s.q(new, 4)
    check(s.run(q, new, window=window), *s.expect(q, new, window), F16)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("top_k", [1, 3, 4])
def test_relay_rows_of_blocks_that_the_prefix_cuts(dtype, top_k):
    """Sequences far longer than the prefix, whose last block is cut anywhere."""
    for P in (96, 100, 127):
        s = Shared(P, [1, 60, 200, 333], 2, 32, dtype, "same", 32, seed=P)
        new = [1, 1, 2, 1]
        q = s.q(new, 4)
        check(s.run(q, new, window=32, relay=True, relay_top_k=top_k), *s.expect(q, new, 32, True, top_k), dtype)
        check(s.run(q, new, window=32, relay=False), *s.expect(q, new, 32, False), dtype)


def test_many_sequences_and_row_tiles():
    own = [1 + (i * 37) % 50 for i in range(150)]
    s = Shared(200, own, 1, 64, BF16, "same", 16, seed=1)
    new = [1 + i % 2 for i in range(150)]
    new = [min(a, b) for a, b in zip(new, own)]
    q = s.q(new, 8)
    for window in (DENSE, 30):
        check(s.run(q, new, window=window, max_query_len=2), *s.expect(q, new, window), BF16)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_mixed_batch(dtype):
    """Sequences without new tokens, in a long chunk, with new tokens among the prefix's rows,
    and shorter than the prefix, beside ones that share."""
    s = Shared(200, [1, 5, 100, 40, 30, 2], 2, 64, dtype, "same", 16, seed=3)
    new = [1, 0, 60, 100, 2, 1]
    q = s.q(new, 4)
    for window in (DENSE, 48):
        check(s.run(q, new, window=window), *s.expect(q, new, window), dtype)
    s.lens[5] = 150  # shorter than the prefix
    s.k[6], s.v[6] = s.k[6][:0], s.v[6][:0]
    k0, v0 = s.k[0], s.v[0]
    cases = s.expect(q[:-1], new[:-1] + [0], 48)
    got = s.run(q, new, window=48)
    check(got[:-1], *cases, dtype)
    s.k[0], s.v[0] = k0[:150], v0[:150]
    check(got[-1:], *s.expect(q[-1:], [0] * 5 + [1], 48), dtype)


def test_any_common_length_gives_the_same():
    """A shorter prefix, none, one beyond its table, a negative one."""
    s = Shared(320, [1, 90, 20], 2, 64, BF16, "same", 16, seed=5)
    new = [1, 2, 1]
    q = s.q(new, 4)
    o = s.expect(q, new, 64)
    for P in (320, 319, 64, 1):
        check(s.run(q, new, window=64, prefix=s.prefix(P)), *o, BF16)
    for n in (0, -5, 10 ** 9):
        check(s.run(q, new, window=64, prefix=cra.SharedPrefix(s.table[0, :20].contiguous(), s.ints([n]))), *o, BF16)
    check(s.run(q, new, window=64, prefix=cra.SharedPrefix(s.table[0, :0], s.ints([7]))), *o, BF16)


def test_padding_and_out():
    s = Shared(100, [4, 9], 2, 64, F16, "same", 16)
    q = s.q([1, 1], 4)
    rows = torch.full((1, 4, 5, 64), 3.0, dtype=F16, device=DEV)
    rows[:, :, 1:3] = q.to(DEV).transpose(0, 1)
    cu = s.ints([1, 2, 3])
    want = s.run(q, [1, 1], window=DENSE)
    with torch.no_grad():
        y = cra.cron_root_attention_paged(rows, s.cache, s.table, s.ints(s.lens), cu, window=DENSE, prefix=s.prefix())
        assert torch.equal(y[0, :, 1:3].transpose(0, 1), want) and y[0, :, 0].abs().max() == 0 and y[0, :, 3:].abs().max() == 0
        out = torch.full_like(rows, 7.0)
        z = cra.cron_root_attention_paged(rows, s.cache, s.table, s.ints(s.lens), cu, window=DENSE, prefix=s.prefix(), out=out)
        assert z is out and torch.equal(out[0, :, 1:3], y[0, :, 1:3])
        assert bool((out[0, :, 0] == 7).all()) and bool((out[0, :, 3:] == 7).all())
        odd = torch.zeros(1, 4, 5, 65, dtype=F16, device=DEV)[..., 1:]
        odd.copy_(rows)
        assert torch.equal(cra.cron_root_attention_paged(odd, s.cache, s.table, s.ints(s.lens), cu, window=DENSE,
                                                         prefix=s.prefix()), y)


@pytest.mark.parametrize("dtype,store", [(F16, "same"), (BF16, "same"), (F32, "same"), (BF16, "e4m3")])
def test_what_is_not_finite_reaches_who_sees_it(dtype, store):
    """Infinities and NaN in rows of the prefix: dense, all see them; under a window, who does."""
    P = 200
    s = Shared(P, [1, 30, 90, 400], 1, 64, dtype, store, 16, seed=8)
    new = [1] * 4
    q = s.q(new, 2)
    clean = s.run(q, new, window=64, relay=False)
    s.v[0][150, 0, 3] = math.inf
    s.v[0][151, 0, 4] = math.nan
    s.write()
    y = s.run(q, new, window=64, relay=False).float()
    # rows 150, 151 are in the windows of positions up to 150 + 63: the first one's and no other's; no block starts there
    assert torch.equal(y[1:], clean[1:].float()) or float((y[1:] - clean[1:].float()).abs().max()) < 1e-2
    assert bool(y[1:].isfinite().all())
    if store == "same":
        assert bool((y[0, :, 3] == math.inf).all()) and bool(y[0, :, 4].isnan().all())
        assert bool(y[0, :, :3].isfinite().all())
        y = s.run(q, new, window=DENSE).float()
        assert bool((y[:, :, 3] == math.inf).all()) and bool(y[:, :, 4].isnan().all()) and bool(y[:, :, :3].isfinite().all())
    else:
        assert bool(y[0].isnan().any())


def test_pages_outside_the_cache():
    s = Shared(160, [1, 20, 33], 2, 64, BF16, "same", 16)
    new = [1, 1, 1]
    q = s.q(new, 4)
    x = s.prefix()
    x.page_table[3] = 10 ** 6
    assert bool(s.run(q, new, window=DENSE, prefix=x).isnan().all())
    # the sequences' own tables are not looked at for the prefix's rows
    s.table[:, :10] = -1
    want = s.expect(q, new, DENSE)
    x = cra.SharedPrefix(s.ints([0] * 10), s.ints([160]))
    x.page_table.copy_(x.page_table)  # any valid pages: only finiteness is looked at
    s.cache.k.nan_to_num_(0.0), s.cache.v.nan_to_num_(0.0)
    assert bool(s.run(q, new, window=DENSE, prefix=x).isfinite().all()) and want[0].isfinite().all()


def test_captured_step_replays_over_growing_sequences():
    s = Shared(128, [40, 60, 20], 2, 64, F16, "same", 16, seed=2)
    lens, x = s.ints([128 + 5, 128 + 30, 128 + 1]), s.prefix()
    q = torch.randn(3, 4, 1, 64, device=DEV, dtype=F16)

    def step():
        return cra.cron_root_attention_paged(q, s.cache, s.table, lens, window=50, prefix=x, relay=True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(stream):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y = step()
    torch.cuda.current_stream().wait_stream(stream)
    with torch.no_grad():
        for P in (128, 100, 0, 128):
            lens += 3
            x.length.fill_(P)
            q.copy_(torch.randn_like(q))
            graph.replay()
            want = step()
            torch.cuda.synchronize()
            assert torch.equal(y, want), P
            plain = cra.cron_root_attention_paged(q, s.cache, s.table, lens, window=50, relay=True)
            assert float((y.float() - plain.float()).abs().max()) < 4e-3


def test_runs_agree_bit_for_bit():
    s = Shared(1000, [1 + 13 * i for i in range(20)], 4, 128, BF16, "same", 16)
    q = s.q([1] * 20, 8)
    first = s.run(q, [1] * 20, window=DENSE)
    for _ in range(4):
        assert torch.equal(s.run(q, [1] * 20, window=DENSE), first)


def test_two_streams_at_once():
    work = []
    for seed, (P, own) in enumerate([(700, [3 + 11 * i for i in range(30)]), (2500, [40 + i for i in range(17)])]):
        s = Shared(P, own, 2, 64, F16, "same", 16, seed=seed)
        q = s.q([1] * len(own), 8)
        work.append((s, q, s.run(q, [1] * len(own), window=DENSE), torch.cuda.Stream()))
    torch.cuda.synchronize()
    results = []
    for _ in range(10):
        for s, q, _, stream in work:
            with torch.cuda.stream(stream):
                results.append(s.run(q, [1] * len(s.own), window=DENSE))
    torch.cuda.synchronize()
    for i, y in enumerate(results):
        assert torch.equal(y, work[i % 2][2])


def test_two_graphs_of_one_pool():
    a, b = Shared(300, [5, 90, 33], 2, 64, BF16, "e4m3", 16, seed=1), Shared(2300, [50, 4], 2, 64, BF16, "e4m3", 16, seed=2)
    stream, graphs, pool = torch.cuda.Stream(), [], None
    stream.wait_stream(torch.cuda.current_stream())
    for s in (a, b):
        q, x, lens = s.q([1] * len(s.own), 4).to(DEV)[:, :, None], s.prefix(), s.ints(s.lens)
        run = lambda: cra.cron_root_attention_paged(q, s.cache, s.table, lens, window=60, prefix=x)
        with torch.no_grad(), torch.cuda.stream(stream):
            want = run().clone()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, pool=pool, stream=stream):
                y = run()
            pool = pool or g.pool()
        graphs.append((g, y, want, q, x, lens))
    torch.cuda.current_stream().wait_stream(stream)
    for i in (0, 1, 1, 0, 1, 0):
        g, y, want = graphs[i][:3]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_lengths_that_do_not_fit():
    """Sequences longer than the bound are NaN, empty and shorter ones than the prefix their own."""
    s = Shared(200, [0, 30, 300, 7], 2, 64, F16, "same", 16)
    s.lens = [0, 230, 500, 120]
    q = s.q([1] * 4, 4)
    want = cra.cron_root_attention_paged(q.to(DEV)[:, :, None], s.cache, s.table, s.ints(s.lens), window=64, max_seqlen=250)
    for x in (s.prefix(), s.prefix(150), cra.SharedPrefix(s.prefix().page_table, s.ints([-3])),
              cra.SharedPrefix(s.table[0, :4].contiguous(), s.ints([1000]))):
        got = s.run(q, [1] * 4, packed=False, prefix=x, window=64, max_seqlen=250)
        assert got[2].isnan().all() and want[2].isnan().all()
        assert bool((got[0] == 0).all())
        for b in (1, 3):
            off = (got[b].float() - want[b, :, 0].float()).abs().max()
            assert float(off) <= 2 * 2.0 ** -11 * float(s.v[0].float().abs().max())  # two roundings of P, V each


def test_more_sequences_than_one_look():
    own = [(i * 37) % 90 for i in range(700)]
    s = Shared(96, own, 1, 32, BF16, "same", 16)
    new = [min(1, n) for n in own]
    q = s.q(new, 2)
    check(s.run(q, new, window=DENSE, max_query_len=1), *s.expect(q, new, DENSE), BF16)


def test_pages_behind_4_gib():
    """Rows of pages whose bytes and elements lie behind 2^32."""
    pages, page, H, D = 8800, 1024, 2, 128
    big = cra.PagedKVCache(pages, H, D, page, BF16, None, device=DEV)
    small = cra.PagedKVCache(6, H, D, page, BF16, None, device=DEV)
    assert big.k.numel() > 1 << 31
    n, new, P = [5000, 4500], [1, 1], 4096
    high, low = (torch.tensor([[*x, y], [*x, z]], dtype=torch.int32)
                 for x, y, z in (((8799, 8780, 8500, 8797), 8790, 8401), ((5, 0, 2, 3), 4, 1)))
    table = cra.RotaryTable(D, 8192, device=DEV)
    g = torch.Generator().manual_seed(0)
    results = []
    for cache, t in ((big, high.to(DEV)), (small, low.to(DEV))):
        g.manual_seed(0)
        x = torch.randn(1, sum(n), 6, D, generator=g).to(BF16).to(DEV).transpose(1, 2)
        x[:, :, 5000:5000 + P] = x[:, :, :P]  # the same prefix
        with torch.no_grad():
            cu = Shared.ints([0, 5000, 9500])
            q = cache.append(x[:, :2], x[:, 2:4], x[:, 4:], t, Shared.ints(n), cu, table=table, norm=True)
            last = q[:, :, [4999, 9499]].transpose(0, 2).contiguous()
            results.append([q, *cache.read(t, Shared.ints(n)),
                            cra.cron_root_attention_paged(last, cache, t, Shared.ints(n), window=DENSE,
                                                          prefix=cra.SharedPrefix(t[0, :4].contiguous(), Shared.ints([P])))])
    for y, z in zip(*results):
        assert torch.equal(y, z)


def test_layer_step():
    """A layer that appends and attends behind a prefix gives what it gives without."""
    torch.manual_seed(0)
    table = cra.RotaryTable(64, 1024, device=DEV)
    layer = cra.CronRootAttention(256, 4, n_kv_heads=2, rotary=table, qk_norm=True).to(DEV).to(BF16)
    s = Shared(160, [8, 20, 33], 2, 64, BF16, "same", 16)
    xs = torch.randn(3, 1, 256, device=DEV, dtype=BF16)
    lens = s.ints(s.lens)
    with torch.no_grad():
        a = layer(xs, cache=s.cache, batch=cra.PagedBatch(s.table, lens, window=DENSE))
        b = layer(xs, cache=s.cache, batch=cra.PagedBatch(s.table, lens, window=DENSE, prefix=s.prefix()))
    assert float((a.float() - b.float()).abs().max()) <= 4 * 2.0 ** -8 * float(a.float().abs().max())


def test_refusals():
    s = Shared(64, [1, 2], 2, 64, BF16, "same", 16)
    q = s.q([1, 1], 4)
    x = s.prefix()

    def no(error, prefix, **kw):
        with pytest.raises(error):
            s.run(q, [1, 1], prefix=prefix, **kw)
    no(ValueError, x)
    no(TypeError, (x.page_table, x.length), window=DENSE)
    no(TypeError, cra.SharedPrefix(x.page_table.long(), x.length), window=DENSE)
    no(TypeError, cra.SharedPrefix(x.page_table, 64), window=DENSE)
    no(ValueError, cra.SharedPrefix(x.page_table[None], x.length), window=DENSE)
    no(ValueError, cra.SharedPrefix(x.page_table, s.ints([1, 2])), window=DENSE)
    no(ValueError, cra.SharedPrefix(x.page_table.cpu(), x.length), window=DENSE)
    no(ValueError, cra.SharedPrefix(x.page_table, x.length.cpu()), window=DENSE)
    no(ValueError, x, window=0)


@pytest.mark.parametrize("store", ["same", "int8"])
@pytest.mark.parametrize("window,relay", [(DENSE, False), (32, True), (40, False)])
def test_the_prefix_is_read_through_its_own_table(store, window, relay):
    """With its pages gone from the sequences' tables the results stay (the prefix ends where a page does, and a block)."""
    s = Shared(160, [1, 20, 90], 2, 64, BF16, store, 16, seed=4)
    new = [1, 1, 2]
    q = s.q(new, 4)
    own = s.prefix()
    x = cra.SharedPrefix(own.page_table.clone(), own.length)
    s.table[:, :10] = -1
    check(s.run(q, new, window=window, relay=relay, prefix=x), *s.expect(q, new, window, relay), BF16)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rows_in_int8_are_rounded_once_with_p(dtype):
    """Codes are exact, their scale goes with P: a result is off by the rounding of P and its own, two alike and
    independent, sqrt(2) times one (the noise of 65536 elements' mean square is below 1%; 2.5% are given). A rounding
    of V beside them would be sqrt(3) in fp16."""
    s = Shared(1500, [1] * 32, 2, 128, dtype, "int8", 16, seed=6)
    new = [1] * 32
    q = s.q(new, 16)
    o = s.expect(q, new, DENSE)[0]
    one = (o.to(dtype).double() - o).norm()
    assert float((s.run(q, new, window=DENSE).double().cpu() - o).norm() / one) < math.sqrt(2) * 1.025
