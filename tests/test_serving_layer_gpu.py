"""The operators together, as a layer uses them: norm, rotation, attention and their
gradients in training; cache, chunks and single tokens in serving; both the same
function where they have one plan."""
import math

import pytest
import torch

import cron_root_attention as cra
from cron_root_attention import _native
from cron_root_attention.core import _attention_with_plan

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(dtype=torch.bfloat16, seed=0, **kw):
    torch.manual_seed(seed)
    layer = cra.CronRootAttention(256, 4, n_kv_heads=2, **kw).to(DEV, dtype)
    with torch.no_grad():
        for p in (layer.q_norm, layer.k_norm):
            if p is not None:
                p.add_(0.2 * torch.randn_like(p))
    return layer


def test_training_step_through_the_layer():
    """Layer = projections, norm + rotation, attention, projection: the same calls one by one give the same numbers."""
    table = cra.RotaryTable(64, 4096, interleaved=True)  # made on the CPU: the layer brings it along
    layer = make(rotary=table, qk_norm=True)
    x = torch.randn(2, 300, 256, device=DEV).bfloat16().requires_grad_(True)
    y = layer(x)
    dy = torch.randn_like(y)
    got = torch.autograd.grad(y, [x, *layer.parameters()], dy)

    def split(t, h):
        return t.view(2, 300, h, 64).transpose(1, 2)
    q, k, v = split(layer.q_proj(x), 4), split(layer.k_proj(x), 2), split(layer.v_proj(x), 2)
    q, k = cra.qk_norm_rotary(q, k, layer.q_norm, layer.k_norm, table.to(DEV))
    z = layer.o_proj(cra.cron_root_attention(q, k, v, kv_groups=2).transpose(1, 2).reshape(2, 300, 256))
    want = torch.autograd.grad(z, [x, *layer.parameters()], dy)
    assert torch.equal(y, z)
    for a, b in zip(got, want):
        # the same kernels on the same rows, in other layouts; projections' gradients sum 600 rows of bf16
        assert float((a.float() - b.float()).norm() / b.float().norm()) < 2 ** -7
    assert all(bool(g.isfinite().all()) and bool(g.any()) for g in got)


@pytest.mark.parametrize("storage,page", [(None, 64), (torch.float8_e4m3fn, 16), (torch.int8, 32)])
def test_serving_equals_training_rows(storage, page):
    """Chunks and single tokens of ragged sequences through the layer's cache against its own training path over the
    whole sequences with the same window and relay switch."""
    W = 50
    layer = make(torch.float16, rotary=cra.RotaryTable(32, 4096, device=DEV, scaling={
        "type": "yarn", "factor": 2.0, "original_positions": 1024}), qk_norm=True).eval()
    lens = [2500, 700, 61]
    xs = [torch.randn(1, n, 256, device=DEV).half() for n in lens]

    def whole(x):
        n = x.shape[1]
        q, k, v = (p(x).view(1, n, -1, 64).transpose(1, 2) for p in (layer.q_proj, layer.k_proj, layer.v_proj))
        q, k = cra.qk_norm_rotary(q, k, layer.q_norm, layer.k_norm, layer.rotary)
        if storage is not None:  # what an 8-bit cache gives back
            c = cra.PagedKVCache(-(-n // page), 2, 64, page, torch.float16, storage, device=DEV)
            t = torch.arange(c.num_pages, device=DEV).int()[None]
            ln = torch.tensor([n], dtype=torch.int32, device=DEV)
            c.write(k, v, t, ln)
            # relay rows are ranked by the keys as they were
            kq, vq = c.read(t, ln, n)
            o = torch.empty(1, 4, n, 64, device=DEV).half()
            at = 0
            for m in (n // 2, n - n // 2):
                o[:, :, at:at + m] = cra.cron_root_attention_paged(
                    q[:, :, at:at + m], c, t, ln - (n - at - m), window=W, relay=True)
                at += m
            assert kq.shape == k.shape and vq.dtype == v.dtype
        else:
            o = _attention_with_plan(q, k, v, min(W, n), True, kv_groups=2)
        return layer.o_proj(o.transpose(1, 2).reshape(1, n, 256))
    with torch.no_grad():
        want = [whole(x) for x in xs]
        pages = [-(-n // page) for n in lens]
        cache = cra.PagedKVCache(sum(pages), 2, 64, page, torch.float16, storage, device=DEV)
        order = torch.randperm(sum(pages)).int()
        table = torch.full((3, max(pages)), -1, dtype=torch.int32)
        at = 0
        for b, c in enumerate(pages):
            table[b, :c] = order[at:at + c]
            at += c
        table = table.to(DEV)
        done, got = [0, 0, 0], [[], [], []]
        for step in ([1200, 300, 60], [1299, 1, 1], [1, 399, 0]):
            new = [min(m, lens[b] - done[b]) for b, m in enumerate(step)]
            cu = [0]
            for m in new:
                cu.append(cu[-1] + m)
            x = torch.cat([xs[b][:, done[b]:done[b] + m] for b, m in enumerate(new)], 1)
            done = [d + m for d, m in zip(done, new)]
            y = layer(x, cache=cache, batch=cra.PagedBatch(
                table, torch.tensor(done, dtype=torch.int32, device=DEV),
                torch.tensor(cu, dtype=torch.int32, device=DEV), max_query_len=max(new), window=W, relay=True))
            for b in range(3):
                got[b].append(y[:, cu[b]:cu[b + 1]])
    assert done == lens
    for b in range(3):
        g, w = torch.cat(got[b], 1).float(), want[b].float()
        # fp16 attention on both sides, each within eps of its exact value per unit of |v|, through one projection
        assert float((g - w).norm() / w.norm()) < 2 ** -8
    # a decoding step of the batch form: one token of each sequence
    with torch.no_grad():
        x = torch.randn(3, 1, 256, device=DEV).half()
        room = torch.cat([table, torch.full((3, 1), -1, dtype=torch.int32, device=DEV)], 1)
        y = layer(x, cache=cache, batch=cra.PagedBatch(table, torch.tensor(lens, dtype=torch.int32, device=DEV)))
        z = layer(x.view(1, 3, 256), cache=cache, batch=cra.PagedBatch(
            room, torch.tensor(lens, dtype=torch.int32, device=DEV),
            torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=DEV), max_query_len=1))
    # (the projections of 3 rows run as one product or three: fp16 rounding of the library's order)
    assert float((y.view(-1) - z.view(-1)).abs().max()) <= 2 ** -6 * float(y.abs().max())


def test_the_cached_path_takes_no_gradients():
    layer = make(rotary=cra.RotaryTable(64, 64, device=DEV))
    cache = cra.PagedKVCache(2, 2, 64, device=DEV)
    batch = cra.PagedBatch(torch.zeros(1, 1, dtype=torch.int32, device=DEV),
                           torch.ones(1, dtype=torch.int32, device=DEV))
    x = torch.randn(1, 1, 256, device=DEV).bfloat16()
    with pytest.raises(NotImplementedError):
        layer(x, cache=cache, batch=batch)
    with torch.no_grad():
        assert layer(x, cache=cache, batch=batch).shape == x.shape


def test_python_path_equals_the_operators(monkeypatch):
    """Without the C++ operators the ctypes path launches the same kernels: equal bit for bit."""
    g = torch.Generator(device=DEV).manual_seed(2)
    q, k = (torch.randn(2, h, 77, 64, generator=g, device=DEV).half() for h in (4, 2))
    w = torch.rand(64, generator=g, device=DEV).half()
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    table = cra.RotaryTable(32, 100, device=DEV)
    pos = torch.randint(0, 100, (2, 77), generator=g, device=DEV)
    pages = torch.tensor([[3, 0], [1, 2]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([77, 100], dtype=torch.int32, device=DEV)

    def everything():
        leaves = [x.clone().requires_grad_(True) for x in (q, k, w, w)]
        y = cra.qk_norm_rotary(*leaves, table, pos)
        out = [*y, *torch.autograd.grad(y, leaves, (dq, dk))]
        y = cra.rotary_embedding(leaves[0], leaves[1], table, pos)
        out += [*y, *torch.autograd.grad(y, leaves[:2], (dq, dk))]
        with torch.no_grad():
            out.append(cra.rotary_embedding(q, None, table))
            cache = cra.PagedKVCache(4, 2, 64, 64, torch.float16, torch.float8_e4m3fn, device=DEV)
            cache.write(k, k, pages, lens)
            out += [cache.k.float(), cache.k_scale, cache.k_norm]
            out.append(cra.cron_root_attention_paged(q, cache, pages, lens))
            out.append(cra.cron_root_attention_paged(q[:, :, :1], cache, pages, lens, window=9, relay=True))
        return [x.detach() for x in out]
    fast = everything()
    assert _native.fast_op("rotary") is not None
    monkeypatch.setattr(_native, "fast_op", lambda name: None)
    slow = everything()
    assert len(fast) == len(slow)
    for a, b in zip(fast, slow):
        assert a.shape == b.shape and a.stride() == b.stride() and torch.equal(a, b)


def test_captured_decoding_of_a_layer():
    """Projections, norm, rotation, cache write and attention in one graph, replayed over growing sequences."""
    layer = make(torch.bfloat16, rotary=cra.RotaryTable(64, 512, device=DEV), qk_norm=True).eval()
    caches = [cra.PagedKVCache(8, 2, 64, device=DEV) for _ in range(2)]
    table = torch.arange(8, device=DEV).int().view(2, 4)
    lens = torch.tensor([62, 9], dtype=torch.int32, device=DEV)
    first = torch.randn(1, 71, 256, device=DEV).bfloat16()
    cu = torch.tensor([0, 62, 71], dtype=torch.int32, device=DEV)
    with torch.no_grad():
        for c in caches:
            layer(first, cache=c, batch=cra.PagedBatch(table, lens, cu))
        x = torch.zeros(2, 1, 256, device=DEV).bfloat16()
        batch = cra.PagedBatch(table, lens)
        warm = cra.PagedKVCache(8, 2, 64, device=DEV)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer(x, cache=warm, batch=batch)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer(x, cache=caches[0], batch=batch)
        for i in range(4):
            lens.add_(1)
            x.copy_(torch.randn(x.shape, device=DEV))
            graph.replay()
            torch.cuda.synchronize()
            got = y.clone()
            assert torch.equal(got, layer(x, cache=caches[1], batch=batch)), i
