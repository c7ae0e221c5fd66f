"""One serving step of a layer in 8 bits: joint projection, new tokens appended with norm
and rotation, attention behind a shared prefix, output projection."""
import pytest
import torch

import cron_root_attention as cra

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def make(seed=0, **kw):
    torch.manual_seed(seed)
    layer = cra.CronRootAttention(512, 8, n_kv_heads=2, **kw).to(DEV, BF16).eval()
    return layer


def copy_of(layer, **kw):
    other = make(**kw)
    other.load_state_dict(layer.state_dict())
    return other


def test_the_layer_is_its_operators_one_by_one():
    table = cra.RotaryTable(64, 512, device=DEV)
    layer = make(rotary=table, qk_norm=True, bias=True)
    with torch.no_grad():
        for n in "qkvo":
            getattr(layer, n + "_proj").bias.normal_()
    joint = torch.cat([layer.q_proj.weight, layer.k_proj.weight, layer.v_proj.weight])
    bias = torch.cat([layer.q_proj.bias, layer.k_proj.bias, layer.v_proj.bias])
    wo, bo = cra.E4M3Weight.from_dense(layer.o_proj.weight), layer.o_proj.bias.detach().clone()
    wqkv = cra.E4M3Weight.from_dense(joint)
    assert layer.to_e4m3() is layer and layer.to_e4m3() is layer
    assert {n.split(".")[0] for n in layer.state_dict()} == {"qkv_proj", "o_proj", "q_norm", "k_norm"}
    x = torch.randn(2, 130, 512, device=DEV, dtype=BF16)
    with torch.no_grad():
        y = layer(x)
        h = cra.linear_e4m3(x, wqkv, bias.detach()).view(2, 130, 12, 64).transpose(1, 2)
        q, k = cra.qk_norm_rotary(h[:, :8], h[:, 8:10], layer.q_norm, layer.k_norm, table)
        o = cra.cron_root_attention(q, k, h[:, 10:], kv_groups=4)
        want = cra.linear_e4m3(o.transpose(1, 2).reshape(2, 130, 512), wo, bo)
        assert torch.equal(y, want)
        other = torch.randn_like(x)
        h2 = cra.linear_e4m3(other, wqkv, bias.detach()).view(2, 130, 12, 64).transpose(1, 2)
        q, k = cra.qk_norm_rotary(h[:, :8], h2[:, 8:10], layer.q_norm, layer.k_norm, table)
        o = cra.cron_root_attention(q, k, h2[:, 10:], kv_groups=4)
        assert torch.equal(layer(x, kv=other), cra.linear_e4m3(o.transpose(1, 2).reshape(2, 130, 512), wo, bo))
    with pytest.raises(NotImplementedError):
        layer(x.requires_grad_())


@pytest.mark.parametrize("storage", [None, torch.float8_e4m3fn, torch.int8])
def test_serving_a_batch_behind_a_prefix(storage):
    """A common prompt is stored once; requests behind it go on in chunks and single tokens. What comes out is near the
    layer in 16 bits over whole sequences: its 8-bit products are off by the roundings of x and w to 3 bits, 2^-4 of
    a product at most each, independent ones over 512 columns; 2^-3 of the norm is asked for."""
    P, chunk, steps, N = 96, 20, 4, 5
    table = cra.RotaryTable(64, 512, device=DEV)
    dense = make(rotary=table, qk_norm=True)
    layer = copy_of(dense, rotary=table, qk_norm=True).to_e4m3()
    page, width = 16, 10
    cache = cra.PagedKVCache(6 + N * 4, 2, 64, page, BF16, storage, device=DEV)
    pages = torch.full((N, width), -1, dtype=torch.int32, device=DEV)
    pages[:, :6] = torch.arange(6, device=DEV)
    pages[:, 6:] = 6 + torch.arange(N * 4, device=DEV).view(N, 4)
    xs = torch.randn(N, P + chunk + steps, 512, device=DEV, dtype=BF16)
    xs[:, :P] = xs[:1, :P]
    got = torch.empty_like(xs)
    whole = 1 << 16

    def ints(*x):
        return torch.tensor(x, dtype=torch.int32, device=DEV)
    with torch.no_grad():
        got[:, :P] = layer(xs[:1, :P], cache=cache, batch=cra.PagedBatch(pages[:1], ints(P), window=whole))
        prefix = cra.SharedPrefix(pages[0, :6].contiguous(), ints(P))
        lens = ints(*[P + chunk] * N)
        batch = cra.PagedBatch(pages, lens, window=whole, prefix=prefix)
        got[:, P:P + chunk] = layer(xs[:, P:P + chunk], cache=cache, batch=batch)
        x = xs[:, :1].clone()
        lens += 1
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        x.copy_(xs[:, P + chunk:P + chunk + 1])
        with torch.cuda.stream(stream):
            layer(x, cache=cache, batch=batch)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                y = layer(x, cache=cache, batch=batch)
        torch.cuda.current_stream().wait_stream(stream)
        for i in range(steps):
            x.copy_(xs[:, P + chunk + i:P + chunk + i + 1])
            graph.replay()
            got[:, P + chunk + i:P + chunk + i + 1] = y
            lens += 1
        q, k, v = dense._projected(xs, xs)
        q, k = cra.qk_norm_rotary(q, k, dense.q_norm, dense.k_norm, table)
        k, v = (t.float().repeat_interleave(4, 1) for t in (k, v))
        s = (q.float() @ k.transpose(-1, -2).contiguous()) / 8
        n = s.shape[-1]
        p = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1), float("-inf")).softmax(-1)
        want = dense.o_proj((p @ v).to(BF16).transpose(1, 2).reshape(N, n, 512))
    for part in (slice(0, P), slice(P, P + chunk), slice(P + chunk, n)):
        a, b = got[:, part].double(), want[:, part].double()
        assert float((a - b).norm() / b.norm()) < 2.0 ** -3
    # the same step without naming the prefix
    with torch.no_grad():
        lens -= 1
        a = layer(x, cache=cache, batch=batch)
        b = layer(x, cache=cache, batch=cra.PagedBatch(pages, lens, window=whole))
    assert float((a.double() - b.double()).norm() / b.double().norm()) < 2.0 ** -4
