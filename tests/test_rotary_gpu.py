"""The rotary operators on the GPU against their formulas in 64 bits.

Tolerances count roundings. One output rounding: eps/2 of the value (plus half
the smallest subnormal). fp32 arithmetic in units of u = 2^-24: cos, sin and the
two products of a pair are off by at most 4 u (|a| + |b|) m together (m the
table's multiplier); a mean of D squares is off by at most D u, so a normed value
by (D/2 + 8) u. The backward's formula adds such terms; a weight's gradient sums
n rows, each addition off by u of the sum of magnitudes so far.
"""
import math

import pytest
import torch

import cron_root_attention as cra
from cron_root_attention.rotary import rotary_frequencies

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
YARN = {"type": "yarn", "factor": 4.0, "original_positions": 512}


def rows(B, H, S, D, dtype, layout, gen):
    x = torch.randn(B, S, H + 1, D, generator=gen).to(dtype).to(DEV)
    if layout == "slice":        # rows of a wider projection, one element further: unaligned for some types
        return x[:, :, 1:].transpose(1, 2)
    x = x[:, :, 1:].contiguous()
    return x.transpose(1, 2) if layout == "bshd" else x.transpose(1, 2).contiguous()


def turn64(z, pos, table, scaling, base, back=False):
    """Rotation in 64 bits of z [B, H, S, D] by pos [B or 1, S]; also |a| + |b| of each element's pair."""
    rot = table.rotary_dim
    f, m = rotary_frequencies(rot, base, scaling)
    ang = pos.double().cpu()[:, None, :, None] * f
    c, s = ang.cos() * m, ang.sin() * m * (-1 if back else 1)
    y, mag = z.clone(), z.abs()
    ia = torch.arange(0, rot, 2) if table.interleaved else torch.arange(rot // 2)
    ib = ia + 1 if table.interleaved else ia + rot // 2
    a, b = z[..., ia], z[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * m
    return y, mag


def norm64(x, w, eps):
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    return x * r * (1 if w is None else w), r


def close(got, ref, extra, what):
    """One rounding to got's type, and `extra` from fp32 arithmetic."""
    fi = torch.finfo(got.dtype)
    tol = fi.eps / 2 * ref.abs() + extra + fi.smallest_normal * fi.eps / 2
    bad = (got.double().cpu() - ref).abs() - tol
    assert bool((bad <= 0).all()), f"{what}: {float(bad.max()):.3e} above the bound at {int((bad > 0).sum())} elements"


SHAPES = [
    # B, Hq, Hkv, S, D, rot
    (1, 2, 1, 1, 64, 64),
    (2, 4, 2, 33, 128, 128),
    (1, 8, 2, 130, 256, 256),
    (3, 3, 3, 17, 32, 16),
    (1, 5, 1, 70, 80, 20),     # odd head counts, 2-element chunks
    (1, 2, 2, 9, 96, 24),      # 4-element chunks
    (2, 2, 1, 31, 33, 32),     # odd head dim: single elements
    (1, 1, 1, 5, 7, 2),
    (1, 2, 2, 6, 255, 254),    # two pairs a lane
    (1, 12, 4, 300, 64, 32),
]


@pytest.mark.parametrize("B,Hq,Hkv,S,D,rot", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_forward_and_backward(B, Hq, Hkv, S, D, rot, dtype, interleaved):
    g = torch.Generator().manual_seed(S * D + rot)
    layout = ("bhsd", "bshd", "slice")[(S + D) % 3]
    q, k = rows(B, Hq, S, D, dtype, layout, g), rows(B, Hkv, S, D, dtype, layout, g)
    dq, dk = rows(B, Hq, S, D, dtype, "bshd", g), rows(B, Hkv, S, D, dtype, "slice", g)
    scaling = YARN if S % 2 else None
    table = cra.RotaryTable(rot, 5000, scaling=scaling, interleaved=interleaved, device=DEV)
    pos = torch.randint(0, 5000, (B, S), generator=g, dtype=torch.int64 if S % 3 else torch.int32).to(DEV)
    q.requires_grad_(True), k.requires_grad_(True)
    yq, yk = cra.rotary_embedding(q, k, table, pos)
    gq, gk = torch.autograd.grad((yq, yk), (q, k), (dq, dk))
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(cra.rotary_embedding(q, k, table, pos), (yq, yk)))
        assert torch.equal(cra.rotary_embedding(q, None, table, pos), yq)
    for x, y, dy, gx, n in ((q, yq, dq, gq, "q"), (k, yk, dk, gk, "k")):
        assert y.dtype == dtype and y.shape == x.shape
        ref, mag = turn64(x.detach().double().cpu(), pos, table, scaling, 10000.0)
        close(y.detach(), ref, 4 * U * mag, n)
        ref, mag = turn64(dy.double().cpu(), pos, table, scaling, 10000.0, back=True)
        close(gx, ref, 4 * U * mag, "d" + n)


@pytest.mark.parametrize("B,Hq,Hkv,S,D,rot", SHAPES)
@pytest.mark.parametrize("dtype,wdtype", [(torch.float16, torch.float16), (torch.float16, torch.float32),
                                          (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_rotary_forward_and_backward(B, Hq, Hkv, S, D, rot, dtype, wdtype, interleaved):
    g = torch.Generator().manual_seed(7 * S + D)
    eps = 1e-6
    layout = ("slice", "bhsd", "bshd")[(S + D) % 3]
    q, k = (3 * rows(B, Hq, S, D, dtype, layout, g)), rows(B, Hkv, S, D, dtype, layout, g)
    dq, dk = rows(B, Hq, S, D, dtype, "bhsd", g), rows(B, Hkv, S, D, dtype, "bshd", g)
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(wdtype).to(DEV) for _ in range(2))
    table = cra.RotaryTable(rot, 5000, interleaved=interleaved, device=DEV)
    pos = torch.randint(0, 5000, (S,), generator=g).to(DEV)
    leaves = [x.requires_grad_(True) for x in (q, k, wq, wk)]
    yq, yk = cra.qk_norm_rotary(q, k, wq, wk, table, pos, eps=eps)
    got = torch.autograd.grad((yq, yk), leaves, (dq, dk))
    again = torch.autograd.grad(cra.qk_norm_rotary(q, k, wq, wk, table, pos, eps=eps), leaves, (dq, dk))
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    for x, w, y, dy, gx, gw, n in ((q, wq, yq, dq, got[0], got[2], "q"), (k, wk, yk, dk, got[1], got[3], "k")):
        x64, w64 = x.detach().double().cpu(), w.detach().double().cpu()
        z, r = norm64(x64, w64, eps)
        ref, mag = turn64(z, pos[None], table, None, 10000.0)
        close(y.detach(), ref, (D / 2 + 12) * U * mag, n)
        dz, dmag = turn64(dy.double().cpu(), pos[None], table, None, 10000.0, back=True)
        hat, gg = x64 * r, dz * w64
        dot = (gg * hat).mean(-1, keepdim=True)
        dots = (dmag * w64.abs() * hat.abs()).mean(-1, keepdim=True)
        ref = r * (gg - hat * dot)
        close(gx, ref, (2 * D + 24) * U * r * (dmag * w64.abs() + hat.abs() * dots), "d" + n)
        nrow = B * x.shape[1] * S
        ref = (dz * hat).sum((0, 1, 2))
        close(gw, ref, (nrow + D / 2 + 16) * U * (dmag * hat.abs()).sum((0, 1, 2)), "dw" + n)


def test_many_rows():
    """More rows than the backward has workgroups: each strides over several; the weights' gradients over all of them."""
    g = torch.Generator(device=DEV).manual_seed(3)
    B, Hq, Hkv, S, D = 2, 7, 5, 6000, 128
    q, k = (torch.randn(B, H, S, D, generator=g, device=DEV).bfloat16() for H in (Hq, Hkv))
    dq, dk = (torch.randn(B, H, S, D, generator=g, device=DEV).bfloat16() for H in (Hq, Hkv))
    wq, wk = (1 + 0.2 * torch.randn(D, generator=g, device=DEV) for _ in range(2))
    table = cra.RotaryTable(64, S, device=DEV)
    leaves = [x.requires_grad_(True) for x in (q, k, wq, wk)]
    y = cra.qk_norm_rotary(q, k, wq, wk, table)
    got = torch.autograd.grad(y, leaves, (dq, dk))
    # the same rows in small calls
    for h in (0, 3, 6):
        sl = q.detach()[:1, h:h + 1, 5000:5100]
        one = cra.qk_norm_rotary(sl, None, wq.detach(), None, table, torch.arange(5000, 5100, device=DEV))
        assert torch.equal(one, y[0].detach()[:1, h:h + 1, 5000:5100])
    x, w, dy = q.detach().double(), wq.detach().double(), dq.double()
    r = (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    dz, dmag = turn64(dy.cpu(), torch.arange(S)[None], table, None, 10000.0, back=True)
    hat = (x * r).cpu()
    ref = (dz * hat).sum((0, 1, 2))
    # sums of 84000 rows run over at least 1024 partial sums: at most 128 + 1024 additions each
    close(got[2], ref, 1300 * U * (dmag * hat.abs()).sum((0, 1, 2)), "dwq")


def test_gradients_against_differences():
    g = torch.Generator().manual_seed(11)
    B, H, S, D = 1, 2, 9, 64
    q, k = (torch.randn(B, H, S, D, generator=g).to(DEV) for _ in range(2))
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(DEV) for _ in range(2))
    cq, ck = (torch.randn(B, H, S, D, generator=g).to(DEV) for _ in range(2))
    table = cra.RotaryTable(48, 64, interleaved=True, device=DEV)

    def loss(*xs):
        y = cra.qk_norm_rotary(*xs, table)
        return (y[0].double() * cq).sum() + (y[1].double() * ck).sum()
    xs = [x.requires_grad_(True) for x in (q, k, wq, wk)]
    grads = torch.autograd.grad(loss(*xs), xs)
    h = 2.0 ** -7
    for i, gr in enumerate(grads):
        u = torch.randn(xs[i].shape, generator=g).to(DEV)
        with torch.no_grad():
            lo, hi = ([x + s * h * u if j == i else x for j, x in enumerate(xs)] for s in (-1, 1))
            diff = float(loss(*hi) - loss(*lo)) / (2 * h)
        want = float((gr.double() * u).sum())
        # 1152 outputs of magnitude 1-4, each off by at most 40 u: 2^-12 / h in all at most; third order h^2
        assert abs(diff - want) <= 1152 * 4 * 40 * U / (2 * h) * 0.1 + 64 * h * h * (1 + abs(want)), (i, diff, want)


def test_positions_outside_the_table_give_nan():
    table = cra.RotaryTable(32, 10, device=DEV)
    q = torch.ones(1, 1, 4, 64, device=DEV, dtype=torch.float16)
    pos = torch.tensor([-1, 9, 10, 1 << 40], device=DEV)
    y = cra.rotary_embedding(q, None, table, pos)
    bad = y.isnan()
    assert bad[0, 0, [0, 2, 3], :32].all() and not bad[0, 0, :, 32:].any() and not bad[0, 0, 1].any()


def test_norm_alone_and_without_weights():
    g = torch.Generator().manual_seed(5)
    q = torch.randn(2, 3, 5, 64, generator=g).bfloat16().to(DEV).requires_grad_(True)
    y = cra.qk_norm_rotary(q, None, None, None, eps=1e-5)
    ref, _ = norm64(q.detach().double().cpu(), None, 1e-5)
    close(y.detach(), ref, 48 * U * ref.abs(), "y")
    (gq,) = torch.autograd.grad(y.sum(), q)  # an expanded upstream gradient
    x = q.detach().double().cpu()
    r = (x.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    close(gq, r * (1 - x * r * (x * r).mean(-1, keepdim=True)),
          200 * U * r * (1 + (x * r).abs() * (x * r).abs().mean(-1, keepdim=True)), "dq")
    zero = cra.qk_norm_rotary(torch.zeros(1, 1, 1, 64, device=DEV), None, None, None)
    assert bool((zero == 0).all())


def test_one_output_without_gradient_and_expanded_inputs():
    table = cra.RotaryTable(64, 8, device=DEV)
    one = torch.randn(1, 1, 8, 64, device=DEV, requires_grad=True)
    q, k = one.expand(2, 4, 8, 64), one.expand(2, 2, 8, 64)  # shared rows: strides of 0
    w = torch.ones(64, device=DEV, requires_grad=True)
    yq, yk = cra.qk_norm_rotary(q, k, w, w, table)
    g1 = torch.autograd.grad(yq.sum(), (one, w), retain_graph=True)
    g2 = torch.autograd.grad(yk.sum(), (one, w), retain_graph=True)
    both = torch.autograd.grad(yq.sum() + yk.sum(), (one, w))
    for a, b, c in zip(g1, g2, both):
        assert torch.allclose(a + b, c, rtol=1e-5, atol=1e-5)
    gq, = torch.autograd.grad(cra.rotary_embedding(q, k, table)[1].sum(), one)
    assert gq.shape == one.shape and bool(gq.isfinite().all())


def test_refusals_on_the_gpu():
    t = cra.RotaryTable(32, 8, device=DEV)
    q = torch.zeros(1, 2, 4, 32, device=DEV)
    for bad in (lambda: cra.rotary_embedding(q, q, cra.RotaryTable(32, 8)),
                lambda: cra.rotary_embedding(q, q[:, :, :3], t),
                lambda: cra.rotary_embedding(torch.zeros(1, 1, 9, 32, device=DEV), None, t),
                lambda: cra.rotary_embedding(q, None, cra.RotaryTable(64, 8, device=DEV)),
                lambda: cra.rotary_embedding(q, None, t, torch.zeros(1, 5, dtype=torch.int32, device=DEV)),
                lambda: cra.rotary_embedding(q, None, t, torch.zeros(4, dtype=torch.int32)),
                lambda: cra.rotary_embedding(q[:, :, :0], None, t),
                lambda: cra.qk_norm_rotary(q, q, torch.ones(31, device=DEV), None),
                lambda: cra.qk_norm_rotary(q, None, None, torch.ones(32, device=DEV)),
                lambda: cra.qk_norm_rotary(q, None, None, None, positions=torch.zeros(4, device=DEV).int()),
                lambda: cra.qk_norm_rotary(q, None, None, None, eps=-1.0)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: cra.rotary_embedding(q, q.half(), t), lambda: cra.rotary_embedding(q.double(), None, t),
                lambda: cra.rotary_embedding(q, None, t, torch.zeros(4, device=DEV)),
                lambda: cra.rotary_embedding(q, None, None),
                lambda: cra.qk_norm_rotary(q, q, torch.ones(32, device=DEV).half(), None)):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(NotImplementedError):
        cra.rotary_embedding(torch.zeros(1, 1, 1, 300, device=DEV), None, t)


def test_captured_step_replays():
    """Forward and backward captured once: every replay equals the eager step on the same inputs."""
    B, H, S, D = 1, 4, 65, 64
    table = cra.RotaryTable(D, S, device=DEV)
    q, k = (torch.randn(B, H, S, D, device=DEV).half().requires_grad_(True) for _ in range(2))
    w = torch.rand(D, device=DEV).half().requires_grad_(True)
    dy = torch.randn(B, H, S, D, device=DEV).half()

    def step():
        y = cra.qk_norm_rotary(q, k, w, w, table)
        return [*y, *torch.autograd.grad(y, (q, k, w), (dy, dy))]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        with torch.no_grad():
            q.copy_(torch.randn(q.shape, device=DEV)), k.copy_(torch.randn(k.shape, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.detach().clone() for x in out]
        want = [x.detach() for x in step()]
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


@pytest.mark.parametrize("path", ["op", "function"])
@pytest.mark.parametrize("norm", [False, True])
def test_positions_and_table_changed_before_the_backward(norm, path, monkeypatch):
    """A buffer of positions (or the table) that is overwritten between forward and backward raises, as any saved tensor."""
    if path == "function":
        monkeypatch.setattr(cra.rotary._native, "fast_op", lambda name: None)
    for change in ("none", "positions", "table"):
        table = cra.RotaryTable(32, 50, device="cuda")
        pos = torch.arange(8, device="cuda")
        q = torch.randn(1, 2, 8, 32, device="cuda", requires_grad=True)
        w = torch.randn(32, device="cuda", requires_grad=True)
        y = cra.qk_norm_rotary(q, None, w, None, table, pos) if norm else cra.rotary_embedding(q, None, table, pos)
        if change == "positions":
            pos.add_(1)
        elif change == "table":
            table.table.mul_(2)
        if change == "none":
            y.sum().backward()
            assert q.grad is not None
        else:
            with pytest.raises(RuntimeError, match="inplace operation"):
                y.sum().backward()


@pytest.mark.parametrize("path", ["op", "function"])
@pytest.mark.parametrize("norm", [False, True])
def test_second_derivatives_raise(norm, path, monkeypatch):
    """Gradients formed under create_graph are right; differentiating them again raises instead of leaving terms out."""
    if path == "function":
        monkeypatch.setattr(cra.rotary._native, "fast_op", lambda name: None)
    table = cra.RotaryTable(32, 8, device=DEV)
    q, k = (torch.randn(1, H, 8, 32, device=DEV, requires_grad=True) for H in (4, 2))

    def y():
        return cra.qk_norm_rotary(q, k, None, None, table) if norm else cra.rotary_embedding(q, k, table)

    def loss():
        return sum((t * t * t).sum() for t in y())

    plain = torch.autograd.grad(loss(), (q, k))
    for a, b in zip(plain, torch.autograd.grad(loss(), (q, k), create_graph=True)):
        assert torch.equal(a, b)
        with pytest.raises(RuntimeError, match="no second derivative"):
            b.sum().backward(retain_graph=True)


def test_tables_that_the_kernels_cannot_read():
    q = torch.randn(1, 2, 8, 32, device=DEV)
    for change in (lambda t: t.half(), lambda t: t.t().contiguous().t(), lambda t: t[:, :16], lambda t: t[:, ::2]):
        table = cra.RotaryTable(32, 50, device=DEV)
        table.table = change(table.table)
        with pytest.raises(ValueError, match="contiguous float32"):
            cra.rotary_embedding(q, None, table)


@pytest.mark.parametrize("path", ["op", "function"])
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("present", ["q wq", "q k wq", "q k wk", "q k wq wk", "q k"])
def test_gradients_with_a_tensor_or_weight_absent(present, turned, path, monkeypatch):
    """One tensor, one weight, no table: every input that is there gets its gradient, whatever stands before it."""
    if path == "function":
        monkeypatch.setattr(cra.rotary._native, "fast_op", lambda name: None)
    g = torch.Generator().manual_seed(21)
    B, S, D, eps = 2, 13, 64, 1e-6
    have = present.split()
    q, k = (torch.randn(B, H, S, D, generator=g).to(DEV) for H in (4, 2))
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(DEV) for _ in range(2))
    dys = [torch.randn(B, H, S, D, generator=g).to(DEV) for H in (4, 2)]
    args = {n: x.requires_grad_(True) for n, x in dict(q=q, k=k, wq=wq, wk=wk).items() if n in have}
    table = cra.RotaryTable(48, S, device=DEV) if turned else None
    y = cra.qk_norm_rotary(q, args.get("k"), args.get("wq"), args.get("wk"), table, eps=eps)
    y = (y,) if torch.is_tensor(y) else y
    torch.autograd.backward(y, dys[:len(y)])
    for x, w, dy, n in ((q, "wq", dys[0], "q"), (k, "wk", dys[1], "k")):
        if n not in have:
            continue
        dz, dmag = dy.double().cpu(), dy.double().cpu().abs()
        if turned:
            dz, dmag = turn64(dz, torch.arange(S)[None], table, None, 10000.0, back=True)
        x64 = x.detach().double().cpu()
        w64 = args[w].detach().double().cpu() if w in have else torch.ones(D, dtype=torch.float64)
        hat, r = norm64(x64, None, eps)
        gg = dz * w64
        dots = (dmag * w64.abs() * hat.abs()).mean(-1, keepdim=True)
        close(x.grad, r * (gg - hat * (gg * hat).mean(-1, keepdim=True)),
              (2 * D + 24) * U * r * (dmag * w64.abs() + hat.abs() * dots), "d" + n)
        if w in have:
            assert args[w].grad is not None, w
            close(args[w].grad, (dz * hat).sum((0, 1, 2)),
                  (B * x.shape[1] * S + D / 2 + 16) * U * (dmag * hat.abs()).sum((0, 1, 2)), "d" + w)


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (64, torch.float32), (33, torch.float16), (256, torch.bfloat16)])
def test_weight_gradients_with_eps_zero(D, dtype):
    """Threads behind the last row add nothing to the weights' gradients, with eps = 0 too."""
    g = torch.Generator().manual_seed(D)
    for B, Hq, Hkv, S in ((1, 1, 1, 1), (2, 5, 3, 10), (1, 7, 1, 129)):
        q, k = (torch.randn(B, H, S, D, generator=g).to(dtype).to(DEV).requires_grad_(True) for H in (Hq, Hkv))
        wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(dtype).to(DEV).requires_grad_(True) for _ in range(2))
        dys = [torch.randn(B, H, S, D, generator=g).to(dtype).to(DEV) for H in (Hq, Hkv)]
        got = torch.autograd.grad(cra.qk_norm_rotary(q, k, wq, wk, eps=0.0), (q, k, wq, wk), dys)
        assert all(bool(x.isfinite().all()) for x in got)
        for x, dy, gw in ((q, dys[0], got[2]), (k, dys[1], got[3])):
            hat, _ = norm64(x.detach().double().cpu(), None, 0.0)
            dz = dy.double().cpu()
            close(gw, (dz * hat).sum((0, 1, 2)), (B * x.shape[1] * S + D / 2 + 16) * U * (dz * hat).abs().sum((0, 1, 2)), "dw")


@pytest.mark.parametrize("path", ["op", "function"])
def test_tangents_are_refused(path, monkeypatch):
    """Forward-mode derivatives are not built: a dual tensor raises instead of losing its tangent."""
    from torch.autograd import forward_ad
    if path == "function":
        monkeypatch.setattr(cra.rotary._native, "fast_op", lambda name: None)
    table = cra.RotaryTable(32, 8, device=DEV)
    q, k = (torch.randn(1, H, 8, 32, device=DEV) for H in (4, 2))
    w = torch.rand(32, device=DEV)
    with forward_ad.dual_level():
        dq, dk, dw = (forward_ad.make_dual(x, torch.ones_like(x)) for x in (q, k, w))
        calls = [lambda: cra.rotary_embedding(dq, k, table), lambda: cra.rotary_embedding(q, dk, table),
                 lambda: cra.rotary_embedding(dq, None, table), lambda: cra.qk_norm_rotary(dq, k, w, w, table),
                 lambda: cra.qk_norm_rotary(q, k, w, dw, table), lambda: cra.qk_norm_rotary(q, None, dw, None)]
        for call in calls:
            with pytest.raises(RuntimeError, match="jvp"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="jvp"):
                call()
        cra.qk_norm_rotary(q, k, w, w, table)  # without a tangent


@pytest.mark.parametrize("path", ["op", "function"])
def test_a_table_that_wants_a_gradient_is_refused(path, monkeypatch):
    """The angles' gradient is not built: asked for, it raises instead of staying away."""
    if path == "function":
        monkeypatch.setattr(cra.rotary._native, "fast_op", lambda name: None)
    table = cra.RotaryTable(32, 8, device=DEV)
    table.table.requires_grad_(True)
    q = torch.randn(1, 2, 8, 32, device=DEV)
    for leaf in (q, q.clone().requires_grad_(True)):
        for call in (lambda: cra.rotary_embedding(leaf, None, table), lambda: cra.qk_norm_rotary(leaf, None, None, None, table)):
            with pytest.raises(NotImplementedError, match="no gradient"):
                call()
    with torch.no_grad():
        assert cra.rotary_embedding(q, None, table).isfinite().all()


@pytest.mark.parametrize("path", ["op", "function"])
def test_positions_and_weights_in_any_layout(path, monkeypatch):
    """Strided, shared and one-row positions, weights that are a slice: as their contiguous copies."""
    if path == "function":
        monkeypatch.setattr(cra.rotary._native, "fast_op", lambda name: None)
    B, S, D = 3, 20, 64
    table = cra.RotaryTable(D, 200, device=DEV)
    q, k = (torch.randn(B, H, S, D, device=DEV) for H in (4, 2))
    wide = torch.randint(0, 200, (2 * B, 3 * S), device=DEV)
    w = torch.randn(2 * D, device=DEV)[::2].requires_grad_(True)
    for pos in (wide[::2, ::3], wide[:B, :S].int()[:, :], wide[:1, S:2 * S], wide[0, ::3], wide[:1, :S].expand(B, S),
                wide[:B, :1].expand(B, S), wide[:S, :B].t() if 2 * B >= S else wide.t()[:S, :B].t()):
        a = cra.qk_norm_rotary(q, k, w, None, table, pos)
        b = cra.qk_norm_rotary(q, k, w.detach().contiguous(), None, table, pos.contiguous())
        assert all(torch.equal(x, y) for x, y in zip(a, b)), (pos.shape, pos.stride())
        full = pos.expand(B, S) if pos.dim() == 2 else pos[None].expand(B, S)
        for i in range(B):  # each sequence by itself
            c = cra.qk_norm_rotary(q[i:i + 1], k[i:i + 1], w, None, table, full[i].contiguous())
            assert all(torch.equal(x, y[i:i + 1]) for x, y in zip(c, a))
    gw, = torch.autograd.grad(a[0].sum(), w)
    assert gw.shape == (D,) and gw.isfinite().all()
