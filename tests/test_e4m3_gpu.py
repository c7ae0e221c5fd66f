"""Linear layers in 8 bits on the GPU against a 64-bit oracle over the same codes.

Codes and scales are exact (the same rounding in PyTorch on the CPU). A result sums
products p = c s d t: the 8-bit matrix core cuts what it adds, by no more than 2^-13.3 of
sum |p| for codes of any bits (measured), taken as 2^-12; fp32 results sum bf16 products
exactly but for fp32 additions, one for every 32 columns and a few within the instruction,
(K / 16 + 16) 2^-24 of sum |p|. Then one rounding (eps / 2 of the result; a bias is added
before it, in fp32: 2^-24 of both).
"""
import math

import pytest
import torch

import cron_root_attention as cra

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def quantise(x, rows):
    """Codes, scales [R / rows, C / 128] and values (fp64) of x [R, C]; CPU."""
    R, C = x.shape
    f = torch.nn.functional.pad(x.float(), (0, -C % 128, 0, -R % rows)).unflatten(0, (-1, rows)).unflatten(2, (-1, 128))
    most = f.abs().amax((1, 3))
    part, power = torch.frexp(most.double() / 448)
    scale = torch.ldexp(torch.ones_like(part), (power - (part == 0.5).int()).clamp_min(-126))
    scale = torch.where(most > 0, scale, 2.0 ** -126)
    fine = most.isfinite()
    scale = torch.where(fine, scale, 1.0)
    y = (f.double() / scale[:, None, :, None]).float()
    y = torch.where(fine[:, None, :, None], y, math.nan)
    codes = y.to(torch.float8_e4m3fn)
    values = codes.double() * scale[:, None, :, None]
    return (codes.flatten(2).flatten(0, 1)[:R, :C], scale.float(), values.flatten(2).flatten(0, 1)[:R, :C])


def same_codes(a, b):
    a, b = a.cpu(), b.cpu()
    nan = a.float().isnan()
    assert torch.equal(nan, b.float().isnan())
    return torch.equal(a.contiguous().view(torch.uint8)[~nan], b.contiguous().view(torch.uint8)[~nan])


def check(y, xv, wv, bias, dtype):
    K = xv.shape[1]
    xv, wv = xv.to(DEV), wv.to(DEV)
    ref, mag = xv @ wv.t().contiguous(), xv.abs() @ wv.abs().t().contiguous()
    off = mag * ((K / 16 + 16) * 2.0 ** -24 if dtype == F32 else 2.0 ** -12)
    if bias is not None:
        off = off + 2.0 ** -24 * (mag + bias.double().abs().to(DEV))
        ref = ref + bias.double().to(DEV)
    off = off + torch.finfo(dtype).eps / 2 * (ref.abs() + off) + torch.finfo(dtype).tiny
    bad = ~((y.double() - ref).abs() <= off)
    assert y.dtype == dtype and not bool(bad.any()), f"{int(bad.sum())} off, worst {float(((y.double() - ref).abs() - off).max())}"


def make(M, N, K, dtype, seed=0, wdtype=BF16):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, K, generator=g) * torch.exp(2 * torch.randn(M, 1, generator=g))).to(dtype)
    w = (torch.randn(N, K, generator=g) * 0.05).to(wdtype)
    return x, w


SIZES = [(1, 1, 1), (1, 513, 4100), (2, 100, 130), (3, 16, 128), (4, 129, 127), (5, 64, 1000), (16, 40, 256),
         (17, 300, 520), (33, 17, 2100), (64, 256, 384), (65, 129, 129), (130, 64, 8), (200, 1000, 640), (300, 3, 700),
         (1, 64, 20000)]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(dtype, M, N, K):
    x, w = make(M, N, K, dtype, seed=M + N + K)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(1)).to(dtype) if M % 2 else None
    weight = cra.E4M3Weight.from_dense(w.to(DEV))
    codes, scale, wv = quantise(w, 128)
    assert same_codes(weight.codes, codes)
    assert torch.equal(weight.scales.cpu(), scale)
    assert torch.equal(weight.dense().double().cpu(), wv)
    y = cra.linear_e4m3(x.to(DEV), weight, None if bias is None else bias.to(DEV))
    assert y.shape == (M, N) and y.is_contiguous()
    check(y, quantise(x, 1)[2], wv, bias, dtype)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("M,N,K", [(4100, 4097, 200), (2100, 2052, 1100), (16390, 1030, 128)])
def test_large_tiles(dtype, M, N, K):
    x, w = make(M, N, K, dtype, seed=7)
    weight = cra.E4M3Weight.from_dense(w.to(DEV))
    check(cra.linear_e4m3(x.to(DEV), weight), quantise(x, 1)[2], quantise(w, 128)[2], None, dtype)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("M", [1, 4, 9, 40, 70])
def test_rows_come_back_from_an_identity(dtype, M):
    """Against the unit matrix a row's 8-bit values come out, exactly."""
    K = 300
    weight = cra.E4M3Weight.from_dense(torch.eye(K, device=DEV))
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=g) * torch.exp(3 * torch.randn(M, 3, generator=g)).repeat_interleave(100, 1)
    x[0, :128] = 0
    x[-1, 130] = 448 * 2.0 ** 3
    x[-1, 131] = 449.0
    x = x.to(dtype)
    y = cra.linear_e4m3(x.to(DEV), weight)
    v = quantise(x, 1)[2]
    low = v.abs() >= torch.finfo(dtype).tiny  # fp16 rounds what lies below its smallest normal number
    assert torch.equal(y.double().cpu()[low], v[low])
    assert bool(((y.double().cpu() - v).abs() <= torch.finfo(dtype).tiny * torch.finfo(dtype).eps).all())


@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e30, 3e38])
@pytest.mark.parametrize("M", [2, 80])
def test_scales_at_the_ends(scale, M):
    x, w = make(M, 130, 256, F32, seed=3, wdtype=F32)
    x = (x / x.abs().amax() * scale)
    w = w / 8
    weight = cra.E4M3Weight.from_dense(w.to(DEV))
    y = cra.linear_e4m3(x.to(DEV), weight)
    xv, wv = quantise(x, 1)[2], quantise(w, 128)[2]
    ref, mag = xv @ wv.t(), xv.abs() @ wv.abs().t()
    off = 32 * 2.0 ** -24 * mag + 256 * 2.0 ** -126 + 2.0 ** -24 * ref.abs()
    assert bool(((y.double().cpu() - ref).abs() <= off).all())


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("M", [3, 20, 100])
def test_what_is_not_finite_stays_in_its_row_or_block(dtype, M):
    x, w = make(M, 300, 400, dtype, seed=5, wdtype=F32)
    x[1, 7], x[M - 1, 399] = math.inf, math.nan
    w[140, 3] = -math.inf
    y = cra.linear_e4m3(x.to(DEV), cra.E4M3Weight.from_dense(w.to(DEV))).cpu()
    bad = torch.zeros(M, 300, dtype=torch.bool)
    bad[1] = bad[M - 1] = True
    bad[:, 128:256] = True
    assert torch.equal(y.isnan(), bad)


@pytest.mark.parametrize("M", [3, 30, 100])
def test_layouts_of_x(M):
    N, K = 96, 264
    x, w = make(M, N, K, BF16, seed=9)
    weight, x = cra.E4M3Weight.from_dense(w.to(DEV)), x.to(DEV)
    want = cra.linear_e4m3(x, weight)
    wide = torch.full((M, K + 24), math.nan, device=DEV, dtype=BF16)
    for at in (0, 8, 1):  # rows apart, and between 16-byte addresses
        wide[:, at:at + K] = x
        assert torch.equal(cra.linear_e4m3(wide[:, at:at + K], weight), want)
    assert torch.equal(cra.linear_e4m3(x.t().contiguous().t(), weight), want)
    deep = x[None, :, None].expand(2, M, 1, K)
    assert torch.equal(cra.linear_e4m3(deep, weight), want[None, :, None].expand(2, M, 1, N))
    assert torch.equal(cra.linear_e4m3(x[0], weight), want[0]) or M > 4  # other kernels, other sums
    assert cra.linear_e4m3(x[:0], weight).shape == (0, N)
    assert cra.linear_e4m3(x[None, :0], weight).shape == (1, 0, N)


def test_weights_that_are_in_8_bits_already():
    _, w = make(1, 200, 300, F32, seed=2)
    a = cra.E4M3Weight.from_dense(w.to(DEV))
    for scales in (a.scales, a.scales.to(torch.float8_e8m0fnu)):
        b = cra.E4M3Weight.from_tensors(a.codes, scales)
        assert same_codes(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    with pytest.raises(ValueError):
        cra.E4M3Weight.from_tensors(a.codes, a.scales * 1.5)
    with pytest.raises(ValueError):
        cra.E4M3Weight.from_tensors(a.codes, a.scales * 0)
    with pytest.raises(ValueError):
        cra.E4M3Weight.from_tensors(a.codes, a.scales[:1])
    with pytest.raises(TypeError):
        cra.E4M3Weight.from_tensors(a.codes.float(), a.scales)
    # rows apart and of every type
    for dtype in (F16, BF16, F32):
        v = w.to(dtype).to(DEV)
        wide = torch.zeros(200, 333, dtype=dtype, device=DEV)
        wide[:, 3:303] = v
        a, b = cra.E4M3Weight.from_dense(v), cra.E4M3Weight.from_dense(wide[:, 3:303])
        c = cra.E4M3Weight.from_dense(v.t().contiguous().t())
        assert same_codes(a.codes, b.codes) and same_codes(a.codes, c.codes)
        assert torch.equal(a.scales, b.scales) and torch.equal(a.scales, c.scales)


def test_modules():
    torch.manual_seed(0)
    lin = [torch.nn.Linear(192, n, device=DEV, dtype=BF16) for n in (128, 40)]
    m = cra.E4M3Linear.from_linear(*lin)
    x = torch.randn(2, 7, 192, device=DEV, dtype=BF16)
    with torch.no_grad():
        y = m(x)
        assert y.shape == (2, 7, 168)
        want = torch.cat([f(x) for f in lin], -1).double()
        assert float((y.double() - want).norm() / want.norm()) < 2.0 ** -4  # two roundings to 3 bits, at random
    other = cra.E4M3Linear.from_linear(torch.nn.Linear(192, 168, device=DEV, dtype=BF16))
    other.load_state_dict(m.state_dict())
    with torch.no_grad():
        assert torch.equal(other(x), y)
        assert torch.equal(other.half()(x.half()), m.half()(x.half()))
    with pytest.raises(ValueError):
        cra.E4M3Linear.from_linear(lin[0], torch.nn.Linear(192, 8, bias=False, device=DEV, dtype=BF16))


@pytest.mark.parametrize("M", [2, 24, 100])
def test_captured_and_replayed_on_another_stream(M):
    x, w = make(M, 256, 512, F16, seed=1)
    x, weight = x.to(DEV), cra.E4M3Weight.from_dense(w.to(DEV))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        cra.linear_e4m3(x, weight)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y = cra.linear_e4m3(x, weight)
    torch.cuda.current_stream().wait_stream(stream)
    for i in range(3):
        x.copy_(torch.randn_like(x))
        graph.replay()
        want = cra.linear_e4m3(x, weight)
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_two_streams_at_once():
    work = []
    for i, (M, N, K) in enumerate([(40, 600, 2048), (1, 2000, 4096), (400, 700, 900)]):
        x, w = make(M, N, K, BF16, seed=i)
        x, w = x.to(DEV), cra.E4M3Weight.from_dense(w.to(DEV))
        work.append((x, w, cra.linear_e4m3(x, w), torch.cuda.Stream()))
    torch.cuda.synchronize()
    results = []
    for _ in range(10):
        for x, w, _, stream in work:
            with torch.cuda.stream(stream):
                results.append(cra.linear_e4m3(x, w))
    torch.cuda.synchronize()
    for i, y in enumerate(results):
        assert torch.equal(y, work[i % 3][2])


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("M,N,K", [(1000, 1300, 520), (130, 200, 2900), (70, 1030, 1400), (1100, 2050, 300)])
def test_tiles_of_64_and_128(dtype, M, N, K):
    x, w = make(M, N, K, dtype, seed=M)
    b = torch.randn(N, generator=torch.Generator().manual_seed(5)).to(dtype)
    y = cra.linear_e4m3(x.to(DEV), cra.E4M3Weight.from_dense(w.to(DEV)), b.to(DEV))
    check(y, quantise(x, 1)[2], quantise(w, 128)[2], b, dtype)


@pytest.mark.parametrize("M,N,K", [(600000, 64, 4096), (300000, 8192, 128)])
def test_rows_behind_2_31_elements(M, N, K):
    g = torch.Generator(device=DEV).manual_seed(0)
    x, w = torch.randn(M, K, device=DEV, dtype=BF16, generator=g), torch.randn(N, K, device=DEV, dtype=BF16, generator=g)
    w = cra.E4M3Weight.from_dense(w)
    y = cra.linear_e4m3(x, w)
    for at in (0, M // 2 + 17, M - 40):
        part = cra.linear_e4m3(x[at:at + 40], w)
        # sums in another order, cut at 2^-13.3 of sum |p|: a rounding may fall to the other side
        off = torch.finfo(BF16).eps * part.float().abs() + 2 * 2.0 ** -12 * K
        assert bool(((y[at:at + 40].float() - part.float()).abs() <= off).all())
        assert float((y[at:at + 40].float() - part.float()).norm()) <= 2.0 ** -8 * float(part.float().norm())


def test_runs_agree_bit_for_bit():
    for M in (1, 50, 500, 3000):
        x, w = make(M, 1500, 1000, BF16, seed=M)
        x, weight = x.to(DEV), cra.E4M3Weight.from_dense(w.to(DEV))
        y = cra.linear_e4m3(x, weight)
        for _ in range(3):
            assert torch.equal(cra.linear_e4m3(x, weight), y)


def test_refusals():
    x, w = make(4, 64, 128, BF16)
    x, weight = x.to(DEV), cra.E4M3Weight.from_dense(w.to(DEV))
    bias = torch.zeros(64, device=DEV, dtype=BF16)

    def no(error, *a):
        with pytest.raises(error):
            cra.linear_e4m3(*a)
    no(ValueError, x[:, :64], weight)
    no(TypeError, x.double(), weight)
    no(TypeError, x, w.to(DEV))
    no(TypeError, x, weight, bias.float())
    no(ValueError, x, weight, bias[:32])
    no(ValueError, x, weight, bias.cpu())
    no(RuntimeError, x.cpu(), weight)
    no(NotImplementedError, x.clone().requires_grad_(), weight)
    no(NotImplementedError, x, weight, bias.clone().requires_grad_())
    import torch.autograd.forward_ad as ad
    with ad.dual_level():
        no(NotImplementedError, ad.make_dual(x, x), weight)
    for bad in (w.to(DEV)[0], w.to(DEV).double()):
        with pytest.raises((ValueError, TypeError)):
            cra.E4M3Weight.from_dense(bad)
    with pytest.raises(RuntimeError):
        cra.E4M3Weight.from_dense(w)
    with pytest.raises(ValueError):
        cra.E4M3Weight.from_dense(w.to(DEV)[:, :0])


@pytest.mark.parametrize("power", [-126, -125, -120, -117, -116, -100])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,N", [(2, 130), (9, 3200), (70, 130), (1000, 2400), (4100, 4097)])
def test_every_code_counts_at_the_smallest_scales(dtype, power, M, N):
    """Weights, and rows, of one element each that is a code times a scale near the smallest: the product with a
    power of two is exact."""
    K = 256
    codes = torch.arange(1, 127, dtype=torch.uint8).view(torch.float8_e4m3fn)  # 2^-9 .. 448
    values = codes.float().double()
    at = torch.arange(N) % 126
    w = torch.zeros(N, K, dtype=torch.uint8)
    w[torch.arange(N), torch.arange(N) % K] = torch.arange(1, 127, dtype=torch.uint8)[at]
    scales = torch.full((-(-N // 128), 2), 2.0 ** power)
    weight = cra.E4M3Weight.from_tensors(w.view(torch.float8_e4m3fn).to(DEV), scales.to(DEV))
    big = 2.0 ** 100
    y = cra.linear_e4m3(torch.full((M, K), big, dtype=dtype, device=DEV), weight)
    assert torch.equal(y.double().cpu(), (values[at] * 2.0 ** power * big).expand(M, N))
    if dtype == F32:  # (in bf16 the smallest elements of x are not numbers of their own)
        row = torch.arange(M) % 126
        x = torch.zeros(M, K, dtype=torch.float64)
        x[torch.arange(M), torch.arange(M) % K] = values[row] * 2.0 ** power
        x[torch.arange(M), (torch.arange(M) % K) // 128 * 128 + 127] = 448 * 2.0 ** power  # the block's scale
        x[torch.arange(M) % 128 == 127] = 0
        weight = cra.E4M3Weight.from_tensors(torch.zeros(N, K, dtype=torch.float8_e4m3fn, device=DEV),
                                             torch.full((-(-N // 128), 2), big, device=DEV))
        weight._codes[:, :] = 0x38  # ones
        weight._codes[:, 127::128] = 0
        y = cra.linear_e4m3(x.float().to(DEV), weight)
        want = torch.where(torch.arange(M) % 128 == 127, 0.0, values[row] * 2.0 ** power * big)
        assert torch.equal(y.double().cpu(), want[:, None].expand(M, N))
