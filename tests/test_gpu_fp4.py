"""The 4-bit weights on the GPU against float64.

Products of small whole numbers have exact fp32 sums in any order: there the output is the exact one, rounded.  Elsewhere: the
output's rounding, HALF |y|, and fp32 sums of K + 1 terms, each addition off by 2^-24 of a partial sum of at most
sum |x||w| + |b| (an instruction that cuts off instead of rounding: 2^-23)."""

import pytest
import torch

from oracle import fp4 as O

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
HALF = {BF: 2.0 ** -8, HF: 2.0 ** -11}
E8 = torch.float8_e8m0fnu


def _bytes(t):
    return t.view(torch.uint8).cpu()


# ------------------------------------------------------------------------------------------------ quantizer
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (5, 480), (130, 512), (17, 544), (64, 4096), (2, 50016)])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_quantizer(dev, rows, cols, dtype):
    from atma_amd.kernel import dequantize_weight_fp4, quantize_weight_fp4
    g = torch.Generator().manual_seed(rows * cols)
    w = (torch.randn(rows, cols, generator=g) * torch.exp(2 * torch.randn(rows, cols // 32, generator=g)).repeat_interleave(32, 1))
    w[0, :32] = 0
    w = w.to(dtype)
    data, scale = quantize_weight_fp4(w.to(dev))
    assert data.shape == (rows, cols // 2) and data.dtype == torch.uint8
    assert scale.shape == (rows, cols // 32) and scale.dtype == E8
    codes, s = O.quantize(w)
    assert torch.equal(O.scale_values(scale.cpu()), s)
    assert torch.equal(data.cpu(), O.pack(codes))
    for out in (BF, HF, F32):
        v = dequantize_weight_fp4(data, scale, out)
        assert v.dtype == out and torch.equal(v.cpu(), O.values(data, scale).to(out))   # (float64 to 16 bits rounds once)


def test_quantizer_borders(dev):
    """Values half way between two neighbours, largest magnitudes around 7 2^e, the ends of the scales' range, zeros."""
    from atma_amd.kernel import quantize_weight_fp4
    half = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], dtype=torch.float64)
    around = torch.cat((half * (1 - 2.0 ** -20), half, half * (1 + 2.0 ** -20), -half))
    rows = []
    for e in (-140, -126, -125, -60, 0, 3, 100, 125):
        for top in (6.0, 7.0, 7.0 * (1 + 2.0 ** -22), 1.75 * 4 * (1 - 2.0 ** -23)):
            rows.append(torch.cat((around[:31], torch.tensor([top], dtype=torch.float64))) * 2.0 ** e)
    rows.append(torch.full((32,), 3.4e38, dtype=torch.float64))
    rows.append(torch.zeros(32, dtype=torch.float64))
    w = torch.stack(rows).float()
    data, scale = quantize_weight_fp4(w.to(dev))
    codes, s = O.quantize(w)
    assert torch.equal(O.scale_values(scale.cpu()), s)
    assert torch.equal(data.cpu(), O.pack(codes))


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_quantizer_not_finite(dev, dtype, bad):
    from atma_amd.kernel import dequantize_weight_fp4, linear_fp4, quantize_weight_fp4
    w = torch.randn(4, 128, generator=torch.Generator().manual_seed(1)).to(dtype)
    clean = quantize_weight_fp4(w.to(dev))
    w[2, 70] = bad
    data, scale = quantize_weight_fp4(w.to(dev))
    assert _bytes(scale)[2, 2] == 255
    v = dequantize_weight_fp4(data, scale, F32).cpu()
    assert v[2, 64:96].isnan().all() and v.isnan().sum() == 32
    same = torch.ones(4, 4, dtype=torch.bool)
    same[2, 2] = False
    assert torch.equal(_bytes(scale)[same], _bytes(clean[1])[same])
    for rows in (1, 40, 300):
        y = linear_fp4(torch.ones(rows, 128, dtype=BF, device=dev), data, scale)
        assert y[:, 2].isnan().all() and y.isnan().sum() == rows


def test_quantizer_strides_and_no_rows(dev):
    from atma_amd.kernel import dequantize_weight_fp4, quantize_weight_fp4
    w = torch.randn(40, 200, generator=torch.Generator().manual_seed(2)).to(BF)
    want = O.quantize(w[:, 4:132])
    for view in (w.to(dev)[:, 4:132], w.to(dev).t().contiguous().t()[:, 4:132]):
        data, scale = quantize_weight_fp4(view)
        assert torch.equal(data.cpu(), O.pack(want[0])) and torch.equal(O.scale_values(scale.cpu()), want[1])
    wide = torch.zeros(40, 100, dtype=torch.uint8, device=dev)
    wide[:, 3:67] = data
    s = torch.zeros(40, 9, dtype=torch.uint8, device=dev)
    s[:, 5:] = scale.view(torch.uint8)
    v = dequantize_weight_fp4(wide[:, 3:67], s.view(E8)[:, 5:], BF)
    assert torch.equal(v, dequantize_weight_fp4(data, scale, BF))
    data, scale = quantize_weight_fp4(torch.zeros(0, 64, device=dev))
    assert data.shape == (0, 32) and scale.shape == (0, 2) and dequantize_weight_fp4(data, scale).shape == (0, 64)


# ------------------------------------------------------------------------------------------------ products
def _whole(rows, cols, g):
    """x of small whole numbers and the weights' codes and scales (1, 2 or 4): sums are multiples of 0.5 below 2^22."""
    return torch.randint(-4, 5, (rows, cols), generator=g).double()


def _weight(n, k, g, dev, spread=3):
    codes = torch.randint(0, 16, (n, k), generator=g)
    scale = (127 + torch.randint(0, spread, (n, k // 32), generator=g)).to(torch.uint8).view(E8)
    return O.pack(codes).to(dev), scale.to(dev)


def _gate(y):
    a, gate = y.chunk(2, 1)
    return gate * a.clamp_min(0).square()


# (rows, features, K): every number of rows, features and K that leaves a tile, a group or a block of K unfilled
SHAPES = [(1, 1, 32), (1, 16, 64), (1, 100, 288), (1, 1024, 4096), (2, 33, 96), (7, 48, 544), (15, 17, 160), (16, 256, 1024),
          (17, 31, 256), (16, 5000, 512), (31, 130, 992), (32, 64, 2048), (32, 8200, 320), (33, 40, 128), (48, 1000, 1024), (63, 65, 64), (64, 512, 4096),
          (65, 129, 224), (100, 2048, 512), (128, 128, 128), (129, 257, 416), (200, 1001, 2048), (256, 256, 192), (257, 500, 1056),
          (300, 4096, 256), (777, 1001, 512), (1000, 300, 96), (1500, 2600, 64), (2999, 640, 160)]


@pytest.mark.parametrize("rows,n,k", SHAPES)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_products_of_whole_numbers(dev, rows, n, k, dtype):
    from atma_amd.kernel import linear_fp4, linear_gated_fp4
    g = torch.Generator().manual_seed(rows + 7 * n + 13 * k)
    x = _whole(rows, k, g)
    data, scale = _weight(2 * n, k, g, dev, 2)
    w = O.values(data, scale)
    bias = torch.randint(-8, 9, (2 * n,), generator=g).float()
    xd = x.to(dtype).to(dev)
    y, size = O.linear(x, w, bias)
    assert size.max() < 2 ** 22
    for b in (None, bias, bias.to(dtype)):
        want = y if b is not None else y - bias.double()
        got = linear_fp4(xd, data[:n], scale[:n], None if b is None else b[:n].to(dev))
        assert got.dtype == dtype and torch.equal(got.cpu(), want[:, :n].to(dtype))
        a = want[:, :n].clamp_min(0)
        # relu(a)^2 and its product with the gate are rounded in fp32, then once to the output
        act = (want[:, n:].float() * (a.float() * a.float())).to(dtype)
        got = linear_gated_fp4(xd, data, scale, None if b is None else b.to(dev))
        assert torch.equal(got.cpu(), act)


@pytest.mark.parametrize("rows,n,k", [(1, 1024, 4096), (3, 77, 2080), (16, 512, 1024), (32, 300, 4096), (50, 333, 1024),
                                      (130, 260, 2048), (700, 520, 1024), (1, 40, 16384), (300, 64, 8192)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_products(dev, rows, n, k, dtype):
    from atma_amd.kernel import linear_fp4, linear_gated_fp4, quantize_weight_fp4
    g = torch.Generator().manual_seed(rows + n + k)
    x = (torch.randn(rows, k, generator=g) * (1 + 7 * (torch.rand(k, generator=g) < 0.01))).to(dtype)
    data, scale = quantize_weight_fp4((torch.randn(2 * n, k, generator=g) / k ** 0.5).to(dev))
    w = O.values(data, scale)
    bias = (0.1 * torch.randn(2 * n, generator=g)).to(dtype)
    y, size = O.linear(x, w, bias)
    noise = (k + 1) * 2.0 ** -23 * (size + bias.double().abs())
    got = linear_fp4(x.to(dev), data[:n], scale[:n], bias[:n].to(dev)).cpu().double()
    err = (got - y[:, :n]).abs()
    assert (err <= HALF[dtype] * y[:, :n].abs() + noise[:, :n] * (1 + HALF[dtype])).all(), err.max()
    # over many values: a rounding's error is at most HALF / sqrt(3) of the value rms; fp32 sums are far below
    rms = (err.square().sum() / y[:, :n].square().sum()).sqrt()
    print(f"rms error {rms:.2e}", flush=True)
    assert rms <= HALF[dtype] / 3 ** 0.5 * 1.05 + 2.0 ** -20
    a, gate = y[:, :n].clamp_min(0), y[:, n:]
    want, da, dg = gate * a.square(), noise[:, :n], noise[:, n:]
    got = linear_gated_fp4(x.to(dev), data, scale, bias.to(dev)).cpu().double()
    # d(gate a^2) <= a^2 dgate + 2 |gate| a da + second order; two fp32 products; the output's rounding (fp16: or half its least step)
    allowed = (a + da).square() * dg + gate.abs() * (2 * a + da) * da + 2.0 ** -23 * want.abs()
    allowed = allowed * (1 + HALF[dtype]) + HALF[dtype] * want.abs() + 2.0 ** -25
    assert ((got - want).abs() <= allowed).all(), ((got - want).abs() / allowed).max()


@pytest.mark.parametrize("rows", [1, 20, 40, 300])
def test_far_scales_and_fp16_limits(dev, rows):
    """Scales over the whole range in bf16; in fp16 the weights as ``dequantize_weight_fp4`` gives them."""
    from atma_amd.kernel import dequantize_weight_fp4, linear_fp4
    g = torch.Generator().manual_seed(3)
    codes = torch.randint(0, 16, (96, 64), generator=g)
    codes[:, 32:] = 0
    for dtype, lo, hi in ((BF, 2, 200), (HF, 96, 143)):
        sc = torch.randint(lo, hi, (96, 2), generator=g).to(torch.uint8).view(E8)
        data = O.pack(codes).to(dev)
        x = torch.zeros(rows, 64)
        x[:, 5] = 1   # one product a sum: the weight itself
        y = linear_fp4(x.to(dtype).to(dev), data, sc.to(dev)).cpu()
        v = dequantize_weight_fp4(data, sc.to(dev), dtype).cpu()
        assert torch.equal(v, O.values(data, sc).to(dtype))
        want = v[:, 5].expand(rows, 96)
        inf = v[:, :32].isinf().any(1)   # (0 times an infinite weight is NaN)
        assert torch.equal(y[:, ~inf], want[:, ~inf])


@pytest.mark.parametrize("rows", [1, 9, 40, 130, 300])
@pytest.mark.parametrize("name", ["linear_fp4", "linear_gated_fp4"])
def test_strides(dev, rows, name):
    """Rows apart, views that start anywhere, scales and biases at any byte, rows of a transposed matrix."""
    import atma_amd.kernel as kernel
    f = getattr(kernel, name)
    g = torch.Generator().manual_seed(4)
    n, k = 70, 160
    x = torch.randn(rows, k, generator=g).to(BF).to(dev)
    data, scale = _weight(n, k, g, dev)
    bias = torch.randn(n, generator=g).to(BF).to(dev)
    want = f(x, data, scale, bias)
    wide = torch.full((rows, k + 24), float("nan"), dtype=BF, device=dev)
    for at in (8, 3):
        wide[:, at:at + k] = x
        assert torch.equal(f(wide[:, at:at + k], data, scale, bias), want)
    assert torch.equal(f(x.t().contiguous().t(), data, scale, bias), want)
    assert torch.equal(f(x[:1].expand(rows, k), data, scale, bias), want[:1].expand_as(want))
    wd = torch.full((n, k // 2 + 48), 0x77, dtype=torch.uint8, device=dev)
    for at in (16, 5):
        wd[:, at:at + k // 2] = data
        assert torch.equal(f(x, wd[:, at:at + k // 2], scale, bias), want)
    ws = torch.full((n, 11), 255, dtype=torch.uint8, device=dev)
    ws[:, 3:8] = scale.view(torch.uint8)
    assert torch.equal(f(x, data, ws.view(E8)[:, 3:8], bias), want)
    held = torch.full((2 * n + 1,), float("nan"), dtype=BF, device=dev)
    held[1:n + 1] = bias
    assert torch.equal(f(x, data, scale, held[1:n + 1]), want)
    held[1::2] = bias
    assert torch.equal(f(x, data, scale, held[1::2]), want)


@pytest.mark.parametrize("name", ["linear_fp4", "linear_gated_fp4"])
def test_no_rows_grad_and_devices(dev, name):
    import atma_amd.kernel as kernel
    f = getattr(kernel, name)
    g = torch.Generator().manual_seed(5)
    data, scale = _weight(32, 64, g, dev)
    out = f(torch.zeros(0, 64, dtype=BF, device=dev), data, scale)
    assert out.shape == (0, 32 if name == "linear_fp4" else 16)
    x = torch.zeros(2, 64, dtype=BF, device=dev, requires_grad=True)
    with pytest.raises(RuntimeError, match="inference"):
        f(x, data, scale)
    with torch.no_grad():
        f(x, data, scale)
    with pytest.raises(RuntimeError, match="GPU only"):
        f(x.detach(), data.cpu(), scale)


@pytest.mark.parametrize("rows", [1, 33, 300])
def test_nothing_behind_the_rows(dev, rows):
    """Outputs of a call lie between rows of other values, which stay."""
    from atma_amd import _lib
    g = torch.Generator().manual_seed(6)
    n, k, ld = 37, 96, 41
    x = _whole(rows, k, g).to(BF).to(dev)
    data, scale = _weight(2 * n, k, g, dev)
    for gated in (False, True):
        y = torch.full((rows + 2, ld), -7.0, dtype=BF, device=dev)
        f = _lib.load().atma_linear_gated_fp4 if gated else _lib.load().atma_linear_fp4
        rc = f(x.data_ptr(), k, data.data_ptr(), k // 2, scale.data_ptr(), k // 32, None, 0, y[1].data_ptr() + 2, ld, rows, n, k,
               _lib.ATMA_BF16, _lib.stream_handle(dev))
        _lib.check(rc, "linear")
        full, _ = O.linear(x.cpu(), O.values(data, scale))
        want = torch.full((rows + 2, ld), -7.0, dtype=BF)
        a, gate = full[:, :n].clamp_min(0).float(), full[:, n:].float()
        want[1:rows + 1, 1:n + 1] = (gate * (a * a) if gated else full[:, :n]).to(BF)
        assert torch.equal(y.cpu(), want)


def test_streams_graphs_and_compile(dev):
    """On another stream, captured and replayed with new inputs, and through torch.compile."""
    from atma_amd.kernel import linear_fp4, linear_gated_fp4, quantize_weight_fp4
    g = torch.Generator().manual_seed(7)
    up = quantize_weight_fp4(torch.randn(256, 64, generator=g).to(dev))
    down = quantize_weight_fp4(torch.randn(64, 128, generator=g).to(dev))

    def mlp(x):
        return linear_fp4(linear_gated_fp4(x, *up), *down)

    xs = [torch.randn(24, 64, generator=g).to(BF).to(dev) for _ in range(3)]
    want = [mlp(x) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mlp(xs[0])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want[0])
    held = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mlp(held)
    for i in (1, 2, 0, 1):
        held.copy_(xs[i])
        graph.replay()
        assert torch.equal(out, want[i])
    compiled = torch.compile(mlp, backend="aot_eager")
    with torch.no_grad():
        assert torch.equal(compiled(xs[2]), want[2])
