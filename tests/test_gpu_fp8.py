"""The 8-bit inference operators (``kernel/fp8.py``) against float64 (``oracle/fp8.py``).

Tolerances, all derived:

* the quantizers are exact: inputs of 16 or 32 bits, power-of-two scales, one rounding -- equal to the oracle;
* a quantized norm or activation h: within half an e4m3 step of the exact value, max(2^-4 |h|, 2^-10 scale), a relative
  2^-16 of it more for the fp32 arithmetic before, and the scale equal unless the block's largest value is within 2^-16 of the
  border;
* a product: half a step of the output type (bf16 2^-8, fp16 2^-11, relative) plus what the matrix instruction drops: each
  of the eight products that it aligns to the largest loses less than 2^-13 of that one, at most 8 * 2^-13 of the sum of
  magnitudes."""

import pytest
import torch

from oracle import fp8 as O

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DROP = 2.0 ** -10
DT = [torch.bfloat16, torch.float16]


def _g(seed):
    return torch.Generator().manual_seed(seed)


def _rows(rows, dim, seed, dtype=torch.float32):
    """Rows of different size, some channels large, one row of zeros."""
    g = _g(seed)
    x = torch.randn(rows, dim, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))
    x = x * (1 + 15 * (torch.rand(dim, generator=g) < 0.02))
    if rows > 2:
        x[1] = 0
    return x.to(dtype)


def _codes(scale):
    return scale.cpu().contiguous().view(torch.uint8)


def _same_codes(scale, exact):
    assert scale.dtype == torch.float8_e8m0fnu
    assert torch.equal(_codes(scale), (torch.log2(exact) + 127).to(torch.uint8))


def _same(data, exact):
    d = data.cpu().float().double()
    assert torch.equal(torch.isnan(d), torch.isnan(exact))
    assert torch.equal(torch.nan_to_num(d), torch.nan_to_num(exact))


def _near_quantized(data, scale, h):
    """data, scale against the exact h."""
    s = torch.exp2(_codes(scale).double() - 127)
    exact = O.scales(h)
    for t in (1 - 2.0 ** -16, 1 + 2.0 ** -16):   # equal, or the largest value on the border
        exact = torch.where(s == exact, exact, O.scales(h * t))
    assert torch.equal(s, exact)
    full = O.spread(s, *h.shape)
    v = data.cpu().float().double() * full
    bound = torch.maximum(2.0 ** -4 * h.abs(), 2.0 ** -10 * full) * (1 + 2.0 ** -6) + 2.0 ** -16 * h.abs()
    assert not torch.isnan(v).any() and ((v - h).abs() <= bound).all()


# ------------------------------------------------------------------------------------------------ quantizers
@pytest.mark.parametrize("dtype", [torch.float32, *DT])
@pytest.mark.parametrize("rows,dim", [(1, 16), (3, 112), (5, 128), (17, 144), (4, 640), (33, 1024), (2, 4112)])
def test_quantize_rows(dev, rows, dim, dtype):
    from atma_amd.kernel import quantize_fp8
    x = _rows(rows, dim, rows + dim, dtype)
    data, scale = quantize_fp8(x.to(dev))
    q, s = O.quantize(x)
    assert data.shape == (rows, dim) and data.dtype == torch.float8_e4m3fn and scale.shape == s.shape
    _same(data, q)
    _same_codes(scale, s)


@pytest.mark.parametrize("dtype", [torch.float32, *DT])
@pytest.mark.parametrize("rows,dim", [(1, 16), (127, 128), (129, 144), (256, 272), (300, 1024)])
def test_quantize_weight(dev, rows, dim, dtype):
    from atma_amd.kernel import quantize_weight_fp8
    x = (_rows(rows, dim, rows * dim) * 0.02).to(dtype)
    data, scale = quantize_weight_fp8(x.to(dev))
    q, s = O.quantize(x, 128)
    assert scale.shape == s.shape
    _same(data, q)
    _same_codes(scale, s)


@pytest.mark.parametrize("weight", [False, True])
def test_quantize_extreme_values(dev, weight):
    """The ends of the scales' range, subnormals, borders of a scale, ties, infinities and NaN beside ordinary values."""
    from atma_amd.kernel import quantize_fp8, quantize_weight_fp8
    x = torch.randn(8, 128, generator=_g(5))
    x[0], x[1] = 3.4028234e38, 1e-42
    x[2, :4] = torch.tensor([448.0, 449.0, 17.0, 19.0])
    x[3, 0], x[4, 0] = 448.0000305, 447.99997
    x[5, 0], x[5, 1], x[5, 2] = float("inf"), float("-inf"), float("nan")
    x[6] = float("nan")
    x[7] = torch.arange(128) * 2.0 ** -10
    if weight:
        x = torch.cat([x[2:], torch.zeros(2, 128)])
        x[4] = torch.nan_to_num(x[4], 1.0)
    data, scale = (quantize_weight_fp8 if weight else quantize_fp8)(x.to(dev))
    q, s = O.quantize(x, 128 if weight else 1)
    _same(data, q)
    _same_codes(scale, s)


def test_quantize_strided_and_empty(dev):
    """Rows of a wider tensor, at odd offsets, transposed, broadcast; no rows."""
    from atma_amd.kernel import quantize_fp8, quantize_weight_fp8
    big = _rows(40, 700, 3).to(dev)
    for x in (big[:, :256], big[3:29:2, 1:145], big.bfloat16()[:, 3:163], big.t()[:144, :32], big[0].expand(6, 700)[:, :640]):
        for f, tall in ((quantize_fp8, 1), (quantize_weight_fp8, 128)):
            data, scale = f(x)
            q, s = O.quantize(x.cpu(), tall)
            _same(data, q)
            _same_codes(scale, s)
    data, scale = quantize_fp8(big[:0, :256])
    assert data.shape == (0, 256) and scale.shape == (0, 2)


# ------------------------------------------------------------------------------------------------ the norm
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,dim", [(1, 16), (7, 112), (33, 128), (5, 640), (12, 1024), (3, 2064), (9, 4096)])
def test_residual_norm(dev, rows, dim, dtype):
    from atma_amd.kernel import residual_rms_norm_fp8
    branch, res = _rows(rows, dim, dim, dtype), _rows(rows, dim, dim + 1, dtype)
    w = (1 + 0.1 * torch.randn(dim, generator=_g(2))).to(dtype)
    data, scale, stream = residual_rms_norm_fp8(branch.to(dev), res.to(dev), w.to(dev), 1e-6)
    h, s = O.residual_norm(branch, res, w, 1e-6, dtype)
    assert torch.equal(stream.cpu(), s)
    _near_quantized(data, scale, h)
    start = branch.to(dev)
    data, scale, stream = residual_rms_norm_fp8(start, None, w.to(dev), 1e-6)
    assert stream is start
    _near_quantized(data, scale, O.residual_norm(branch, None, w, 1e-6, dtype)[0])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,parts,mu", [(1, 1, 0), (8, 4, 0), (5, 8, 8), (32, 2, 16)])
def test_residual_norm_partial_sums(dev, rows, parts, mu, dtype):
    """Partial sums with biases and the low-rank term: the stream is residual_rms_norm's, the norm that of the stream."""
    from atma_amd.kernel import residual_rms_norm_fp8
    from atma_amd.kernel.decode_fusions import PartialSums, residual_rms_norm
    g, D = _g(rows), 1024
    p = torch.randn(parts, rows, D, generator=g).to(dev)
    b = [torch.randn(D, generator=g).to(dtype).to(dev) for _ in range(2)]
    res, w = _rows(rows, D, 4, dtype).to(dev), (1 + 0.1 * torch.randn(D, generator=g)).to(dtype).to(dev)
    mx, mw = (torch.randn(rows, mu, generator=g).to(dtype).to(dev), torch.randn(D, mu, generator=g).to(dtype).to(dev)) if mu \
        else (None, None)
    ps = PartialSums(p, b, mu_x=mx, mu_w=mw, dtype=dtype)
    for r in (res, None):   # joining a stream, starting one
        data, scale, stream = residual_rms_norm_fp8(ps, r, w, 1e-6)
        assert torch.equal(stream, residual_rms_norm(ps, r, w, 1e-6)[1])
        _near_quantized(data, scale, O.residual_norm(stream.cpu(), None, w.cpu(), 1e-6, dtype)[0])


def test_residual_norm_strided_and_empty(dev):
    from atma_amd.kernel import residual_rms_norm_fp8
    big = _rows(20, 600, 9, torch.bfloat16).to(dev)
    w = torch.ones(256, dtype=torch.bfloat16, device=dev)
    for branch, res in ((big[:10, :256], big[10:, 8:264]), (big[:10, 1:257], big[10:, 3:259]),
                        (big[0, :256].expand(4, 256), big[1:5, :256])):
        data, scale, stream = residual_rms_norm_fp8(branch, res, w, 1e-6)
        h, s = O.residual_norm(branch.cpu(), res.cpu(), w.cpu(), 1e-6, torch.bfloat16)
        assert torch.equal(stream.cpu(), s)
        _near_quantized(data, scale, h)
    data, scale, stream = residual_rms_norm_fp8(big[:0, :256], big[:0, :256], w, 1e-6)
    assert data.shape == stream.shape == (0, 256) and scale.shape == (0, 2)


# ------------------------------------------------------------------------------------------------ products
def _operands(dev, M, N, K, seed):
    """An 8-bit x and weight and their float64 values."""
    from atma_amd.kernel import quantize_fp8, quantize_weight_fp8
    x, xs = quantize_fp8(_rows(M, K, seed).to(dev))
    w, ws = quantize_weight_fp8((_rows(N, K, seed + 1) / K ** 0.5).to(dev))
    return x, xs, w, ws, O.values(x, xs), O.values(w, ws, 128)


def _near_product(y, exact, size):
    err = (y.cpu().double() - exact).abs()
    assert (err <= HALF[y.dtype] * exact.abs() + DROP * size + torch.finfo(y.dtype).smallest_normal).all(), \
        (err / (exact.abs() + size).clamp_min(1e-30)).max().item()


SHAPES = [(1, 1, 16), (1, 1024, 4096), (2, 7, 128), (16, 40, 144), (17, 129, 272), (31, 1001, 1024), (32, 128, 112),
          (33, 16, 128), (33, 129, 1040), (64, 256, 640), (100, 257, 2048), (129, 1000, 384), (257, 130, 1024),
          (300, 512, 528), (700, 72, 896),
          # more than one tile of features a workgroup for few rows, and tiles for them; each tile shape, one and two
          # tiles a workgroup, one block of K
          (9, 6200, 144), (20, 6150, 272), (5, 12300, 128), (2000, 1000, 528), (2100, 2001, 528), (4000, 4001, 272),
          (8100, 4090, 272), (4100, 4097, 80),
          # few rows in groups of 32: features in sixteens and in two sixteens, long K, waves without a block, the last
          # group of one token, past the split's borders
          (64, 1024, 4096), (250, 500, 1552), (97, 2500, 272), (65, 8190, 144), (129, 1001, 16), (33, 40, 8208),
          (30, 12288, 400), (16, 24570, 144), (15, 24577, 144), (65, 8193, 144)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear(dev, M, N, K, dtype):
    from atma_amd.kernel import linear_fp8
    x, xs, w, ws, xv, wv = _operands(dev, M, N, K, M + N + K)
    exact, size = O.linear(xv, wv)
    y = linear_fp8(x, xs, w, ws, out_dtype=dtype)
    assert y.shape == (M, N) and y.dtype == dtype and y.is_contiguous()
    _near_product(y, exact, size)
    for bt in (dtype, torch.float32):
        b = torch.randn(N, generator=_g(1)).to(bt)
        _near_product(linear_fp8(x, xs, w, ws, b.to(dev), out_dtype=dtype), exact + b.double(), size)


@pytest.mark.parametrize("M,H,K", [(1, 128, 16), (1, 4096, 1024), (9, 256, 144), (16, 384, 1040), (32, 128, 2048),
                                   (33, 128, 128), (64, 256, 272), (100, 640, 1024), (129, 128, 384), (300, 512, 640),
                                   (2001, 1024, 272), (770, 4096, 144), (4201, 2048, 144), (4090, 2048, 912),
                                   (8190, 2048, 912),
                                   # few rows: all of K in LDS and one block more, the last group of one token, the
                                   # largest grid and past it
                                   (3, 256, 4608), (17, 256, 4624), (128, 4096, 80), (129, 4096, 80), (500, 1024, 272),
                                   (1, 32896, 144)])
@pytest.mark.parametrize("bias", [None, torch.bfloat16, torch.float32])
def test_linear_gated(dev, M, H, K, bias):
    from atma_amd.kernel import linear_gated_fp8
    x, xs, w, ws, xv, wv = _operands(dev, M, 2 * H, K, M + H + K)
    b = None if bias is None else torch.randn(2 * H, generator=_g(1)).to(bias)
    y, size = O.linear(xv, wv, b)
    data, scale = linear_gated_fp8(x, xs, w, ws, None if b is None else b.to(dev))
    assert data.shape == (M, H) and scale.shape == (M, H // 128)
    # what the instruction drops in a and gate reaches h = gate relu(a)^2 to first order, and its square
    a, gate = y.chunk(2, 1)
    da, dg = (DROP * size).chunk(2, 1)
    h, pos = O.gated(y), a.clamp_min(0)
    dh = dg * (pos + da).square() + gate.abs() * (2 * pos + da) * da
    s = torch.exp2(_codes(scale).double() - 127)
    full = O.spread(s, M, H)
    v = data.cpu().float().double() * full
    bound = torch.maximum(2.0 ** -4 * (h.abs() + dh), 2.0 ** -10 * full) * (1 + 2.0 ** -6) + dh
    assert not torch.isnan(v).any() and ((v - h).abs() <= bound).all()
    top, slack = h.abs().reshape(M, -1, 128).amax(2), dh.reshape(M, -1, 128).amax(2)
    low = O.scales((top - slack).clamp_min(0).reshape(-1, 1)).reshape(M, -1)
    high = O.scales((top + slack).reshape(-1, 1)).reshape(M, -1)
    assert ((s >= low) & (s <= high)).all()


@pytest.mark.parametrize("M", [5, 40, 300])
def test_products_leave_rows_apart(dev, M):
    """A row of zeros gives the bias; a NaN value, an infinite one before quantizing and a NaN scale reach their row only."""
    from atma_amd.kernel import linear_fp8, linear_gated_fp8, quantize_fp8
    _, _, w, ws, _, wv = _operands(dev, 4, 256, 272, 1)
    x = _rows(M, 272, 8)
    x[0], x[2, 140], x[3, 7] = 0, float("nan"), float("inf")
    x8, xs = quantize_fp8(x.to(dev))
    xs.view(torch.uint8)[4, 1] = 255   # a NaN scale
    b = torch.randn(256, generator=_g(2)).bfloat16()
    y = linear_fp8(x8, xs, w, ws, b.to(dev)).cpu()
    keep = [i for i in range(M) if i not in (2, 3, 4)]
    assert torch.isnan(y[[2, 3, 4]]).all() and torch.equal(y[0], b)
    exact, size = O.linear(O.values(x8, xs)[keep], wv, b)
    _near_product(y[keep], exact, size)
    data, scale = linear_gated_fp8(x8, xs, w, ws)
    d = data.cpu().float()
    assert torch.isnan(d[[2, 3, 4]]).all() and not torch.isnan(d[keep]).any() and (d[0] == 0).all()
    assert (_codes(scale)[[0, 2, 3, 4]] == 1).all()


@pytest.mark.parametrize("M", [3, 50, 260])
def test_products_at_other_layouts(dev, M):
    """x and weight as slices of wider or misaligned tensors, broadcast rows, scales contiguous, transposed and at odd
    offsets: equal to the same call on fresh tensors.  The bytes behind K and behind the last scale are not used."""
    from atma_amd.kernel import linear_fp8, linear_gated_fp8
    K = 1040   # nine blocks: contiguous scales have rows of 9 bytes
    x, xs, w, ws, _, _ = _operands(dev, M, 256, K, 6)
    want, (gd, gs) = linear_fp8(x, xs, w, ws), linear_gated_fp8(x, xs, w, ws)

    def wide(t, off, value):
        u = t.view(torch.uint8)
        held = torch.full((u.shape[0] + 1, (u.shape[1] + 63) // 16 * 16), value, dtype=torch.uint8, device=dev)
        held[:u.shape[0], off:off + u.shape[1]] = u
        return held.view(t.dtype)[:u.shape[0], off:off + u.shape[1]]

    def turned(t):
        return t.view(torch.uint8).t().contiguous().t().view(t.dtype)

    for x2, xs2, w2, ws2 in ((wide(x, 0, 127), wide(xs, 0, 255), wide(w, 16, 127), wide(ws, 4, 255)),
                             (wide(x, 5, 127), xs.contiguous(), wide(w, 3, 127), ws.contiguous()),
                             (turned(x), turned(xs), turned(w), turned(ws)),
                             (x, wide(xs, 1, 255), w, wide(ws, 2, 255))):
        assert torch.equal(linear_fp8(x2, xs2, w2, ws2), want)
        d, s = linear_gated_fp8(x2, xs2, w2, ws2)
        assert torch.equal(d.view(torch.uint8), gd.view(torch.uint8)) and torch.equal(_codes(s), _codes(gs))
    one = linear_fp8(x[:1].expand(M, K), xs[:1].expand(M, 9), w, ws)
    assert torch.equal(one, one[:1].expand_as(one))


def test_quantize_more_rows_than_a_launch_holds(dev):
    """67 million short rows: the rows at the seam of two launches and the last ones as in a call of their own."""
    from atma_amd.kernel import quantize_fp8
    M, seam = 67_108_900, 4 * (2 ** 24 - 1)
    x = torch.zeros(M, 16, dtype=torch.bfloat16, device=dev)
    parts = [slice(0, 7), slice(seam - 5, seam + 9), slice(M - 30, M)]
    for i, p in enumerate(parts):
        x[p] = _rows(p.stop - p.start, 16, i, torch.bfloat16).to(dev)
    data, scale = quantize_fp8(x)
    for p in parts:
        d, s = quantize_fp8(x[p].clone())
        assert torch.equal(data[p].view(torch.uint8), d.view(torch.uint8))
        assert torch.equal(scale[p].view(torch.uint8), s.view(torch.uint8))
    assert (scale.view(torch.uint8)[10:seam - 10] == 1).all()


def test_one_row_at_any_stride(dev):
    """A single row whose row stride says nothing (expanded, shorter than the row): x, weight, residual, quantizer input."""
    from atma_amd.kernel import linear_fp8, quantize_fp8, quantize_weight_fp8, residual_rms_norm_fp8
    x, xs, w, ws, _, _ = _operands(dev, 1, 1, 144, 3)
    want = linear_fp8(x, xs, w, ws)
    for stride in (0, 1, 16):
        one = lambda t: t.as_strided(t.shape, (stride, 1))   # noqa: E731
        assert torch.equal(linear_fp8(one(x), one(xs), one(w), one(ws)), want)
        v = _rows(1, 144, 5, torch.bfloat16).to(dev)
        for f in (quantize_fp8, quantize_weight_fp8):
            assert torch.equal(f(one(v))[0].view(torch.uint8), f(v)[0].view(torch.uint8))
        g = torch.ones(144, dtype=torch.bfloat16, device=dev)
        assert torch.equal(residual_rms_norm_fp8(one(v), one(v), g, 1e-6)[2], residual_rms_norm_fp8(v, v, g, 1e-6)[2])


@pytest.mark.parametrize("M", [3, 50, 300])
def test_products_with_a_bias_anywhere(dev, M):
    """A bias at an odd offset, with a stride, expanded: equal to the call on a fresh copy."""
    from atma_amd.kernel import linear_fp8, linear_gated_fp8
    x, xs, w, ws, _, _ = _operands(dev, M, 256, 144, 4)
    held = torch.randn(600, generator=_g(1)).bfloat16().to(dev)
    for b in (held[1:257], held[3:515:2], held[7].expand(256)):
        assert torch.equal(linear_fp8(x, xs, w, ws, b), linear_fp8(x, xs, w, ws, b.clone()))
        for p, q in zip(linear_gated_fp8(x, xs, w, ws, b), linear_gated_fp8(x, xs, w, ws, b.clone())):
            assert torch.equal(p.view(torch.uint8), q.view(torch.uint8))
    for bad in (float("-inf"), float("nan")):   # a pruned feature (0 after the activation), a lost one
        b = torch.zeros(256)
        b[5] = bad
        data, scale = linear_gated_fp8(x, xs, w, ws, b.to(dev))
        d = data.cpu().float()
        clean = linear_gated_fp8(x, xs, w, ws, torch.zeros(256, device=dev))
        assert (d[:, 5] == 0).all() if bad == float("-inf") else torch.isnan(d[:, 5]).all()
        assert not torch.isnan(torch.cat([d[:, :5], d[:, 6:]], 1)).any() and scale.shape == clean[1].shape


def test_products_of_no_rows(dev):
    from atma_amd.kernel import linear_fp8, linear_gated_fp8
    x, xs, w, ws, _, _ = _operands(dev, 4, 256, 128, 1)
    assert linear_fp8(x[:0], xs[:0], w, ws).shape == (0, 256)
    d, s = linear_gated_fp8(x[:0], xs[:0], w, ws)
    assert d.shape == (0, 128) and s.shape == (0, 1)


def test_offsets_past_32_bits(dev):
    """Rows of x more than 4 GiB behind its start, rows of y more than 4 GiB, quantizer inputs of more than 4 GiB."""
    from atma_amd.kernel import linear_fp8, quantize_fp8
    M, pitch, K, N = 9000, 1 << 19, 144, 256
    x, xs, w, ws, _, _ = _operands(dev, 64, N, K, 2)
    big = torch.zeros(M * pitch, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn).view(M, pitch)
    rows = torch.tensor([0, 255, 4096, 8191, 8192, 8447, M - 1], device=dev)
    big.view(torch.uint8)[rows, :K] = x[:7].view(torch.uint8)
    bs = torch.full((M, 4), 127, dtype=torch.uint8, device=dev)
    bs[rows, :2] = xs[:7].view(torch.uint8)
    want = linear_fp8(x, xs, w, ws)[:7]
    y = linear_fp8(big[:, :K], bs.view(torch.float8_e8m0fnu)[:, :2], w, ws)
    assert torch.equal(y[rows], want) and y.abs().sum(1).ne(0).sum() <= 7
    del big, y
    M, N = 44000, 50304
    x, xs, w, ws, _, _ = _operands(dev, 8, N, 128, 3)
    y = linear_fp8(x.view(torch.uint8).repeat(M // 8, 1).view(torch.float8_e4m3fn),
                   xs.contiguous().view(torch.uint8).repeat(M // 8, 1).view(torch.float8_e8m0fnu), w, ws)
    want = linear_fp8(x, xs, w, ws)
    for at in (0, 21344, M - 8):
        assert torch.equal(y[at:at + 8], want)
    del y
    big = torch.zeros(9000, 1 << 18, dtype=torch.bfloat16, device=dev)
    v = _rows(7, 144, 4, torch.bfloat16).to(dev)
    big[rows, :144] = v
    data, scale = quantize_fp8(big[:, :144])
    d, s = quantize_fp8(v)
    assert torch.equal(data[rows].view(torch.uint8), d.view(torch.uint8)) and torch.equal(_codes(scale[rows]), _codes(s))


# ------------------------------------------------------------------------------------------------ together
def _chain(branch, res, w, fc, proj):
    from atma_amd.kernel import linear_fp8, linear_gated_fp8, residual_rms_norm_fp8
    h, hs, stream = residual_rms_norm_fp8(branch, res, w, 1e-6)
    a, as_ = linear_gated_fp8(h, hs, *fc)
    return linear_fp8(a, as_, *proj, out_dtype=branch.dtype), stream


def _chain_operands(dev, rows, seed):
    from atma_amd.kernel import quantize_weight_fp8
    g = _g(seed)
    fc = (*quantize_weight_fp8((torch.randn(1024, 256, generator=g) / 16).to(dev)), torch.randn(1024, generator=g).bfloat16().to(dev))
    proj = (*quantize_weight_fp8((torch.randn(256, 512, generator=g) / 23).to(dev)), torch.randn(256, generator=g).bfloat16().to(dev))
    w = torch.ones(256, dtype=torch.bfloat16, device=dev)
    return _rows(rows, 256, seed, torch.bfloat16).to(dev), _rows(rows, 256, seed + 1, torch.bfloat16).to(dev), w, fc, proj


@pytest.mark.parametrize("rows", [1, 32, 200])
def test_chain_follows_the_exact_mlp(dev, rows):
    """Norm, gated projection and second projection as a served block runs them, against float64 of the 8-bit weights:
    three roundings of activations to 8 bits (2^-4 at most each, 0.026 rms) enter h, whose square doubles them."""
    branch, res, w, fc, proj = _chain_operands(dev, rows, 3)
    y, stream = _chain(branch, res, w, fc, proj)
    h, s = O.residual_norm(branch.cpu(), res.cpu(), w.cpu(), 1e-6, torch.bfloat16)
    a, _ = O.linear(h, O.values(*fc[:2], 128), fc[2].cpu())
    exact, _ = O.linear(O.gated(a), O.values(*proj[:2], 128), proj[2].cpu())
    assert torch.equal(stream.cpu(), s)
    assert ((y.cpu().double() - exact).norm() / exact.norm()).item() <= 4 * 0.026


def test_chain_captured_and_on_another_stream(dev):
    """Captured into a graph and replayed with other inputs and eager work between; on a side stream; both equal."""
    branch, res, w, fc, proj = _chain_operands(dev, 40, 5)
    want = _chain(branch, res, w, fc, proj)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _chain(branch, res, w, fc, proj)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    static = branch.clone()
    with torch.cuda.graph(graph):
        out = _chain(static, res, w, fc, proj)
    for i in range(4):
        static.copy_(branch * (i + 1))
        graph.replay()
        eager = _chain(branch * (i + 1), res, w, fc, proj)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


@pytest.mark.parametrize("rows", [5, 200])
def test_chain_compiles_as_one_graph(dev, rows):
    branch, res, w, fc, proj = _chain_operands(dev, rows, 5)
    want = _chain(branch, res, w, fc, proj)
    compiled = torch.compile(_chain, fullgraph=True, backend="aot_eager")
    with torch.no_grad():
        got = compiled(branch, res, w, fc, proj)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_calls_under_modes_and_subclasses_are_dispatched(dev):
    """What watches torch calls sees the operators; a subclass is not launched past."""
    from torch.utils._python_dispatch import TorchDispatchMode
    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    branch, res, w, fc, proj = _chain_operands(dev, 5, 5)
    want = _chain(branch, res, w, fc, proj)
    with Watch():
        got = _chain(branch, res, w, fc, proj)
    for name in ("residual_rms_norm_fp8", "linear_gated_fp8", "linear_fp8"):
        assert any(f"atma_hip.{name}" in s for s in seen)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_same_bits_every_time(dev):
    """Nothing depends on the order in which workgroups run: calls repeat bit for bit."""
    branch, res, w, fc, proj = _chain_operands(dev, 300, 7)
    first = _chain(branch, res, w, fc, proj)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, _chain(branch, res, w, fc, proj)))


# ------------------------------------------------------------------------------------------------ the MLP and the engine
def _mlp(dev, dim, dtype=torch.bfloat16, seed=0):
    from atma_amd.layers.global_attention import MLP
    torch.manual_seed(seed)
    return MLP(dim).to(dtype).to(dev)


def _exact_mlp(m, h):
    a, _ = O.linear(h, O.values(m.fc_weight.view(torch.float8_e4m3fn), m.fc_scale.view(torch.float8_e8m0fnu), 128), m.fc_bias.cpu())
    y, _ = O.linear(O.gated(a), O.values(m.proj_weight.view(torch.float8_e4m3fn), m.proj_scale.view(torch.float8_e8m0fnu), 128),
                    m.proj_bias.cpu())
    return y


@pytest.mark.parametrize("dtype", DT)
def test_mlp_module(dev, dtype):
    """``Fp8MLP`` of rows and of batches, against float64 of its 8-bit weights (two roundings of activations to 8 bits, the
    first one doubled by the square, 0.026 rms each); ``half()`` leaves the weights alone; grad mode without leaves works,
    with one is refused."""
    from atma_amd.layers.global_attention import Fp8MLP
    m = Fp8MLP(_mlp(dev, 256, dtype))
    assert m.fc_weight.dtype == torch.uint8 and m.half().fc_weight.dtype == torch.uint8
    m = Fp8MLP(_mlp(dev, 256, dtype))
    x = torch.randn(3, 50, 256, generator=_g(1)).to(dtype)
    y = m(x.to(dev))
    assert y.shape == x.shape and y.dtype == dtype
    exact = _exact_mlp(m, x.double().view(-1, 256))
    assert ((y.cpu().double().view(-1, 256) - exact).norm() / exact.norm()).item() <= 4 * 0.026
    assert torch.equal(m(x[1].to(dev)), y[1]) and torch.equal(m(x.to(dev), defer=True), y)
    with pytest.raises(ValueError):
        m(x.to(dev).float())
    with pytest.raises(RuntimeError, match="inference"):
        m(x.to(dev).requires_grad_())


def test_block_stream_takes_the_fused_norm(dev):
    """The decoder block's stream route quantizes in the norm; a hook on the MLP, which it would not call, sends it through
    the modules, whose norm is rounded to 16 bits on the way."""
    from atma_amd.engine.model import Atma
    from atma_amd.engine import AtmaConfig
    hf = AtmaConfig(vocab_size=64, num_hidden_layers=1, hidden_size=256, head_dim=64)
    block = Atma(hf).init_weights(0.05, 1).to(dev, torch.bfloat16).quantize_mlps().blocks[0]
    with torch.no_grad():
        block.norm1.weight.fill_(1), block.norm2.weight.fill_(1)
    block.attn = torch.nn.Identity()
    block.attn.forward = lambda h, defer=False: h
    x, res = (torch.randn(9, 256, generator=_g(i)).bfloat16().to(dev) for i in (1, 2))
    with torch.no_grad():
        y, s = block.forward_stream(x, res)
        h, s1 = block.norm1.add_norm(x, res)
        data, scale, s2 = block.norm2.add_norm_fp8(h, s1)
        assert torch.equal(s, s2) and torch.equal(y, block.mlp.forward_fp8(data, scale, torch.bfloat16))
        calls = []
        handle = block.mlp.register_forward_hook(lambda *a: calls.append(1))
        y2, s3 = block.forward_stream(x, res)
        handle.remove()
        assert calls == [1] and torch.equal(s3, s2)
        exact = _exact_mlp(block.mlp, O.residual_norm(s2.cpu(), None, torch.ones(256), 1e-6, torch.bfloat16)[0])
        for out in (y, y2):
            assert ((out.cpu().double() - exact).norm() / exact.norm()).item() <= 4 * 0.026


def test_block_wider_than_the_fused_norm(dev):
    """Rows of more than 4,096 are normed by the module and quantized by the MLP."""
    from atma_amd.engine import AtmaConfig
    from atma_amd.engine.model import AtmaDecoderBlock
    from atma_amd.layers.global_attention import Fp8MLP
    D = 4160
    with torch.device(dev), torch.no_grad():
        block = AtmaDecoderBlock(0, AtmaConfig(vocab_size=64, num_hidden_layers=1, hidden_size=D, head_dim=64)).bfloat16()
        block.mlp = Fp8MLP(block.mlp)
        block.norm1.weight.fill_(1), block.norm2.weight.fill_(1)
        block.attn = torch.nn.Identity()
        block.attn.forward = lambda h, defer=False: h
        x, res = (torch.randn(5, D, generator=_g(i), device="cpu").bfloat16().to(dev) for i in (1, 2))
        y, s = block.forward_stream(x, res)
        h, s1 = block.norm1.add_norm(x, res)
        h, s2 = block.norm2.add_norm(h, s1)
        assert torch.equal(s, s2) and torch.equal(y, block.mlp(h))


def test_engine_with_8_bit_mlps(dev):
    """A greedy generation with ``Config.fp8_mlp``: every prefill and decode step near the whole-model oracle on the 8-bit
    weights' values.  Each of the four blocks' MLP branches is off by 4 * 0.026 of itself at most (above) and no larger than
    the stream it joins, coherently 4 * 0.104 in all, and the 16-bit route adds 5e-2.  Captured decode equals eager."""
    from atma_amd.engine import Config, LLMEngine
    from oracle import model as OM
    from tests.test_gpu_engine import _drive, _model, _prompts
    runs = []
    for eager in (True, False):
        hf, model, sd = _model(torch.bfloat16)
        cfg = Config(kvcache_block_size=16, max_num_seqs=4, max_num_batched_tokens=4096, max_model_len=160,
                     num_kvcache_blocks=64, enforce_eager=eager, hf_config=hf, fp8_mlp=True)
        engine = LLMEngine(cfg, model=model)
        runs.append(_drive(engine, _prompts([17, 40, 129], 2), new_tokens=4)[1])
        engine.exit()
    for a, b in zip(*runs):
        assert a[3] == b[3] and torch.equal(a[2], b[2])
    for i, b in enumerate(model.blocks):
        for n in ("fc", "proj"):
            sd[f"blocks.{i}.mlp.{n}.weight"] = O.values(getattr(b.mlp, n + "_weight").view(torch.float8_e4m3fn),
                                                       getattr(b.mlp, n + "_scale").view(torch.float8_e8m0fnu), 128)
    kw = dict(num_layers=hf.num_hidden_layers, H=hf.num_attention_heads, Hkv=hf.num_key_value_heads, dk=hf.head_dim)
    for is_prefill, hist, logits, _ in runs[0]:
        for row, h in enumerate(hist):
            ref = OM.atma_logits(sd, torch.tensor(h)[None], **kw)[0, -1]
            assert ((logits[row].double() - ref).norm() / ref.norm()).item() <= 4 * 0.104 + 5e-2, (is_prefill, len(h))
