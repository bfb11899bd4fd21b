"""``residual_rms_norm_fp8`` in the form that a prefill gives it (a 16-bit base, three biases and the low-rank term, from
8,192 rows on eight rows a wave) and with values that are not finite.

The stream is ``residual_rms_norm``'s, bit for bit, and near the float64 sum: a base, three biases and a term of up to 16 products in fp32
(fewer than 32 roundings of 2^-24 of the largest of them, which is below 2^-18 of what they add in magnitude), rounded to the
branch's type (half a step), the residual added and rounded again.  The norm is that of the stream: within half an e4m3 step of its
float64 value, 2^-16 of it more for the fp32 arithmetic before, and the scale equal but within 2^-16 of a border."""

import pytest
import torch

from oracle import fp8 as O

pytestmark = pytest.mark.gpu

DT = [torch.bfloat16, torch.float16]
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _g(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _randn(dev, seed, *shape):
    return torch.randn(*shape, generator=_g(dev, seed), device=dev)


def _scales(h):
    """``oracle.fp8.scales`` of rows of finite values, without its loops (|h| far above the smallest scale, or 0)."""
    top = torch.nn.functional.pad(h.abs(), (0, -h.shape[1] % 128)).view(h.shape[0], -1, 128).amax(2)
    _, e = torch.frexp(top / 448)
    e = torch.where(top <= 448 * torch.exp2((e - 1).double()), e - 1, e)
    e = torch.where(top > 448 * torch.exp2(e.double()), e + 1, e)
    return torch.exp2(torch.where(top > 0, e, torch.full_like(e, -126)).double())


def _near(data, scale, h):
    s = torch.exp2(scale.contiguous().view(torch.uint8).double() - 127)
    exact = _scales(h)
    for t in (1 - 2.0 ** -16, 1 + 2.0 ** -16):
        exact = torch.where(s == exact, exact, _scales(h * t))
    assert torch.equal(s, exact)
    full = O.spread(s, *h.shape)
    v = data.float().double() * full
    bound = torch.maximum(2.0 ** -4 * h.abs(), 2.0 ** -10 * full) * (1 + 2.0 ** -6) + 2.0 ** -16 * h.abs()
    assert not torch.isnan(v).any() and ((v - h).abs() <= bound).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,dim,mu", [(1, 1024, 8), (33, 2048, 16), (777, 1040, 4), (8191, 256, 8), (8192, 1024, 8),
                                         (8205, 656, 16), (16389, 144, 4), (9001, 4096, 8), (8193, 1024, 0)])
def test_prefill_form(dev, rows, dim, mu, dtype):
    from atma_amd.kernel import residual_rms_norm_fp8
    from atma_amd.kernel.decode_fusions import PartialSums, residual_rms_norm
    # the base as a slice of wider rows, as a projection's output may be
    base = _randn(dev, 1, rows, dim + 16).to(dtype)[:, :dim]
    biases = [_randn(dev, 2 + i, dim).to(dtype) for i in range(3)]
    res = (4 * _randn(dev, 6, rows, dim)).to(dtype)
    w = (1 + 0.1 * _randn(dev, 7, dim)).to(dtype)
    mx, mw = (_randn(dev, 8, rows, mu).to(dtype), _randn(dev, 9, dim, mu).to(dtype)) if mu else (None, None)
    ps = PartialSums(None, biases, mu_x=mx, mu_w=mw, dtype=dtype, base=base)
    terms = [base.double(), *(b.double().expand(rows, dim) for b in biases)]
    add, size = sum(terms), sum(t.abs() for t in terms)
    if mu:
        add = add + mx.double() @ mw.double().t().contiguous()
        size = size + mx.double().abs() @ mw.double().abs().t().contiguous()
    for r in (res, None):   # joining a stream, starting one
        data, scale, stream = residual_rms_norm_fp8(ps, r, w, 1e-6)
        assert torch.equal(stream, residual_rms_norm(ps, r, w, 1e-6)[1])
        branch_off = HALF[dtype] * add.abs() + 2.0 ** -18 * size
        exact = add if r is None else r.double() + add
        off = branch_off * (1 + HALF[dtype]) + (0 if r is None else HALF[dtype] * exact.abs())
        assert ((stream.double() - exact).abs() <= off).all()
        f = stream.double()
        _near(data, scale, f * torch.rsqrt(f.square().mean(1, keepdim=True) + 1e-6) * w.double())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,dim", [(9, 144), (40, 1024), (12, 4096)])
def test_values_that_are_not_finite(dev, rows, dim, dtype):
    """A NaN takes its row, whose scales are then the smallest; an infinity is NaN in its place and the rest of its row 0; the
    other rows are as without them.  An infinite gain is NaN in its column (0 inf, inf) and in no block's scale."""
    from atma_amd.kernel import residual_rms_norm_fp8
    x, res = _randn(dev, 1, rows, dim).to(dtype), _randn(dev, 2, rows, dim).to(dtype)
    w = (1 + 0.1 * _randn(dev, 3, dim)).to(dtype)
    want, ws, _ = residual_rms_norm_fp8(x, res, w, 1e-6)
    x, res = x.clone(), res.clone()
    inf, nan = float("inf"), float("nan")
    x[1, 3], res[2, dim - 1], x[4, 17] = nan, nan, inf
    res[5, 100], x[5, 101] = -inf, inf
    x[rows - 1, 7], res[rows - 1, 7] = inf, -inf     # their sum is NaN
    data, scale, stream = residual_rms_norm_fp8(x, res, w, 1e-6)
    assert torch.equal(torch.nan_to_num(stream), torch.nan_to_num((x.float() + res.float()).to(dtype)))
    assert torch.equal(torch.isnan(stream), torch.isnan(x + res))
    d, codes = data.float(), scale.view(torch.uint8)
    for row in (1, 2, rows - 1):
        assert torch.isnan(d[row]).all()
    for row, at in ((4, [17]), (5, [100, 101])):
        assert torch.isnan(d[row, at]).all() and torch.isnan(d[row]).sum() == len(at)
        assert (torch.nan_to_num(d[row]) == 0).all()
    bad = [1, 2, 4, 5, rows - 1]
    assert (codes[bad] == 1).all()
    keep = [i for i in range(rows) if i not in bad]
    assert torch.equal(data.view(torch.uint8)[keep], want.view(torch.uint8)[keep])
    assert torch.equal(codes[keep], ws.view(torch.uint8)[keep])
    w2, w0 = w.clone(), w.clone()
    w2[9], w0[9] = inf, 0
    data, scale, _ = residual_rms_norm_fp8(x, res, w2, 1e-6)
    want, ws, _ = residual_rms_norm_fp8(x, res, w0, 1e-6)
    d, other = data.float(), [i for i in range(dim) if i != 9]
    assert torch.isnan(d[:, 9]).all() and torch.equal(scale.view(torch.uint8), ws.view(torch.uint8))
    assert torch.equal(torch.nan_to_num(d[:, other]), torch.nan_to_num(want.float()[:, other]))
