"""Oracle of the 8-bit inference operators (no reference counterpart): plain float64 torch on the CPU.

An 8-bit tensor is e4m3fn values times a power-of-two scale for each 128 values of a row (``tall`` 1) or each 128 x 128
block (``tall`` 128); the functions return the values and the scales apart, both float64."""

import torch

BLOCK, TOP = 128, 448.0


def round_e4m3(x):
    """The e4m3fn value nearest to x (ties to even), |x| <= 448 or NaN: steps of 2^(e - 3) from 2^e on, 2^-9 below 2^-6."""
    _, e = torch.frexp(x.abs().clamp_min(2.0 ** -6))
    step = torch.exp2((e - 1 - 3).double())
    return torch.round(x / step) * step


def scales(x, tall=1):
    """(ceil(rows / tall), ceil(K / 128)): the smallest 2^e, e in [-126, 120], with the block's finite magnitudes <= 448 2^e."""
    rows, K = x.shape
    a = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    out = torch.empty((rows + tall - 1) // tall, (K + BLOCK - 1) // BLOCK, dtype=torch.float64)
    for i in range(out.shape[0]):
        for j in range(out.shape[1]):
            top, e = a[i * tall:(i + 1) * tall, j * BLOCK:(j + 1) * BLOCK].max().item(), -126
            while e < 120 and top > TOP * 2.0 ** e:
                e += 1
            out[i, j] = 2.0 ** e
    return out


def spread(s, rows, K, tall=1):
    """One scale a value."""
    return s.repeat_interleave(tall, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :K]


def quantize(x, tall=1):
    x = x.double()
    s = scales(x, tall)
    q = x / spread(s, *x.shape, tall)
    return torch.where(torch.isfinite(x), round_e4m3(q), torch.full_like(x, float("nan"))), s


def values(data, scale, tall=1):
    """The float64 values of a float8_e4m3fn / float8_e8m0fnu pair."""
    data, scale = data.cpu(), scale.cpu()
    return data.float().double() * spread(torch.exp2(scale.contiguous().view(torch.uint8).double() - 127), *data.shape, tall)


def linear(x, w, bias=None):
    """(x w^T + bias, sum |x| |w|^T) of float64 values: the product and the size of what it adds."""
    y = x @ w.t()
    return (y if bias is None else y + bias.double()), x.abs() @ w.abs().t()


def gated(y):
    a, gate = y.chunk(2, 1)
    return gate * a.clamp_min(0).square()


def residual_norm(branch, residual, weight, eps, dtype):
    """(norm, stream): the stream rounded to ``dtype``, its norm in float64."""
    s = branch if residual is None else (residual.double() + branch.double()).to(dtype)
    f = s.double()
    return f * torch.rsqrt(f.square().mean(1, keepdim=True) + eps) * weight.double(), s
