"""Oracle of the 4-bit weights (no reference counterpart): plain float64 torch on the CPU."""

import torch

GROUP = 32
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def scales(w):
    """(N, K / 32) float64: the smallest 2^e, e in [-125, 125], with the group's magnitudes <= 7 2^e; NaN where one is not finite."""
    top = w.double().abs().view(w.shape[0], -1, GROUP).amax(2)
    out = torch.empty_like(top)
    for i in range(top.shape[0]):
        for j in range(top.shape[1]):
            t, e = top[i, j].item(), -125
            while e < 125 and t > 7 * 2.0 ** e:
                e += 1
            out[i, j] = 2.0 ** e
    return torch.where(top.isfinite(), out, torch.full_like(top, float("nan")))


def nearest(a):
    """The position in GRID of the value nearest to a >= 0; half way goes to the even position."""
    grid = torch.tensor(GRID, dtype=torch.float64)
    d = (a.unsqueeze(-1) - grid).abs()
    d = d + torch.where(torch.arange(8) % 2 == 0, 0.0, 1e-9)   # (the differences of neighbours are 0.5 and more)
    return d.argmin(-1)


def quantize(w):
    """(codes (N, K) 0 to 15, scales (N, K / 32) float64)."""
    w = w.double()
    s = scales(w)
    a = w.abs() / s.repeat_interleave(GROUP, 1)
    return nearest(a) + 8 * torch.signbit(w).long(), s


def pack(codes):
    return (codes[:, ::2] + 16 * codes[:, 1::2]).to(torch.uint8)


def unpack(data):
    return torch.stack((data & 15, data >> 4), 2).flatten(1).long()


def scale_values(scale):
    code = scale.contiguous().view(torch.uint8).double()
    return torch.where(code == 255, torch.full_like(code, float("nan")), torch.exp2(code - 127))


def values(data, scale):
    """The float64 values of a (data, scale) pair."""
    grid = torch.tensor(GRID, dtype=torch.float64)
    grid = torch.cat((grid, -grid))
    return grid[unpack(data.cpu())] * scale_values(scale.cpu()).repeat_interleave(GROUP, 1)


def linear(x, w, bias=None):
    """(x w^T + bias, sum |x| |w|^T) of float64 values."""
    y = x.double() @ w.t()
    return (y if bias is None else y + bias.double()), x.double().abs() @ w.abs().t()
