"""Each kernel of the products with 4-bit weights (``atma_linear_fp4_form``, ``atma_linear_gated_fp4_form``) at sizes that leave its
tiles, its blocks of K and its workgroups' last rounds unfilled.  Products of small whole numbers, whose fp32 sums are exact in
any order: the output is the float64 one, rounded.  Rows of x, w and scales lie between values that would show (NaN, 6 and the
scale NaN), rows of y between others that stay."""

import pytest
import torch

from oracle import fp4 as O

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
E8 = torch.float8_e8m0fnu

# form, rows, features, K
FORMS = [(0, 5, 100, 544), (0, 17, 1, 4128), (0, 777, 100, 1056),
         (1, 50, 2300, 2080), (1, 130, 520, 4128), (1, 1000, 100, 4128),
         (2, 1, 8200, 4128), (2, 7, 16500, 2080), (2, 1000, 300, 1056),
         (3, 3, 50304, 96), (3, 17, 50304, 32), (3, 31, 50304, 1056), (3, 200, 16500, 2080),
         (4, 777, 2300, 1056), (4, 1025, 9, 32), (4, 1041, 1100, 288), (4, 4097, 4100, 96),
         (5, 100, 16500, 288), (5, 257, 8200, 1056), (5, 500, 4100, 288), (5, 4097, 520, 288),
         (6, 200, 50304, 288), (6, 1000, 8200, 544), (6, 2001, 4100, 1056),
         (7, 31, 16500, 1056), (7, 300, 530, 96), (7, 300, 2300, 1056), (7, 1000, 300, 544), (7, 1025, 1, 96),
          (7, 2001, 1, 1056), (7, 4097, 100, 4128),
         (8, 33, 16500, 4128), (8, 100, 8200, 1056), (8, 257, 4100, 1056), (8, 4097, 300, 4128)]
GATED = [(0, 5, 100, 544), (0, 16, 1, 4128), (0, 1000, 100, 2080),
         (5, 70, 8200, 96), (5, 300, 4100, 1056), (5, 1041, 1001, 288),
         (6, 500, 8200, 544), (6, 1000, 4100, 544), (6, 2049, 2300, 1056),
         (8, 63, 4100, 1056), (8, 300, 1001, 544), (8, 1025, 1, 32), (8, 1030, 70, 96), (8, 2001, 1, 1056),
          (8, 4097, 100, 4128)]


def _run(dev, form, rows, n, k, dtype, gated):
    from atma_amd import _lib
    from atma_amd.kernel import linear_fp4, linear_gated_fp4
    lib = _lib.load()
    got = (lib.atma_linear_gated_fp4_form if gated else lib.atma_linear_fp4_form)(rows, n, k)
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:   # (another card has other borders)
        assert got == form, f"{rows} x {k} -> {n} reaches kernel {got}, not {form}"
    g = torch.Generator(device=dev).manual_seed(rows + 3 * n + 7 * k)
    outs = 2 * n if gated else n
    x = torch.full((rows + 1, k + 16), float("nan"), dtype=dtype, device=dev)
    x[:rows, 8:k + 8] = torch.randint(-4, 5, (rows, k), generator=g, device=dev).to(dtype)
    data = torch.full((outs + 1, k // 2 + 32), 0x77, dtype=torch.uint8, device=dev)
    data[:outs, 16:k // 2 + 16] = torch.randint(0, 256, (outs, k // 2), generator=g, device=dev, dtype=torch.uint8)
    scale = torch.full((outs + 1, k // 32 + 3), 255, dtype=torch.uint8, device=dev)
    scale[:outs, 1:k // 32 + 1] = torch.randint(126, 129, (outs, k // 32), generator=g, device=dev).to(torch.uint8)
    x, data, scale = x[:rows, 8:k + 8], data[:outs, 16:k // 2 + 16], scale.view(E8)[:outs, 1:k // 32 + 1]
    bias = torch.randint(-8, 9, (outs,), generator=g, device=dev).float()
    out = (linear_gated_fp4 if gated else linear_fp4)(x, data, scale, bias)
    # every term is a multiple of 1/4 of at most 4 * 12: sums below 2^22 / 4 are exact in fp32
    assert k * 48 + 8 < 2 ** 22 / 4
    values = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device=dev)
    w = torch.stack([values[(data & 15).long()], values[(data >> 4).long()]], 2).reshape(outs, k)
    w *= torch.exp2(scale.view(torch.uint8).double() - 127).repeat_interleave(32, 1)
    assert torch.equal(w[:1].cpu(), O.values(data[:1], scale[:1]))
    y = x.double() @ w.t() + bias.double()
    if gated:
        a = y[:, :n].clamp_min(0).float()
        y = y[:, n:].float() * (a * a)
    assert torch.equal(out, y.to(dtype))
    # the same call through the C entry, into rows apart
    held = torch.full((rows + 2, n + 5), -7.0, dtype=dtype, device=dev)
    entry = lib.atma_linear_gated_fp4 if gated else lib.atma_linear_fp4
    _lib.check(entry(x.data_ptr(), x.stride(0), data.data_ptr(), data.stride(0), scale.data_ptr(), scale.stride(0), bias.data_ptr(),
                     _lib.ATMA_F32, held[1:, 3:].data_ptr(), n + 5, rows, n, k, _lib.ATMA_BF16 if dtype == BF else _lib.ATMA_F16,
                     _lib.stream_handle(dev)), "linear")
    assert torch.equal(held[1:rows + 1, 3:n + 3], out)
    held[1:rows + 1, 3:n + 3] = -7.0
    assert (held == -7).all()


@pytest.mark.parametrize("form,rows,n,k", FORMS)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_forms(dev, form, rows, n, k, dtype):
    _run(dev, form, rows, n, k, dtype, False)


@pytest.mark.parametrize("form,rows,n,k", GATED)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_gated_forms(dev, form, rows, n, k, dtype):
    _run(dev, form, rows, n, k, dtype, True)
