"""4-bit weights whose scales no quantizer gives: 2^-127 and 2^-126 (their values are subnormal in bfloat16 and fp32) and 2^126 and
2^127 (4 and 6 times the first, and 2 and more times the second, are infinities there).  The documents allow any scale.

Each output of the products is one weight times a power of two (no other term), so it is exact."""

import pytest
import torch

from oracle import fp4 as O

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
E8 = torch.float8_e8m0fnu


@pytest.mark.parametrize("code", [0, 1, 2, 126, 252, 253, 254, 255])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_dequantized(dev, code, dtype):
    from atma_amd.kernel import dequantize_weight_fp4
    data = torch.arange(256, dtype=torch.uint8).view(4, 64)
    scale = torch.full((4, 4), code, dtype=torch.uint8).view(E8)
    got, want = dequantize_weight_fp4(data.to(dev), scale.to(dev), dtype).cpu(), O.values(data, scale).to(dtype)
    if code == 255:
        assert got.isnan().all()
    else:
        assert torch.equal(got, want)


# kernel, rows, features, K, gated: each kernel of the products once
SHAPES = [(0, 5, 100, 544, False), (1, 130, 520, 4128, False), (2, 7, 16500, 2080, False), (3, 200, 16500, 2080, False),
          (4, 777, 2300, 1056, False), (5, 257, 8200, 1056, False), (6, 1000, 8200, 544, False), (7, 300, 530, 96, False),
          (8, 257, 4100, 1056, False), (0, 5, 100, 544, True), (5, 300, 4100, 1056, True), (6, 500, 8200, 544, True),
          (8, 63, 4100, 1056, True)]


@pytest.mark.parametrize("form,rows,n,k,gated", SHAPES)
@pytest.mark.parametrize("codes,power", [((0, 1), 100), ((253, 254), -100)], ids=["low", "high"])
def test_products(dev, form, rows, n, k, gated, codes, power):
    from atma_amd import _lib
    from atma_amd.kernel import linear_fp4, linear_gated_fp4
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        lib = _lib.load()
        assert (lib.atma_linear_gated_fp4_form if gated else lib.atma_linear_fp4_form)(rows, n, k) == form
    g = torch.Generator().manual_seed(rows + n + k)
    outs = 2 * n if gated else n
    # magnitudes up to 6, and with the large scales up to 1.5: finite
    nibble = lambda: (torch.randint(0, 4 if power < 0 else 8, (outs, k // 2), generator=g)   # noqa: E731
                      + 8 * torch.randint(0, 2, (outs, k // 2), generator=g))
    data = (nibble() + 16 * nibble()).to(torch.uint8)
    scale = torch.tensor(codes, dtype=torch.uint8)[torch.randint(0, 2, (outs, k // 32), generator=g)].view(E8)
    at = torch.randint(0, k, (rows,), generator=g)
    x = torch.zeros(rows, k, dtype=BF)
    x[torch.arange(rows), at] = 2.0 ** power
    want = O.values(data, scale)[:, at].t() * 2.0 ** power
    if gated:
        want = want[:, n:] * want[:, :n].clamp_min(0).square()
    got = (linear_gated_fp4 if gated else linear_fp4)(x.to(dev), data.to(dev), scale.to(dev)).cpu()
    assert torch.equal(got.double(), want)
