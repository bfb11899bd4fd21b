"""8-bit products of rows that start more than 8 MiB apart (the last token of each long sequence, a single row of a wide
tensor): as the call on a copy."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 2, 5])
def test_products_of_far_rows(dev, rows):
    from atma_amd.kernel import linear_fp8, linear_gated_fp8, quantize_fp8, quantize_weight_fp8
    K, T = 144, 1 << 16   # sequences of 9 MiB
    g = torch.Generator().manual_seed(rows)
    x, xs = quantize_fp8(torch.randn(rows, K, generator=g).to(dev))
    w, ws = quantize_weight_fp8(torch.randn(256, K, generator=g).to(dev))
    h = torch.zeros(rows, T, K, dtype=torch.uint8, device=dev).view(x.dtype)
    h[:, -1].view(torch.uint8).copy_(x.view(torch.uint8))
    far = h[:, -1]
    assert far.stride(0) > 1 << 23
    assert torch.equal(linear_fp8(far, xs, w, ws), linear_fp8(x, xs, w, ws))
    for a, b in zip(linear_gated_fp8(far, xs, w, ws), linear_gated_fp8(x, xs, w, ws)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    # the weight's rows as far apart
    v, vs = w[:rows], ws[:1]
    far_w = torch.zeros(rows, 1 << 24, dtype=torch.uint8, device=dev).view(w.dtype)[:, :K]
    far_w.view(torch.uint8).copy_(v.view(torch.uint8))
    assert torch.equal(linear_fp8(x, xs, far_w, vs), linear_fp8(x, xs, v, vs))
