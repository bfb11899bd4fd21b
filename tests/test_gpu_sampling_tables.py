"""16-bit rows that keep many tokens, some of the border's value among them: the weights come from tables where no top-k is asked
for or it keeps more than 512, and the border's tokens are counted beside them."""

import pytest
import torch

from tests.test_gpu_sampling import BF, HF, _check, _logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [4097, 20000, 65535])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("filters", ["k", "kp", "km", "kpm"])
def test_wide_top_k(dev, V, dtype, filters):
    g = torch.Generator().manual_seed(V)
    ks = [511, 512, 513, 1500, 4000, V - 1]
    rows = len(ks)
    # spread logits around 0, all positive, all negative: both signs of the tables
    logits = _logits(g, rows, V) + torch.tensor([0.0, 0.0, 20.0, -20.0, 0.0, 0.0])[:, None]
    u = torch.rand(rows, generator=g)
    u[3:] = 1 - u[3:] ** 4   # late in the row
    t = [0.7, 1.0, 1.3, 1.0, 2.5, 1.0]
    p = [0.95, 0.999, 0.8, 0.99, 0.9, 0.9999]
    m = [1e-3, 1e-4, 0.02, 1e-6, 0.01, 1e-5]
    _check(dev, logits.to(dtype), u.tolist(), t, ks, p if "p" in filters else None, m if "m" in filters else None, doubtful=1)
