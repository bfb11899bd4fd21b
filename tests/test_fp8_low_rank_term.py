"""Half a low-rank term is refused by ``residual_rms_norm_fp8`` as its other arguments are."""

import pytest
import torch

from atma_amd.kernel import residual_rms_norm_fp8
from atma_amd.kernel.decode_fusions import PartialSums


def test_low_rank_term_without_weights():
    bf = torch.bfloat16
    w, mx, mw = torch.ones(64, dtype=bf), torch.zeros(2, 8, dtype=bf), torch.zeros(64, 8, dtype=bf)
    for x, y in ((mx, None), (mx[0], mw), (mx, mw[:32]), (mx[:1], mw), (mx.float(), mw), (mx[:, :6], mw[:, :6])):
        with pytest.raises(ValueError, match="low-rank"):
            residual_rms_norm_fp8(PartialSums(torch.zeros(3, 2, 64), mu_x=x, mu_w=y, dtype=bf), None, w, 1e-6)
    with pytest.raises(RuntimeError, match="GPU only"):
        residual_rms_norm_fp8(PartialSums(torch.zeros(3, 2, 64), mu_x=mx, mu_w=mw, dtype=bf), None, w, 1e-6)
