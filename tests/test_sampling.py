"""The sampler where no GPU is needed: refusals, at the Python entry point and at the C ABI, and the oracle's own rules."""

import ctypes
import math

import pytest
import torch

from atma_amd import _lib
from oracle import sampling as O


def test_refusals():
    from atma_amd.kernel import sample_tokens
    logits, u = torch.zeros(4, 10), torch.zeros(4)
    for bad in (torch.zeros(10), torch.zeros(4, 0), torch.zeros(4, 10, dtype=torch.float64), torch.zeros(1, (1 << 20) + 1)):
        with pytest.raises(ValueError):
            sample_tokens(bad, u)
    for bad in (torch.zeros(3), torch.zeros(4, 1), torch.zeros(4, dtype=torch.float64)):
        with pytest.raises(ValueError, match="uniform"):
            sample_tokens(logits, bad)
    for name, dtype in (("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32),
                        ("min_p", torch.float32)):
        for bad in (torch.zeros(3, dtype=dtype), torch.zeros(4, dtype=torch.float64), "1", True):
            with pytest.raises(ValueError, match=name):
                sample_tokens(logits, u, **{name: bad})
    with pytest.raises(ValueError, match="top_k"):
        sample_tokens(logits, u, top_k=1.5)
    with pytest.raises(RuntimeError, match="GPU only"):
        sample_tokens(logits, u)


def test_c_refusals():
    lib = _lib.load()
    buf = ctypes.create_string_buffer(64)
    at = ctypes.addressof(buf) // 8 * 8 + 8

    def sample(logits=at, ld=10, uniform=at, ids=at, rows=4, V=10, dtype=_lib.ATMA_BF16):
        return lib.atma_sample_tokens(logits, ld, uniform, None, 1.0, None, 0, None, 1.0, None, 0.0, ids, rows, V, dtype, None)

    assert sample(dtype=5) == 2 and sample(V=0) == 2 and sample(V=(1 << 20) + 1) == 2 and sample(rows=-1) == 2
    assert sample(logits=None) == 1 and sample(uniform=None) == 1 and sample(ids=None) == 1
    assert sample(logits=at + 1) == 1 and sample(ld=9) == 1
    assert sample(rows=0, logits=None) == 0


def test_oracle_rules():
    x = [0.0, 2.0, 1.0, 2.0, -math.inf]
    assert list(O.kept(x, 1.0)) == [1, 3, 2, 0, 4]
    assert list(O.kept(x, 1.0, k=1)) == [1] and list(O.kept(x, 1.0, k=3)) == [1, 3, 2]
    assert list(O.kept([0.0] * 4, 1.0, p=0.5)) == [0, 1] and list(O.kept([0.0] * 4, 1.0, p=0.51)) == [0, 1, 2]
    assert list(O.kept(x, 1.0, p=0.0)) == [1] and list(O.kept(x, 1.0, m=1.0)) == [1, 3] and list(O.kept(x, 1.0, m=0.2)) == [1, 3, 2]
    assert O.draw([0.0] * 4, 0.5, 1.0) == 2 and O.draw([0.0] * 4, 0.49, 1.0) == 1 and O.draw(x, 0.99, 0.0) == 1
    assert O.draw([1.0, math.nan, math.inf], 0.0, 1.0) == 1 and O.draw([-math.inf] * 3, 0.5, 1.0) == 1
    assert O.draw([0.0, math.inf, math.inf], 0.7, 1.0) == 2 and O.draw(x, 1.0, 1.0) == 3 and O.draw(x, math.nan, 1.0) == 0


def test_workspace_of_shared_rows():
    """Asked without a launch; a workspace that is too small, or misaligned, is refused before one."""
    from atma_amd import _lib
    lib = _lib.load()
    size = lib.atma_sample_tokens_workspace
    assert size(1, 50304, _lib.ATMA_F32) > 0 and size(1, 50304, _lib.ATMA_BF16) == 0 and size(1, 65536, _lib.ATMA_BF16) > 0
    assert size(2048, 50304, _lib.ATMA_F32) == 0 and size(1, 1000, _lib.ATMA_F32) == 0
    assert size(4, 50304, _lib.ATMA_F32) == 4 * size(1, 50304, _lib.ATMA_F32)
    for bad in ((0, 50304, 0), (-1, 50304, 0), (1, 0, 0), (1, (1 << 20) + 1, 0), (1, 50304, 77)):
        assert size(*bad) == 0
    need = size(1, 50304, _lib.ATMA_F32)
    call = lambda at, n: lib.atma_sample_tokens_in(64, 50304, 64, None, 1.0, None, 0, None, 1.0, None, 0.0, 64, 1, 50304,   # noqa: E731
                                                   _lib.ATMA_F32, at, n, None)
    assert call(64, need - 1) == call(60, need) == 1   # invalid
