"""Whether a row is shared by workgroups is the library's rule; the Python call leaves the question out where the answer is known.
No GPU: the two agree over sizes around every border."""

import pytest
import torch

from atma_amd import _lib, _ops

CODES = {torch.float32: _lib.ATMA_F32, torch.bfloat16: _lib.ATMA_BF16, torch.float16: _lib.ATMA_F16}


class Asked:
    """The library's answers, without its launches."""

    def __init__(self, lib):
        self.lib, self.given = lib, None

    def atma_sample_tokens_workspace(self, *args):
        return self.lib.atma_sample_tokens_workspace(*args)

    def atma_sample_tokens_in(self, *args):
        self.given = args[-2]
        return 0


@pytest.mark.parametrize("dtype", list(CODES))
def test_no_shared_row_goes_without_its_workspace(monkeypatch, dtype):
    lib = _lib.load()
    asked, shared = Asked(lib), 0
    monkeypatch.setattr(_lib, "load", lambda: asked)
    monkeypatch.setattr(_lib, "stream_handle", lambda device: None)
    ids = torch.zeros(1, dtype=torch.int64)
    for V in (1, 4096, 16384, 31744, 32000, 32001, 32256, 32257, 32768, 33000, 50304, 65535, 65536, 65537, 131072, 1 << 20):
        for rows in (1, 2, 15, 16, 17, 31, 32, 33, 39, 63, 64, 65, 128, 255, 256, 257, 2048):
            logits = torch.empty(1, 1, dtype=dtype).expand(rows, V)
            _ops.sample_into(ids, logits, torch.zeros(1), None, 1.0, None, 0, None, 1.0, None, 0.0)
            need = lib.atma_sample_tokens_workspace(rows, V, CODES[dtype])
            assert asked.given == need, (rows, V)
            shared += need > 0
    assert shared
