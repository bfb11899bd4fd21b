"""Rows of an 8-bit product's operands that start far apart: what the C ABI takes, and what the Python calls copy."""

import ctypes

import pytest
import torch

from atma_amd import _lib, _ops

FAR = 1 << 24   # bytes


def _call(lib, gated, **kw):
    ptr = ctypes.cast(ctypes.create_string_buffer(256), ctypes.c_void_p)
    ptr = ctypes.c_void_p((ptr.value + 63) // 64 * 64)
    a = dict(ldx=144, ldw=144, M=1, N=256)
    a.update(kw)
    # (a bias type that is refused behind the checks of the strides: nothing is launched)
    head = (ptr, a["ldx"], ptr, 4, ptr, a["ldw"], ptr, 4, ptr, 9, ptr, 256)
    if gated:
        return lib.atma_linear_gated_fp8(*head, ptr, 2, a["M"], a["N"], 144, None)
    return lib.atma_linear_fp8(*head, a["M"], a["N"], 144, 1, None)


@pytest.mark.parametrize("gated", [False, True])
def test_the_stride_of_one_row_is_not_used(gated):
    lib = _lib.load()
    for ld in (0, 7, 128, FAR, -16):
        assert _call(lib, gated, ldx=ld) == 2 and b"dtype" in lib.atma_last_error()
        assert _call(lib, gated, ldx=ld, M=2) != 0 and b"rows" in lib.atma_last_error()
    if not gated:
        assert _call(lib, gated, ldw=FAR, N=1) == 2 and b"dtype" in lib.atma_last_error()
    assert _call(lib, gated, ldw=FAR) == 2 and b"8 MiB" in lib.atma_last_error()


def test_far_rows_are_copied():
    x = torch.empty_strided((3, 144), (FAR, 1), dtype=torch.uint8)
    x.copy_(torch.arange(3 * 144).view(3, 144) % 251)
    y = _ops._rows_near(x)
    assert torch.equal(x, y) and 144 <= y.stride(0) <= 1 << 23 and y.data_ptr() % 16 == 0
    near = torch.zeros(3, 1 << 23, dtype=torch.uint8)[:, :144]
    assert _ops._rows_near(near) is near
