"""The 8-bit operators where no GPU is needed: refusals, at the Python entry points and at the C ABI, and the wait states of
the products' copies into LDS."""

import ctypes
import subprocess

import pytest
import torch

from atma_amd import _build, _lib
from tests.test_copy_hazards import check_assembly

FP8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _x(rows, cols, dtype=FP8):
    return torch.zeros(rows, cols).to(dtype)


def _s(rows, n):
    return torch.full((rows, n), 127, dtype=torch.uint8).view(E8)


def test_refusals():
    from atma_amd.kernel import (linear_fp8, linear_gated_fp8, quantize_fp8, quantize_weight_fp8,
                                 residual_rms_norm_fp8)
    for f in (quantize_fp8, quantize_weight_fp8):
        for bad in (torch.zeros(4), torch.zeros(4, 24), torch.zeros(4, 0), torch.zeros(4, 16, dtype=torch.float64),
                    torch.zeros(2, 4, 16)):
            with pytest.raises(ValueError):
                f(bad)
        with pytest.raises(RuntimeError, match="GPU only"):
            f(torch.zeros(4, 16))
    bf = torch.bfloat16
    norm = [torch.zeros(2, 64, dtype=bf), torch.zeros(2, 64, dtype=bf), torch.zeros(64, dtype=bf)]
    for i, bad in ((0, torch.zeros(2, 64)), (0, torch.zeros(2, 2, 64, dtype=bf)), (1, torch.zeros(3, 64, dtype=bf)),
                   (1, torch.zeros(2, 64)), (2, torch.zeros(32, dtype=bf)), (2, torch.zeros(64))):
        with pytest.raises(ValueError):
            residual_rms_norm_fp8(*(bad if j == i else t for j, t in enumerate(norm)), 1e-6)
    for D in (8, 24, 8192):
        with pytest.raises(ValueError):
            residual_rms_norm_fp8(torch.zeros(2, D, dtype=bf), None, torch.zeros(D, dtype=bf), 1e-6)
    with pytest.raises(RuntimeError, match="GPU only"):
        residual_rms_norm_fp8(*norm, 1e-6)
    good = [_x(4, 144), _s(4, 2), _x(256, 144), _s(2, 2)]
    for f in (linear_fp8, linear_gated_fp8):
        for i, bad in ((0, _x(4, 128)), (0, _x(4, 144, bf)), (0, _x(1, 144)[0]), (1, _s(4, 1)), (1, _s(5, 2)),
                       (1, torch.zeros(4, 2)), (2, _x(256, 144, torch.float8_e5m2)), (3, _s(1, 2)), (3, _s(256, 2))):
            with pytest.raises(ValueError):
                f(*(bad if j == i else t for j, t in enumerate(good)))
        for bias in (torch.zeros(128), torch.zeros(256, dtype=torch.float64), torch.zeros(1, 256)):
            with pytest.raises(ValueError):
                f(*good, bias)
        with pytest.raises(RuntimeError, match="GPU only"):
            f(*good)
        with pytest.raises(ValueError):
            f(_x(4, 24), _s(4, 1), _x(256, 24), _s(2, 1))
    with pytest.raises(ValueError, match="out_dtype"):
        linear_fp8(*good, out_dtype=torch.float32)
    with pytest.raises(ValueError, match="multiple of 128"):
        linear_gated_fp8(_x(4, 144), _s(4, 2), _x(128, 144), _s(1, 2))


def test_modules_refuse_the_cpu_and_fp32():
    from atma_amd.engine import Config
    from atma_amd.layers.global_attention import MLP, Fp8MLP, RMSNorm
    with pytest.raises(RuntimeError, match="GPU only"):
        Fp8MLP(MLP(64))
    with pytest.raises(ValueError, match="multiples of 128"):
        Fp8MLP(MLP(48))
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):
        RMSNorm(64).add_norm_fp8(torch.zeros(2, 64, dtype=torch.bfloat16), None)
    assert Config().fp8_mlp is False


def test_entry_points_validate_without_launch():
    lib, null = _lib.load(), None
    ptr = ctypes.cast(ctypes.create_string_buffer(256), ctypes.c_void_p)
    ptr = ctypes.c_void_p((ptr.value + 63) // 64 * 64)
    odd = ctypes.c_void_p(ptr.value + 4)
    BF16, F32 = 1, 0
    for f in (lib.atma_quantize_fp8, lib.atma_quantize_weight_fp8):
        assert f(ptr, 64, ptr, 64, ptr, 4, 0, 64, BF16, null) == 0
        assert f(ptr, 64, ptr, 64, ptr, 4, 2, 40, BF16, null) == 2     # K no multiple of 16
        assert f(ptr, 64, ptr, 64, ptr, 4, 2, 64, 7, null) == 2        # no such type
        assert f(null, 64, ptr, 64, ptr, 4, 2, 64, BF16, null) == 1
        assert f(odd, 64, ptr, 64, ptr, 4, 2, 64, BF16, null) == 1     # unaligned
        assert f(ptr, 48, ptr, 64, ptr, 4, 2, 64, BF16, null) == 1     # rows shorter than K
        assert f(ptr, 256, ptr, 256, ptr, 1, 2, 256, BF16, null) == 1  # scales' rows too short
    n = [ptr, 64, null, 0, null, 0, null, 0, null, 0, null, 0, null, 0, ptr, ptr, 64]
    assert lib.atma_residual_rms_norm_fp8(*n, ptr, 4, 0, 64, 1e-6, BF16, null) == 0
    assert lib.atma_residual_rms_norm_fp8(*n, null, 4, 2, 64, 1e-6, BF16, null) == 1
    assert lib.atma_residual_rms_norm_fp8(*n, ptr, 0, 2, 64, 1e-6, BF16, null) == 1
    assert lib.atma_residual_rms_norm_fp8(*n, ptr, 4, 2, 24, 1e-6, BF16, null) == 1
    assert lib.atma_residual_rms_norm_fp8(*n, ptr, 4, 2, 64, 1e-6, F32, null) == 2
    assert lib.atma_residual_rms_norm_fp8(*n, ptr, 4, (1 << 25) + 1, 64, 1e-6, BF16, null) == 2
    assert lib.atma_quantize_weight_fp8(ptr, 256, ptr, 256, ptr, 2, 65536 * 128, 256, BF16, null) == 2

    def linear(x=ptr, ldx=144, xs=ptr, ldxs=4, w=ptr, ldw=144, ws=ptr, ldws=4, bias=null, bt=F32, y=ptr, ldy=256, M=4, N=256,
               K=144, dt=BF16):
        return lib.atma_linear_fp8(x, ldx, xs, ldxs, w, ldw, ws, ldws, bias, bt, y, ldy, M, N, K, dt, null)

    def gated(x=ptr, ldx=144, xs=ptr, ldxs=4, w=ptr, ldw=144, ws=ptr, ldws=4, bias=null, bt=F32, y=ptr, ldy=256, ys=ptr,
              ldys=2, M=4, N=256, K=144):
        return lib.atma_linear_gated_fp8(x, ldx, xs, ldxs, w, ldw, ws, ldws, bias, bt, y, ldy, ys, ldys, M, N, K, null)

    for f in (linear, gated):
        assert f(M=0) == 0
        assert f(K=136) == 2 and f(K=0) == 2 and f(K=1 << 23) == 2 and f(M=-1) == 2 and f(M=1 << 40) == 2
        assert f(ldx=1 << 24) == 2 and f(bias=ptr, bt=9) == 2
        for bad in (dict(x=null), dict(xs=null), dict(w=null), dict(ws=null), dict(y=null), dict(x=odd), dict(w=odd),
                    dict(ldx=128), dict(ldw=152), dict(ldxs=-1), dict(ldws=-1), dict(ldy=128),
                    dict(bias=ctypes.c_void_p(ptr.value + 2))):
            assert f(**bad) == 1, bad
    assert linear(dt=F32) == 2 and linear(N=0) == 2
    assert gated(N=200) == 2 and gated(ys=null) == 1 and gated(ldys=1) == 1 and gated(ldy=264) == 1


def test_copies_have_their_wait_states(tmp_path):
    src, out = _build.CSRC / "fp8_gemm.hip", tmp_path / "out.s"
    proc = subprocess.run([*_build.compile_command(src), "--cuda-device-only", "-S", str(src), "-o", str(out)],
                          stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert proc.returncode == 0, proc.stdout[-2000:]
    # the scales' copy, a byte from an address a lane, has the 16-byte form's operands: m0 and vector registers
    found, copies = check_assembly(out.read_text().replace("global_load_lds_ubyte ", "global_load_lds_dwordx4 "))
    assert found == [] and copies > 0, "\n".join(found[:20])
