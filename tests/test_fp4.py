"""The 4-bit weights where no GPU is needed: refusals, at the Python entry points and at the C ABI, and the oracle's own rules."""

import ctypes
import subprocess

import pytest
import torch

from atma_amd import _build, _lib
from oracle import fp4 as O
from tests.test_copy_hazards import check_assembly

E8 = torch.float8_e8m0fnu
BF = torch.bfloat16


def _data(n, k):
    return torch.zeros(n, k // 2, dtype=torch.uint8)


def _scale(n, k):
    return torch.full((n, k // 32), 127, dtype=torch.uint8).view(E8)


def test_quantizer_refusals():
    from atma_amd.kernel import dequantize_weight_fp4, quantize_weight_fp4
    for bad in (torch.zeros(4), torch.zeros(4, 48), torch.zeros(4, 0), torch.zeros(4, 32, dtype=torch.float64),
                torch.zeros(2, 4, 32)):
        with pytest.raises(ValueError):
            quantize_weight_fp4(bad)
    with pytest.raises(RuntimeError, match="GPU only"):
        quantize_weight_fp4(torch.zeros(4, 32))
    for data, scale in ((_data(4, 64).to(torch.int8), _scale(4, 64)), (_data(4, 48), _scale(4, 32)),
                        (_data(4, 64), _scale(4, 32)), (_data(4, 64), _scale(3, 64)), (_data(4, 64)[0], _scale(4, 64)),
                        (_data(4, 64), torch.ones(4, 2))):
        with pytest.raises(ValueError):
            dequantize_weight_fp4(data, scale)
    with pytest.raises(ValueError, match="dtype"):
        dequantize_weight_fp4(_data(4, 64), _scale(4, 64), torch.float64)
    with pytest.raises(RuntimeError, match="GPU only"):
        dequantize_weight_fp4(_data(4, 64), _scale(4, 64))


@pytest.mark.parametrize("name", ["linear_fp4", "linear_gated_fp4"])
def test_product_refusals(name):
    import atma_amd.kernel as kernel
    f = getattr(kernel, name)
    good = [torch.zeros(4, 64, dtype=BF), _data(16, 64), _scale(16, 64)]
    for i, bad in ((0, torch.zeros(4, 64)), (0, torch.zeros(4, 96, dtype=BF)), (0, torch.zeros(64, dtype=BF)),
                   (1, _data(16, 96)), (1, _data(16, 64).view(torch.int8)), (2, _scale(16, 32)), (2, _scale(8, 64)),
                   (2, torch.ones(16, 2, dtype=torch.uint8))):
        with pytest.raises(ValueError):
            f(*(bad if j == i else t for j, t in enumerate(good)))
    for bias in (torch.zeros(15), torch.zeros(16, dtype=torch.float64), torch.zeros(1, 16)):
        with pytest.raises(ValueError):
            f(*good, bias)
    with pytest.raises(RuntimeError, match="GPU only"):
        f(*good)
    with pytest.raises(ValueError):
        f(good[0], _data(0, 64), _scale(0, 64))
    if name == "linear_gated_fp4":
        with pytest.raises(ValueError, match="2H"):
            f(good[0], _data(15, 64), _scale(15, 64))


def test_c_refusals():
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    bf16, f32 = _lib.ATMA_BF16, _lib.ATMA_F32

    def quantize(w=at, ldw=64, data=at, ldd=32, scale=at, lds=2, N=4, K=64, dtype=bf16):
        return [f(*p, N, K, dtype, None) for f, p in (
            (lib.atma_quantize_weight_fp4, (w, ldw, data, ldd, scale, lds)),
            (lib.atma_dequantize_weight_fp4, (data, ldd, scale, lds, w, ldw)))]

    assert quantize(dtype=7) == [2, 2] and quantize(K=48) == [2, 2] and quantize(K=0) == [2, 2]
    assert quantize(N=-1) == [2, 2] and quantize(N=1 << 31) == [2, 2] and quantize(K=(1 << 24) + 32) == [2, 2]
    assert quantize(w=None) == [1, 1] and quantize(data=None) == [1, 1] and quantize(scale=None) == [1, 1]
    assert quantize(w=at + 2) == [1, 1] and quantize(ldw=66) == [1, 1] and quantize(ldw=32) == [1, 1]
    assert quantize(data=at + 1) == [1, 1] and quantize(ldd=30) == [1, 1] and quantize(ldd=16) == [1, 1]
    assert quantize(lds=1) == [1, 1] and quantize(N=0, w=None) == [0, 0]

    def linear(x=at, ldx=64, w=at, ldw=32, ws=at, ldws=2, bias=None, bias_dtype=f32, y=at, ldy=16, M=4, N=16, K=64, dtype=bf16):
        return [f(x, ldx, w, ldw, ws, ldws, bias, bias_dtype, y, ldy, M, N, K, dtype, None)
                for f in (lib.atma_linear_fp4, lib.atma_linear_gated_fp4)]

    assert linear(dtype=f32) == [2, 2] and linear(K=48) == [2, 2] and linear(K=(1 << 22) + 32) == [2, 2]
    assert linear(M=-1) == [2, 2] and linear(N=0) == [2, 2] and linear(M=(1 << 30) + 1) == [2, 2] and linear(N=1 << 29) == [2, 2]
    for name in ("x", "w", "ws", "y"):
        assert linear(**{name: None}) == [1, 1]
    assert linear(x=at + 2) == [1, 1] and linear(ldx=68) == [1, 1] and linear(ldx=56) == [1, 1]
    assert linear(w=at + 8) == [1, 1] and linear(ldw=40) == [1, 1] and linear(ldw=16) == [1, 1] and linear(ldws=-1) == [1, 1]
    assert linear(ldy=15) == [1, 1]
    assert linear(ldx=(1 << 22) + 8) == [2, 2] and linear(ldw=(1 << 23) + 16) == [2, 2]
    assert linear(bias=at, bias_dtype=9) == [2, 2] and linear(bias=at + 1) == [1, 1]
    assert linear(M=0, x=None) == [0, 0]


def test_copies_have_their_wait_states(tmp_path):
    src, out = _build.CSRC / "fp4_gemm.hip", tmp_path / "out.s"
    proc = subprocess.run([*_build.compile_command(src), "--cuda-device-only", "-S", str(src), "-o", str(out)],
                          stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert proc.returncode == 0, proc.stdout[-2000:]
    # the copies of a byte, two and four from an address a lane have the 16-byte form's operands: m0 and vector registers
    text = out.read_text()
    for form in ("ubyte", "ushort", "dword"):
        text = text.replace(f"global_load_lds_{form} ", "global_load_lds_dwordx4 ")
    found, copies = check_assembly(text)
    assert found == [] and copies > 0, "\n".join(found[:20])


def test_oracle_rounds_to_the_nearest():
    a = torch.tensor([0, 0.2, 0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, 4.9, 5.0, 5.1, 6, 7], dtype=torch.float64)
    assert [O.GRID[i] for i in O.nearest(a)] == [0, 0, 0, 0.5, 1, 1, 2, 2, 4, 4, 4, 6, 6, 6]
    assert O.scales(torch.tensor([[7.0] * 32 + [7.1] + [0] * 31])).tolist() == [[1.0, 2.0]]
    assert O.pack(torch.tensor([[1, 2, 15, 0]])).tolist() == [[0x21, 0x0f]]
