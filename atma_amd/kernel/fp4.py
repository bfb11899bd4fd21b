"""4-bit weights for inference: their quantizer and its inverse, the product with 16-bit activations and the MLP's gated first
projection (C ABI ``atma_quantize_weight_fp4``, ``atma_dequantize_weight_fp4``, ``atma_linear_fp4``,
``atma_linear_gated_fp4``).

A 4-bit weight matrix (N, K) is a pair ``(data, scale)``: ``data`` uint8 (N, K / 2), two float4 e2m1 values a byte (0, 0.5, 1, 1.5,
2, 3, 4, 6 and their negatives; the even k in the low half), ``scale`` float8_e8m0fnu (a power of two) (N, K / 32), one for
each 32 values along a row.  The scale of a group is the smallest 2^e, e in [-125, 125], that brings its largest magnitude to 7
or less; values are rounded to nearest even, above 6 to 6.  A group that holds an infinity or NaN is NaN as a whole.

No reference counterparts: the served form of ``model/layers.py:19-31`` and ``model/reference.py:22-28`` with weights in 4
bits.  Inference only (an input that requires a gradient is refused in grad mode), on the GPU, graph capturable.  K is a multiple
of 32, up to 2^24 for the quantizer and 2^22 for the products.  There may be no rows; at most 2^31 - 1 to quantize, 2^30 of
x and 2^28 of a weight to multiply.
"""

import torch

from .. import _ops
from .fp8 import _aligned_rows, _dtypes, _placed

_DT = (torch.bfloat16, torch.float16)
_DT32 = (torch.bfloat16, torch.float16, torch.float32)
FP4_SCALE, FP4_GROUP = _ops.FP8_SCALE, _ops.FP4_GROUP
_PITCH_X, _PITCH_W = _ops.FP4_PITCH


def quantize_weight_fp4(weight):
    """A weight matrix to 4 bits: (N, K) in fp32 or 16 bits, K a multiple of 32 -> (data (N, K / 2), scale (N, K / 32)).
    ``linear_gated_fp4`` takes the a and gate rows as one (2H, K) matrix."""
    if weight.dim() != 2 or weight.dtype not in _DT32:
        raise ValueError(f"quantize_weight_fp4: weight must be a matrix of {_dtypes(_DT32)} "
                         f"(got {tuple(weight.shape)} {weight.dtype})")
    if weight.shape[1] < FP4_GROUP or weight.shape[1] % FP4_GROUP:
        raise ValueError(f"quantize_weight_fp4: rows must be a multiple of {FP4_GROUP} long (got {weight.shape[1]})")
    if _placed("quantize_weight_fp4", weight) and _aligned_rows(weight):
        return _ops.fp4_quantize(weight)
    return tuple(_ops.run.quantize_weight_fp4(weight))


def _pair(what, data, scale):
    if data.dim() != 2 or data.dtype != torch.uint8 or data.shape[1] < 16 or data.shape[1] % 16:
        raise ValueError(f"{what}: data must be a matrix of bytes, rows a multiple of 16 long (got {tuple(data.shape)} "
                         f"{data.dtype})")
    if scale.dtype != FP4_SCALE or scale.shape != (data.shape[0], data.shape[1] // 16):
        raise ValueError(f"{what}: scale must be ({data.shape[0]}, {data.shape[1] // 16}) float8_e8m0fnu "
                         f"(got {tuple(scale.shape)} {scale.dtype})")


def dequantize_weight_fp4(data, scale, dtype=torch.bfloat16):
    """The values that a 4-bit weight stands for, (N, K) in fp32 or 16 bits: exact in bfloat16 and fp32, rounded in float16
    below 2^-14 and from 65,520 on."""
    if dtype not in _DT32:
        raise ValueError(f"dequantize_weight_fp4: dtype must be one of {_dtypes(_DT32)} (got {dtype})")
    _pair("dequantize_weight_fp4", data, scale)
    if (_placed("dequantize_weight_fp4", data, scale) and _aligned_rows(data) and scale.stride(1) == 1
            and scale.stride(0) >= scale.shape[1]):
        return _ops.fp4_dequantize(data, scale, dtype)
    return _ops.run.dequantize_weight_fp4(data, scale, dtype)


def _operands(what, x, data, scale, bias):
    """Checks a product's operands; returns its sizes, strides and addresses if it may go straight to its launch (nothing to
    dispatch or to copy), else None."""
    xs, ds, ss = x.shape, data.shape, scale.shape
    if len(xs) != 2 or x.dtype not in _DT:
        raise ValueError(f"{what}: x must be a matrix of {_dtypes(_DT)} (got {tuple(xs)} {x.dtype})")
    if len(ds) != 2 or data.dtype != torch.uint8 or ds[1] < 16 or ds[1] % 16 or scale.dtype != FP4_SCALE or ss != (ds[0], ds[1] // 16):
        _pair(what, data, scale)
    (M, K), (N, half) = xs, ds
    if K != 2 * half or N < 1:
        raise ValueError(f"{what}: x (M, K) and data (N, K / 2), got {tuple(xs)} and {tuple(ds)}")
    if bias is not None and (bias.shape != (N,) or bias.dtype not in _DT32):
        raise ValueError(f"{what}: bias must be ({N},) of {_dtypes(_DT32)}")
    if not _placed(what, x, data, scale, bias):
        return None
    (ldx, ix), (ldw, iw), (lds, js) = x.stride(), data.stride(), scale.stride()
    px, pd = x.data_ptr(), data.data_ptr()
    if (ix == iw == js == 1 and K <= ldx <= _PITCH_X and half <= ldw <= _PITCH_W and not (px | pd | 2 * ldx | ldw) & 15 and lds >= 0
            and (bias is None or bias.stride(0) == 1)):
        return M, N, K, px, ldx, pd, ldw, lds
    return None


def linear_fp4(x, data, scale, bias=None):
    """``F.linear`` with a 4-bit weight: x (M, K) in 16 bits, data (N, K / 2) and scale (N, K / 32), bias (N,) in fp32 or 16 bits
    or None.  The weights are multiplied as ``dequantize_weight_fp4`` gives them in x's type; sums in fp32, one rounding to
    x's type."""
    straight = _operands("linear_fp4", x, data, scale, bias)
    if straight is not None:
        return _ops.fp4_linear_at(x, scale, bias, False, *straight)
    return _ops.run.linear_fp4(x, data, scale, bias)


def linear_gated_fp4(x, data, scale, bias=None):
    """The MLP's first projection with its activation: ``a, gate = linear_fp4(x, data, scale, bias).chunk(2, -1)`` as fp32 sums,
    ``gate * relu(a)^2`` rounded once to x's type.  data (2H, K / 2): the a rows, then the gate rows.  Returns (M, H)."""
    if data.dim() == 2 and data.shape[0] % 2:
        raise ValueError(f"linear_gated_fp4: data (2H, K / 2), got {tuple(data.shape)}")
    straight = _operands("linear_gated_fp4", x, data, scale, bias)
    if straight is not None:
        return _ops.fp4_linear_at(x, scale, bias, True, *straight)
    return _ops.run.linear_gated_fp4(x, data, scale, bias)
