"""8-bit inference: quantizers, the residual norm with an 8-bit output, the block-scaled product and the MLP's gated first
projection (C ABI ``atma_quantize_fp8``, ``atma_quantize_weight_fp8``, ``atma_residual_rms_norm_fp8``,
``atma_linear_fp8``, ``atma_linear_gated_fp8``).

An 8-bit tensor is a pair ``(data, scale)``: ``data`` float8_e4m3fn, ``scale`` float8_e8m0fnu (a power of two), one scale
for each 128 values along a row (activations, ``scale`` (rows, ceil(K / 128))) or for each 128 x 128 block (weights, ``scale``
(ceil(N / 128), ceil(K / 128))); its values are ``data * scale``.  The scale of a block is the smallest 2^e, e in
[-126, 120], that brings its largest finite magnitude to 448 or less; values are rounded to nearest even, infinities and
NaN are stored as NaN and leave the block's other values as they are.

No reference counterparts: the served form of ``model/layers.py:19-31`` and ``model/reference.py:22-28`` with weights and
activations in 8 bits.  Inference only (an input that requires a gradient is refused in grad mode), on the GPU, graph
capturable.  K is a multiple of 16, up to 2^24 for the quantizers and 2^22 for the products.  There may be no rows; at most 2^31
- 1 to quantize, 2^25 to norm, 2^30 to multiply, 8,388,480 of a weight to quantize and 2^28 to multiply with.
"""

import torch

from .. import _ops
from .decode_fusions import PartialSums

_DT = (torch.bfloat16, torch.float16)
_DT32 = (torch.bfloat16, torch.float16, torch.float32)
FP8, FP8_SCALE, FP8_BLOCK = _ops.FP8, _ops.FP8_SCALE, _ops.FP8_BLOCK
_PITCH = _ops.FP8_PITCH
_Tensor, _Parameter = torch.Tensor, torch.nn.Parameter
_grad_enabled, _function_modes = torch.is_grad_enabled, torch._C._len_torch_function_stack
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device


def _placed(what, *ts):
    """Every tensor of a call on one GPU, none of them waiting for a gradient.  Returns whether the call may go straight to
    its launch: that GPU is the current one and nothing watches, transforms or overrides the call."""
    device, grad, plain = ts[0].get_device(), _grad_enabled(), True
    for t in ts:
        if t is not None:
            if t.get_device() != device or device < 0:
                if t.get_device() < 0 or device < 0:
                    raise RuntimeError(f"{what} runs on the GPU only (got a CPU tensor)")
                raise ValueError(f"{what}: every tensor must be on one GPU")
            if grad and t.requires_grad:
                raise RuntimeError(f"{what} is for inference: call it under torch.no_grad(), or detach its inputs")
            if type(t) is not _Tensor and type(t) is not _Parameter:
                plain = False
    return plain and not _ops.watched() and not _function_modes() and device == _current_device()


def _dtypes(dtypes):
    return ", ".join(str(d)[6:] for d in dtypes)


def _matrix(what, name, t, dtypes):
    if t.dim() != 2 or t.dtype not in dtypes:
        raise ValueError(f"{what}: {name} must be a matrix of {_dtypes(dtypes)} (got {tuple(t.shape)} {t.dtype})")
    if t.shape[1] < 16 or t.shape[1] % 16:
        raise ValueError(f"{what}: rows of {name} must be a multiple of 16 long (got {t.shape[1]})")


def _aligned_rows(t):
    """Rows at multiples of 16 bytes that do not overlap."""
    row, one = t.stride()
    return one == 1 and not (t.data_ptr() | row * t.element_size()) & 15 and row >= t.shape[1]


def quantize_fp8(x):
    """Rows to 8 bits: x (M, K) in fp32 or 16 bits, K a multiple of 16 -> (data (M, K), scale (M, ceil(K / 128)))."""
    _matrix("quantize_fp8", "x", x, _DT32)
    if _placed("quantize_fp8", x) and _aligned_rows(x):
        return _ops.fp8_quantize("atma_quantize_fp8", x, x.shape[0])
    return tuple(_ops.run.quantize_fp8(x))


def quantize_weight_fp8(weight):
    """A weight matrix to 8 bits: (N, K) in fp32 or 16 bits, K a multiple of 16 -> (data (N, K), scale (ceil(N / 128),
    ceil(K / 128))).  ``linear_gated_fp8`` takes the a and gate rows as one (2H, K) matrix, H a multiple of 128."""
    _matrix("quantize_weight_fp8", "weight", weight, _DT32)
    if _placed("quantize_weight_fp8", weight) and _aligned_rows(weight):
        return _ops.fp8_quantize("atma_quantize_weight_fp8", weight, (weight.shape[0] + 127) // 128)
    return tuple(_ops.run.quantize_weight_fp8(weight))


def residual_rms_norm_fp8(branch, residual, weight, eps):
    """``residual_rms_norm`` with its norm in 8 bits: ``s = residual + branch`` (rounded to the stream's type),
    ``rms_norm(s) * weight`` quantized from its fp32 values.  ``branch``: (M, D) or ``PartialSums``; ``residual`` None starts
    the stream with the branch; D a multiple of 16, at most 4,096.  Returns (data, scale, s)."""
    what = "residual_rms_norm_fp8"
    if isinstance(branch, PartialSums):
        y, parts, biases, mu_x, mu_w = branch.base, branch.parts, list(branch.biases), branch.mu_x, branch.mu_w
    else:
        y, parts, biases, mu_x, mu_w = branch, None, [], None, None
    src, dtype = (y if parts is None else parts), branch.dtype
    if src.dim() != (2 if parts is None else 3):
        raise ValueError(f"{what}: the branch must be (M, D), partial sums (P, M, D)")
    M, D = shape = src.shape[-2:]
    if dtype not in _DT or D % 16 or not 16 <= D <= 4096 or weight.shape != (D,) or weight.dtype != dtype:
        raise ValueError(f"{what}: unsupported rows of {D} {dtype}, weight {tuple(weight.shape)} {weight.dtype}")
    if src.dtype != (dtype if parts is None else torch.float32) or (parts is not None and not 1 <= parts.shape[0] <= 8):
        raise ValueError(f"{what}: a branch in the stream's type or up to 8 fp32 partial sums")
    if residual is not None and (residual.shape != shape or residual.dtype != dtype):
        raise ValueError(f"{what}: residual must match the branch")
    if len(biases) > 3 or any(b.shape != (D,) or b.dtype != dtype for b in biases):
        raise ValueError(f"{what}: up to three biases ({D},) in the stream's type")
    if mu_x is not None and (mu_w is None or mu_x.dim() != 2 or mu_x.shape[1] not in (4, 8, 16) or mu_x.shape[0] != M
                             or mu_w.shape != (D, mu_x.shape[1]) or mu_x.dtype != dtype or mu_w.dtype != dtype):
        raise ValueError(f"{what}: the low-rank term takes mu_x (M, k) and mu_w (D, k), k 4, 8 or 16")
    keep = residual is not None or src is not branch
    straight = _placed(what, src, residual, weight, mu_x, mu_w, *biases)
    if (straight and mu_x is None and not weight.data_ptr() & 15 and weight.is_contiguous()
            and (_aligned_rows(y) if parts is None else parts.is_contiguous() and not parts.data_ptr() & 15)
            and (residual is None or _aligned_rows(residual))
            and all(b.stride(0) == 1 and not b.data_ptr() & 15 for b in biases)):
        out = _ops.fp8_norm(y, parts, biases, None, None, residual, weight, float(eps), keep)
    else:
        out = _ops.run.residual_rms_norm_fp8(y, parts, biases, mu_x, mu_w, residual, weight, float(eps), keep)
    return out[0], out[1], (out[2] if keep else branch)


def _operands(what, x, x_scale, weight, weight_scale, bias):
    """Checks a product's operands; returns whether it may go straight to its launch (``_placed``, and nothing to copy)."""
    if x.dim() != 2 or x.dtype is not FP8 or x.shape[1] % 16 or x.shape[1] < 16:
        _matrix(what, "x", x, (FP8,))
    if weight.dim() != 2 or weight.dtype is not FP8:
        _matrix(what, "weight", weight, (FP8,))
    (M, K), (N, Kw) = x.shape, weight.shape
    nb = (K + 127) // 128
    if K != Kw or N < 1:
        raise ValueError(f"{what}: x (M, K) and weight (N, K), got {tuple(x.shape)} and {tuple(weight.shape)}")
    if x_scale.dtype != FP8_SCALE or x_scale.shape != (M, nb):
        raise ValueError(f"{what}: x_scale must be ({M}, {nb}) float8_e8m0fnu (got {tuple(x_scale.shape)} {x_scale.dtype})")
    if weight_scale.dtype != FP8_SCALE or weight_scale.shape != ((N + 127) // 128, nb):
        raise ValueError(f"{what}: weight_scale must be ({(N + 127) // 128}, {nb}) float8_e8m0fnu "
                         f"(got {tuple(weight_scale.shape)} {weight_scale.dtype})")
    if bias is not None and (bias.shape != (N,) or bias.dtype not in _DT32):
        raise ValueError(f"{what}: bias must be ({N},) of {_dtypes(_DT32)}")
    if not _placed(what, x, x_scale, weight, weight_scale, bias):
        return False
    (ldx, ix), (ldw, iw) = x.stride(), weight.stride()
    return (ix == iw == x_scale.stride(1) == weight_scale.stride(1) == 1 and K <= ldx <= _PITCH and K <= ldw <= _PITCH
            and not (x.data_ptr() | weight.data_ptr() | ldx | ldw) & 15
            and (bias is None or (bias.stride(0) == 1 and not bias.data_ptr() & 3)))


def linear_fp8(x, x_scale, weight, weight_scale, bias=None, out_dtype=torch.bfloat16):
    """``F.linear`` of 8-bit operands: x (M, K) with x_scale (M, ceil(K / 128)), weight (N, K) with weight_scale
    (ceil(N / 128), ceil(K / 128)); bias (N,) in fp32 or 16 bits or None.  Sums in fp32, one rounding to ``out_dtype``
    (bfloat16 or float16).  The matrix instructions add the products of eight neighbouring k with 14 bits below the largest
    of them, 1.4e-5 of a result of normally distributed values."""
    if out_dtype not in _DT:
        raise ValueError(f"linear_fp8: out_dtype must be bfloat16 or float16 (got {out_dtype})")
    if _operands("linear_fp8", x, x_scale, weight, weight_scale, bias):
        return _ops.fp8_linear(x, x_scale, weight, weight_scale, bias, out_dtype)
    return _ops.run.linear_fp8(x, x_scale, weight, weight_scale, bias, out_dtype)


def linear_gated_fp8(x, x_scale, weight, weight_scale, bias=None):
    """The MLP's first projection with its activation, 8 bits in and out: ``a, gate = linear(x, weight, bias).chunk(2, -1)``
    as fp32 sums, ``gate * relu(a)^2`` quantized once.  Operands as ``linear_fp8``, weight (2H, K) with H a multiple of 128.
    The sums' precision is ``linear_fp8``'s too: a value within it of a rounding border goes to either side (0.1% of normally
    distributed ones), and so does the scale of a block whose largest value lies that close to 448 2^e (4 in 10^5).
    Returns (data (M, H), scale (M, H / 128))."""
    if weight.dim() == 2 and weight.shape[0] % 256:
        raise ValueError(f"linear_gated_fp8: weight (2H, K) with H a multiple of 128 (got {tuple(weight.shape)})")
    if _operands("linear_gated_fp8", x, x_scale, weight, weight_scale, bias):
        return _ops.fp8_linear_gated(x, x_scale, weight, weight_scale, bias)
    return tuple(_ops.run.linear_gated_fp8(x, x_scale, weight, weight_scale, bias))
