"""Next-token sampling: temperature, top-k, top-p and min-p from one given random number a row (C ABI
``atma_sample_tokens``, ``atma_sample_tokens_in``), in one launch, few long rows in three to five.  The reference samples by
temperature alone, with random numbers of its own (``inference/layers/sampler.py:5-10``)."""

import torch

from .. import _ops
from .fp8 import _placed

_DT = (torch.bfloat16, torch.float16, torch.float32)


def _per_row(what, name, v, rows, dtype, off):
    """(tensor or None, number) of a parameter given as a tensor (rows,), a number for every row, or None."""
    if v is None:
        return None, off
    if isinstance(v, torch.Tensor):
        if v.shape != (rows,) or v.dtype != dtype:
            raise ValueError(f"{what}: {name} must be ({rows},) {str(dtype)[6:]} or a number (got {tuple(v.shape)} {v.dtype})")
        return v, off
    if isinstance(v, bool) or not isinstance(v, (int, float) if dtype == torch.float32 else int):
        raise ValueError(f"{what}: {name} must be a tensor or a number (got {type(v).__name__})")
    return None, float(v) if dtype == torch.float32 else min(max(v, 0), 2 ** 31 - 1)


def sample_tokens(logits, uniform, temperature=1.0, top_k=None, top_p=None, min_p=None, ids_out=None):
    """One token id for each row of ``logits`` (rows, V), fp32 or 16 bits, V up to 2^20.

    ``uniform`` (rows,) fp32 holds a random number of [0, 1) for each row (others are taken to its nearest, NaN to 0).
    ``temperature``, ``top_p``, ``min_p`` are (rows,) fp32 and ``top_k`` is (rows,) int32, or numbers for every row; None leaves
    a filter out.  With w_i = exp((x_i - max x) / temperature) and the tokens in the order of falling logits, equal ones by
    index, these are kept: the first ``top_k`` (0 or less, V or more: all); of them those before which less than ``top_p`` of
    their weight lies (1 or more: all; the first always); of them those with w_i >= ``min_p`` (0 or less: all; 1 or more: the
    largest).  The answer is the first index at which the sum of the kept weights, in index order, exceeds ``uniform`` times
    their whole sum, decided as in 64-bit arithmetic; weights below 2^-44 of the largest are 0.

    A row whose temperature is 0, negative or NaN takes its largest logit, the first of equal ones.  A logit of -inf is never
    drawn unless every one is, a row with +inf draws among those, and a row that holds a NaN answers its first NaN, as
    ``argmax`` does.  Returns ids (rows,) int64; with ``ids_out`` (a contiguous int64 (rows,) tensor) they are written there."""
    what = "sample_tokens"
    if logits.dim() != 2 or logits.dtype not in _DT or not 1 <= logits.shape[1] <= 1 << 20:
        raise ValueError(f"{what}: logits must be (rows, 1 to 2^20) in fp32 or 16 bits (got {tuple(logits.shape)} {logits.dtype})")
    rows, V = logits.shape
    if uniform.shape != (rows,) or uniform.dtype != torch.float32:
        raise ValueError(f"{what}: uniform must be ({rows},) float32 (got {tuple(uniform.shape)} {uniform.dtype})")
    temperature, t0 = _per_row(what, "temperature", temperature, rows, torch.float32, 1.0)
    top_k, k0 = _per_row(what, "top_k", top_k, rows, torch.int32, 0)
    top_p, p0 = _per_row(what, "top_p", top_p, rows, torch.float32, 1.0)
    min_p, m0 = _per_row(what, "min_p", min_p, rows, torch.float32, 0.0)
    if logits.requires_grad or uniform.requires_grad:
        logits, uniform = logits.detach(), uniform.detach()
    straight = _placed(what, logits, uniform, temperature, top_k, top_p, min_p)
    if ids_out is not None:
        if ids_out.shape != (rows,) or ids_out.dtype != torch.int64 or not ids_out.is_contiguous() \
                or ids_out.device != logits.device:
            raise ValueError(f"ids_out must be a contiguous int64 ({rows},) tensor on the logits' device")
    if (straight and logits.stride(1) == 1 and (rows < 2 or logits.stride(0) >= V)
            and all(v is None or v.stride(0) == 1 for v in (uniform, temperature, top_k, top_p, min_p))):
        ids = logits.new_empty((rows,), dtype=torch.int64) if ids_out is None else ids_out
        return _ops.sample_into(ids, logits, uniform, temperature, t0, top_k, k0, top_p, p0, min_p, m0)
    ids = _ops.run.sample_tokens(logits, uniform, temperature, t0, top_k, k0, top_p, p0, min_p, m0)
    return ids if ids_out is None else ids_out.copy_(ids)
