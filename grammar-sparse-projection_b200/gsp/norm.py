"""The root-mean-square norm before the head, with the residual's addition and an
output the 8-bit heads take as it is.

    r = rms_norm(x, weight, residual=stream, quantize="fp8")   # or "int8", or None
    logits, value, token = fp8_grammar_logits(r.output, head, mask, out_dtype=x.dtype)
    stream = r.residual

The reference starts at the hidden states (gsp/triton_runtime.py:61-109).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native
from .fp8_head import Fp8Rows
from .int8_head import QuantizedRows

__all__ = ["NormResult", "rms_norm"]

MAX_COLUMNS = 2 ** 24


class NormResult(NamedTuple):
    output: torch.Tensor | QuantizedRows | Fp8Rows  # the norm: x's type, or 8-bit rows with scales
    residual: torch.Tensor | None                   # x + residual in x's type (None without a residual)


def _check_rows(t, x, name):
    if t.device != x.device or t.dtype != x.dtype or t.shape != x.shape:
        raise ValueError(f"{name} must have x's shape, type and device")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} must be contiguous along its rows")


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, *, residual: torch.Tensor | None = None,
             eps: float = 1e-6, quantize: str | None = None, residual_out: torch.Tensor | None = None) -> NormResult:
    """h = x + residual (rounded to x's type; returned as NormResult.residual) and
    y = h / sqrt(mean(h^2) + eps) * weight in fp32, for rows x [N, H] (or [H]) of
    float16, bfloat16 or float32 with any row stride.

    quantize: None: y rounded to x's type; "int8": QuantizedRows, one scale per
    row (quantize_rows_int8's rule); "fp8": Fp8Rows, one scale per 128 columns
    (quantize_rows_fp8's rule). The 8-bit values are taken from y itself, not from
    its rounding to x's type, so they may differ by a step from a norm followed by
    a quantiser. weight [H] of x's type (None: 1). residual_out: where h goes;
    may be `residual` or `x` itself, but share no part of their memory otherwise.
    No gradient: tensors that require one are refused while gradients are recorded,
    and those with a forward-mode tangent.
    """
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor")
    if quantize not in (None, "int8", "fp8"):
        raise ValueError('quantize must be None, "int8" or "fp8"')
    one_row = x.dim() == 1
    rows = x.unsqueeze(0) if one_row else x
    if rows.dim() != 2 or rows.shape[1] < 1:
        raise ValueError("x must have shape [H] or [N, H]")
    if rows.shape[0] >= 2 ** 31 or rows.shape[1] > MAX_COLUMNS:  # (the C entries take 32-bit sizes)
        raise ValueError("x may hold up to 2^31 - 1 rows of 2^24 columns")
    _native.dtype_code(x.dtype)
    count, cols = rows.shape
    if cols > 1 and rows.stride(1) != 1:
        raise ValueError("x must be contiguous along its rows")
    if weight is not None and (weight.device != x.device or weight.dtype != x.dtype or weight.shape != (cols,)
                               or not weight.is_contiguous()):
        raise ValueError("weight must be a contiguous tensor [H] of x's type and device")
    if not 0.0 <= eps < float("inf"):
        raise ValueError("eps must be finite and not negative")
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (residual is not None and residual.requires_grad)
                                    or (residual_out is not None and residual_out.requires_grad)):
        raise ValueError("rms_norm has no gradient: call it without tensors that require one, or under torch.no_grad()")
    if _native.has_tangent(x, weight, residual):
        raise ValueError("rms_norm has no forward-mode gradient")
    if residual is not None:
        residual = residual.unsqueeze(0) if one_row and residual.dim() == 1 else residual
        _check_rows(residual, rows, "residual")
        given = residual_out is not None
        if not given:
            residual_out = torch.empty(rows.shape, dtype=x.dtype, device=x.device)
        else:
            residual_out = residual_out.unsqueeze(0) if one_row and residual_out.dim() == 1 else residual_out
            _check_rows(residual_out, rows, "residual_out")
            if count > 1 and residual_out.stride(0) < cols:
                raise ValueError("residual_out must not overlap itself")
            for t in (rows, residual):
                same = residual_out.data_ptr() == t.data_ptr() and (count == 1 or residual_out.stride(0) == t.stride(0))
                if not same and _native.rows_meet(residual_out, t):
                    raise ValueError("residual_out may be x or residual, but must not overlap a part of them")
            if weight is not None and _native.rows_meet(residual_out, weight.unsqueeze(0)):
                raise ValueError("residual_out must not overlap weight")
    elif residual_out is not None:
        raise ValueError("residual_out without residual")
    dev = x.device
    if quantize is None:
        values, scales, code = torch.empty(rows.shape, dtype=x.dtype, device=dev), None, None
        output = values[0] if one_row else values
    elif quantize == "int8":
        values, scales = torch.empty(rows.shape, dtype=torch.int8, device=dev), torch.empty(count, dtype=torch.float32, device=dev)
        output, code = QuantizedRows(values, scales), _native.DTYPE_I8
    else:
        values = torch.empty(rows.shape, dtype=torch.float8_e4m3fn, device=dev)
        scales = torch.empty(count, (cols + 127) // 128, dtype=torch.float32, device=dev)
        output, code = Fp8Rows(values, scales), _native.DTYPE_E4M3
    if count:
        _native.rms_norm(rows, weight, residual, eps, residual_out, values, scales, code)
        if residual is not None and given:
            _native.written(residual_out)
    return NormResult(output, residual_out[0] if residual_out is not None and one_row else residual_out)
