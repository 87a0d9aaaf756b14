"""The LM head in 8-bit floating point (e4m3) with a scale for each block of 128:
weight in blocks of 128 rows x 128 columns, hidden states in blocks of 128
columns of a request. Half the bytes of a half-precision head, as the int8 head
has, with scales that follow the columns.

    logit[b, v] = sum_j hs[b, j] ws[v // 128, j] sum_{k in block j} q[b, k] w[v, k]

in fp32, rounded once to the logits' type; illegal tokens come out -inf. The
routes are those of triton_runtime (ROUTES): "row-sparse" reads the legal rows
only, "block-sparse" the 32-row groups that hold a legal token of some request on
the tensor cores, "dense-mask" every row; without a mask the dense route is the
plain product, for one request or the positions of a prompt. They agree to fp32
rounding.

    weight = quantize_weight_fp8(lm_head.weight)           # once
    logits, value, token = fp8_grammar_logits(hidden, weight, bitmask, route=...)

The reference has no quantised head (gsp/triton_runtime.py:61-308 takes
floating-point weights); the entry points follow those of gsp.int8_head.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native
from .triton_runtime import ROUTES

__all__ = ["Fp8Rows", "Fp8Weight", "quantize_rows_fp8", "quantize_weight_fp8", "fp8_grammar_logits"]

BLOCK = 128
MAX_HIDDEN = 32768  # the row-sparse kernel keeps a hidden state in shared memory
MAX_VOCAB = 2 ** 30  # and counts legal rows in 32 bits
MAX_COLUMNS = 2 ** 24


class Fp8Rows(NamedTuple):
    values: torch.Tensor  # float8_e4m3fn [N, H]
    scales: torch.Tensor  # float32 [N, ceil(H / 128)]; values[n, k] stands for values[n, k] * scales[n, k // 128]


class Fp8Weight(NamedTuple):
    values: torch.Tensor  # float8_e4m3fn [V, H]
    scales: torch.Tensor  # float32 [ceil(V / 128), ceil(H / 128)]


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _quantize(entry, kind, x, out, scale_rows):
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor")
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError("x must have shape [N, H]")
    if x.shape[1] > 1 and x.stride(1) != 1:
        raise ValueError("x must be contiguous along its rows")
    if x.shape[0] >= 2 ** 31 or x.shape[1] > MAX_COLUMNS:  # (the C entries take 32-bit sizes)
        raise ValueError("x may hold up to 2^31 - 1 rows of 2^24 columns")
    _native.dtype_code(x.dtype)
    shape = (scale_rows, _blocks(x.shape[1]))
    given = out is not None
    if not given:
        out = kind(torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device),
                   torch.empty(shape, dtype=torch.float32, device=x.device))
    else:
        _check_values(out, "out")
        if out.values.shape != x.shape or out.scales.shape != shape or out.values.device != x.device:
            raise ValueError("out must hold [N, H] values and their blocks' scales on x's device")
        if any(_native.rows_meet(a, b) for a, b in ((x, out[0]), (x, out[1]), (out[0], out[1]))):
            raise ValueError("out must not overlap x or itself")
    if x.shape[0]:
        _native.quantize_fp8(entry, x, out.values, out.scales)
        if given:
            _native.written(*out)
    return out


def quantize_rows_fp8(x: torch.Tensor, *, out: Fp8Rows | None = None) -> Fp8Rows:
    """Rows of x [N, H] (float16, bfloat16 or float32) to e4m3 with one scale per
    128 columns: scale = max |x| / 448, value = x / scale to the nearest e4m3
    (ties to even). A block of zeros has scale 0; one that holds an infinity or
    NaN has scale NaN and values 0, so that logits computed from it are NaN. x
    may have any row stride; `out` reuses tensors."""
    return _quantize("gsp_quantize_rows_fp8", Fp8Rows, x, out, x.shape[0] if x.dim() else 0)


def quantize_weight_fp8(weight: torch.Tensor, *, out: Fp8Weight | None = None) -> Fp8Weight:
    """The same for a weight [V, H], with one scale per block of 128 rows x 128 columns."""
    return _quantize("gsp_quantize_weight_fp8", Fp8Weight, weight, out, _blocks(weight.shape[0]) if weight.dim() else 0)


def _check_values(rows, what: str) -> None:
    values, scales = rows
    if not values.is_cuda or scales.get_device() != values.get_device():
        raise ValueError(f"{what} must hold CUDA tensors on one device")
    if values.dtype != torch.float8_e4m3fn or scales.dtype != torch.float32:
        raise ValueError(f"{what} must hold float8_e4m3fn values and float32 scales")
    if values.dim() != 2 or scales.dim() != 2:
        raise ValueError(f"{what} must hold values [N, H] and a scale for each block")
    if not values.is_contiguous() or not scales.is_contiguous():
        raise ValueError(f"{what} must be contiguous")


def _inputs(hidden, weight, bitmask_gpu, out_dtype):
    """Checked operands: (hidden values [B, H], scales or None, mask [B, words] or None, logits dtype)."""
    _check_values(weight, "weight")
    if isinstance(hidden, torch.Tensor):
        if not hidden.is_cuda:
            raise ValueError("hidden and weight must be CUDA tensors")
        values, scales = (hidden.reshape(1, -1) if hidden.dim() == 1 else hidden), None
        if values.dim() != 2:
            raise ValueError("hidden must have shape [D] or [B, D]")
        if not values.is_contiguous():
            raise ValueError("hidden and weight must be contiguous")
        _native.dtype_code(values.dtype)
        dtype = values.dtype if out_dtype is None else out_dtype
    else:
        _check_values(hidden, "hidden")
        values, scales = hidden
        if out_dtype is None:
            raise ValueError("e4m3 hidden states need out_dtype")
        dtype = out_dtype
    _native.dtype_code(dtype)
    if values.get_device() != weight.values.get_device():
        raise ValueError("hidden and weight must be on one device")
    vocab, hidden_dim = weight.values.shape
    batch, width = values.shape
    if batch < 1 or vocab < 1 or hidden_dim < 1:
        raise ValueError("hidden and weight must have at least one row and column")
    if batch >= 2 ** 31 or vocab > MAX_VOCAB:  # (the C entries take 32-bit sizes)
        raise ValueError("hidden may hold up to 2^31 - 1 rows, weight up to 2^30")
    if batch * ((vocab + 31) // 32 * 32) >= 2 ** 32:
        raise ValueError("a call may have up to 2^32 - 1 logits (the vocabulary in whole mask words): project in parts")
    if width != hidden_dim:
        raise ValueError("hidden dimension mismatch")
    if hidden_dim > MAX_HIDDEN:
        raise ValueError(f"hidden dimensions above {MAX_HIDDEN} are not supported")
    if weight.scales.shape != (_blocks(vocab), _blocks(hidden_dim)):
        raise ValueError("weight must hold scales [ceil(V / 128), ceil(H / 128)]")
    if scales is not None and scales.shape != (batch, _blocks(hidden_dim)):
        raise ValueError("hidden must hold scales [B, ceil(H / 128)]")
    mask = bitmask_gpu
    if mask is not None:
        if mask.get_device() != values.get_device() or mask.dtype != torch.int32:
            raise ValueError("bitmask_gpu must be CUDA int32")
        if mask.dim() == 1:
            mask = mask.reshape(1, -1)
        if mask.dim() != 2 or mask.shape[0] != batch or mask.shape[1] < (vocab + 31) // 32:
            raise ValueError("bitmask shape does not match hidden batch/vocabulary")
        if not mask.is_contiguous():
            raise ValueError("bitmask must be contiguous")
    return values, scales, mask, dtype


def fp8_grammar_logits(hidden, weight: Fp8Weight, bitmask_gpu: torch.Tensor | None, *, route: str = "row-sparse",
                       out_dtype: torch.dtype | None = None, return_logits: bool = True):
    """Masked logits of the fp8 head and the fused greedy top-1.

    hidden: [B, D] (or [D]) float16 / bfloat16 / float32, quantised by the call
    (quantize_rows_fp8's rule); or Fp8Rows (then out_dtype says the logits' type,
    otherwise it defaults to hidden's), as gsp.norm.rms_norm writes them.
    bitmask_gpu None: every token is legal. Returns (logits [B, V] or None,
    top_value float32 [B], top_index int64 [B]); top_index equals
    logits.argmax(-1), ties to the lowest id. A call takes up to 2^32 - 1 logits
    (28,268 positions of 151,936 tokens) of up to 2^30 tokens. No gradient.
    Asynchronous, capturable; each call has scratch of its own.
    """
    if route not in ROUTES:
        raise ValueError(f"unknown route {route!r}")
    values, scales, mask, dtype = _inputs(hidden, weight, bitmask_gpu, out_dtype)
    batch, vocab, dev = values.shape[0], weight.values.shape[0], values.device
    logits = torch.empty((batch, vocab), device=dev, dtype=dtype) if return_logits else None
    top_value = torch.empty(batch, device=dev, dtype=torch.float32)
    top_index = torch.empty(batch, device=dev, dtype=torch.int64)
    _native.fp8_logits(route, values, scales, weight.values, weight.scales, mask, dtype, logits=logits,
                       top_value=top_value, top_index=top_index)
    return logits, top_value, top_index
