"""The LM head on int8 weights: half the bytes of a half-precision head.

The weight is quantised once, one scale per vocabulary row (channel); each
step's hidden states are quantised by the call, one scale per request (token).
The product is an exact integer sum, the logit

    logit[b, v] = (float(sum_h q[b, h] w[v, h]) * token_scale[b]) * channel_scale[v]

in fp32, rounded once to the logits' type; illegal tokens come out -inf. The
routes are those of triton_runtime (ROUTES) and give the same bits:
"row-sparse" reads the legal rows only, "block-sparse" the 128-row tiles that
hold a legal token on the tensor cores, "dense-mask" every tile.

    weight = quantize_rows_int8(lm_head.weight)          # once
    logits, value, token = int8_grammar_logits(hidden, weight, bitmask)

The reference has no quantised head (gsp/triton_runtime.py:61-308 takes
floating-point weights); the entry points follow grammar_logits_with_top1 and
bitmask_compact_logits of triton_runtime.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native
from .triton_runtime import ROUTES, mask_stats

__all__ = ["QuantizedRows", "quantize_rows_int8", "int8_grammar_logits", "int8_compact_logits"]

MAX_HIDDEN = 131071  # above it the int32 sums could overflow


class QuantizedRows(NamedTuple):
    values: torch.Tensor  # int8 [N, H]
    scales: torch.Tensor  # float32 [N]; row n stands for values[n] * scales[n]


def quantize_rows_int8(x: torch.Tensor, *, out: QuantizedRows | None = None,
                       reciprocal: bool = False) -> QuantizedRows:
    """Rows of x [N, H] (float16, bfloat16 or float32) to int8: scale =
    max |x| / 127, value = x / scale to the nearest integer (ties to even).

    A row of zeros has scale 0; a row that holds an infinity or NaN has scale
    NaN and values 0, so logits computed from it are NaN. x may have any row
    stride; `out` reuses tensors (for a CUDA graph, or a preallocated head).

    reciprocal: scale = max |x| times the fp32 reciprocal of 127, at most one
    step from the division's. torch computes amax / 127.0 that way on the GPU, so
    these are the values and scales of rows quantised by torch expressions there.
    """
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor")
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError("x must have shape [N, H]")
    if x.shape[1] > 1 and x.stride(1) != 1:
        raise ValueError("x must be contiguous along its rows")
    if x.shape[0] >= 2 ** 31 or x.shape[1] > 2 ** 30:  # (the C entries take 32-bit sizes)
        raise ValueError("x may hold up to 2^31 - 1 rows of 2^30 columns")
    _native.dtype_code(x.dtype)
    given = out is not None
    if not given:
        device = x.device
        out = QuantizedRows(torch.empty(x.shape, dtype=torch.int8, device=device),
                            torch.empty(x.shape[0], dtype=torch.float32, device=device))
    else:
        _check_rows(out, "out")
        if out.values.shape != x.shape or out.values.device != x.device:
            raise ValueError("out must hold [N, H] values on x's device")
    if x.shape[0]:
        _native.quantize_rows_int8(x, out.values, out.scales, reciprocal)
        if given:
            _native.written(*out)
    return out


def _check_rows(rows, what: str) -> None:
    values, scales = rows
    if not values.is_cuda or scales.get_device() != values.get_device():
        raise ValueError(f"{what} must hold CUDA tensors on one device")
    if values.dtype != torch.int8 or scales.dtype != torch.float32:
        raise ValueError(f"{what} must hold int8 values and float32 scales")
    if values.dim() != 2 or scales.shape != values.shape[:1]:
        raise ValueError(f"{what} must hold values [N, H] and scales [N]")
    if not values.is_contiguous() or not scales.is_contiguous():
        raise ValueError(f"{what} must be contiguous")


def _inputs(hidden, weight, bitmask_gpu, out_dtype, reciprocal):
    """Checked operands: (hidden values [B, H], token scales or None, mask [B, words] or None, logits dtype)."""
    _check_rows(weight, "weight")
    if isinstance(hidden, torch.Tensor):
        if not hidden.is_cuda:
            raise ValueError("hidden and weight must be CUDA tensors")
        values, scales = (hidden.reshape(1, -1) if hidden.dim() == 1 else hidden), None
        if values.dim() != 2:
            raise ValueError("hidden must have shape [D] or [B, D]")
        if not values.is_contiguous():
            raise ValueError("hidden and weight must be contiguous")
        dtype = values.dtype
        _native.dtype_code(dtype)
        if out_dtype is not None:
            dtype = out_dtype
    else:
        _check_rows(hidden, "hidden")
        values, scales = hidden
        if out_dtype is None:
            raise ValueError("int8 hidden states need out_dtype")
        if reciprocal:
            raise ValueError("int8 hidden states have their scales already: no reciprocal")
        dtype = out_dtype
    _native.dtype_code(dtype)
    if values.get_device() != weight.values.get_device():
        raise ValueError("hidden and weight must be on one device")
    vocab, hidden_dim = weight.values.shape
    batch, width = values.shape
    if batch < 1 or vocab < 1:
        raise ValueError("hidden and weight must have at least one row")
    if batch >= 2 ** 31 or vocab >= 2 ** 31:  # (the C entries take 32-bit sizes)
        raise ValueError("hidden and weight may hold up to 2^31 - 1 rows")
    if width != hidden_dim:
        raise ValueError("hidden dimension mismatch")
    if hidden_dim > MAX_HIDDEN:
        raise ValueError(f"hidden dimensions above {MAX_HIDDEN} could overflow the integer sums")
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


def int8_grammar_logits(hidden, weight: QuantizedRows, bitmask_gpu: torch.Tensor | None, *,
                        route: str = "row-sparse", out_dtype: torch.dtype | None = None, return_logits: bool = True,
                        reciprocal: bool = False):
    """Masked logits of the int8 head and the fused greedy top-1.

    hidden: [B, D] (or [D]) float16 / bfloat16 / float32, quantised per
    request by the call; or QuantizedRows (then out_dtype says the logits'
    type, otherwise it defaults to hidden's). bitmask_gpu None: every token is
    legal. reciprocal: how the call takes the requests' scales
    (quantize_rows_int8). Returns (logits [B, V] or None, top_value float32 [B],
    top_index int64 [B]); top_index equals logits.argmax(-1), ties to the lowest
    id.
    """
    if route not in ROUTES:
        raise ValueError(f"unknown route {route!r}")
    values, scales, mask, dtype = _inputs(hidden, weight, bitmask_gpu, out_dtype, reciprocal)
    batch, vocab, dev = values.shape[0], weight.values.shape[0], values.device
    logits = torch.empty((batch, vocab), device=dev, dtype=dtype) if return_logits else None
    top_value = torch.empty(batch, device=dev, dtype=torch.float32)
    top_index = torch.empty(batch, device=dev, dtype=torch.int64)
    _native.int8_logits(route, values, scales, weight.values, weight.scales, mask, dtype, logits=logits,
                        top_value=top_value, top_index=top_index, reciprocal=reciprocal)
    return logits, top_value, top_index


def int8_compact_logits(hidden, weight: QuantizedRows, bitmask_gpu: torch.Tensor, *,
                        out_dtype: torch.dtype | None = None, capacity: int | None = None, reciprocal: bool = False):
    """Compact legal logits of the int8 head: (token_ids int64 [N], logits
    [N], offsets int64 [B+1]); request b owns positions offsets[b]:offsets[b+1],
    token ids ascending (bitmask_compact_logits of triton_runtime). Without
    `capacity`, the legal count is measured on the device first (one sync);
    positions past the legal tokens are not written. reciprocal: as for
    int8_grammar_logits."""
    if bitmask_gpu is None:
        raise ValueError("bitmask_gpu must be CUDA int32")
    values, scales, mask, dtype = _inputs(hidden, weight, bitmask_gpu, out_dtype, reciprocal)
    dev = values.device
    if capacity is None:
        capacity = int(sum(mask_stats(mask, weight.values.shape[0])["legal_counts"]))
    elif capacity < 0:
        raise ValueError("capacity must not be negative")
    logits = torch.empty(max(capacity, 1), device=dev, dtype=dtype)
    ids = torch.empty(max(capacity, 1), device=dev, dtype=torch.int64)
    offsets = torch.empty(values.shape[0] + 1, device=dev, dtype=torch.int64)
    _native.int8_compact(values, scales, weight.values, weight.scales, mask, dtype, logits[:capacity] if capacity else
                         None, ids, offsets, reciprocal=reciprocal)
    return ids[:capacity], logits[:capacity], offsets
