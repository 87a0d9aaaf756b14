"""Log probabilities of given tokens, with the entropy, the logsumexp and the top
alternatives, from the logits any route of the head writes; differentiable.

    logits, _, _ = grammar_logits_with_top1(hidden, weight, mask, route=...)
    drawn = sample_logits(logits, uniforms=..., temperature=0.8).token_ids
    r = token_logprobs(logits, drawn, temperature=0.8, top_n=5)      # serving
    loss = -(r.logprobs * advantages).mean() - 0.01 * r.entropy.mean()  # training
    loss.backward()

The distribution is the one over the legal tokens: softmax(logits / temperature),
before top-k, top-p or min-p. The reference's loop takes logits.argmax(-1) alone
(benchmarks/qwen35_adaptive_paired.py:94).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native

__all__ = ["TokenLogprobs", "token_logprobs", "compact_token_logprobs"]

MAX_TOP = 64
MAX_TOKENS = 1024  # given tokens of a row


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor      # float32, shape of token_ids
    entropy: torch.Tensor       # float32 [B]
    logsumexp: torch.Tensor     # float32 [B]: log sum exp(logits / temperature)
    top_ids: torch.Tensor       # int64 [B, top_n], by falling logit, ties by rising id; -1 where fewer are legal
    top_logprobs: torch.Tensor  # float32 [B, top_n]; -inf there


def _check_tokens(token_ids, batch, device, temperature, top_n) -> int:
    """Given tokens of a row."""
    if token_ids.device != device or token_ids.dtype != torch.int64 or not token_ids.is_contiguous():
        raise ValueError("token_ids must be a contiguous int64 tensor on the logits' device")
    if token_ids.dim() not in (1, 2) or token_ids.shape[0] != batch:
        raise ValueError("token_ids must have shape [B] or [B, K]")
    tokens = 1 if token_ids.dim() == 1 else token_ids.shape[1]
    if tokens > MAX_TOKENS:
        raise ValueError(f"token_ids may hold up to {MAX_TOKENS} tokens for each row")
    if not 0 <= top_n <= MAX_TOP:
        raise ValueError(f"top_n must be in 0..{MAX_TOP}")
    if isinstance(temperature, torch.Tensor):
        if (temperature.device != device or temperature.dtype != torch.float32 or temperature.shape != (batch,)
                or not temperature.is_contiguous()):
            raise ValueError("temperature must be a number or a contiguous float32 tensor with one value per request")
        if (temperature.requires_grad and torch.is_grad_enabled()) or _native.has_tangent(temperature):
            raise ValueError("there is no gradient of the temperature")
    elif not 0.0 < temperature < float("inf"):
        raise ValueError("temperature must be positive and finite")
    return tokens


def _outputs(token_ids, batch, top_n, device) -> TokenLogprobs:
    f32 = torch.float32
    return TokenLogprobs(torch.empty(token_ids.shape, dtype=f32, device=device),
                         torch.empty(batch, dtype=f32, device=device), torch.empty(batch, dtype=f32, device=device),
                         torch.empty(batch, top_n, dtype=torch.int64, device=device),
                         torch.empty(batch, top_n, dtype=f32, device=device))


class _Differentiable(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, token_ids, tokens, mask, temperature, top_n):
        out = _outputs(token_ids, rows.shape[0], top_n, rows.device)
        stats = torch.empty(rows.shape[0], 4, dtype=torch.float32, device=rows.device)
        _native.token_logprobs(rows, mask, temperature, token_ids, tokens, top_n, *out, stats=stats)
        ctx.save_for_backward(rows, token_ids, mask, stats)
        ctx.tokens = tokens
        ctx.mark_non_differentiable(out.top_ids, out.top_logprobs)
        ctx.set_materialize_grads(False)
        return tuple(out)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_logprobs, grad_entropy, grad_logsumexp, *_):
        rows, token_ids, mask, stats = ctx.saved_tensors
        grads = [None if g is None else g.contiguous() for g in (grad_logprobs, grad_entropy, grad_logsumexp)]
        grad = torch.empty(rows.shape, dtype=rows.dtype, device=rows.device)
        _native.token_logprobs_grad(rows, mask, token_ids, ctx.tokens, stats, *grads, grad)
        return grad, None, None, None, None, None


def token_logprobs(logits: torch.Tensor, token_ids: torch.Tensor, *, bitmask_gpu: torch.Tensor | None = None,
                   temperature=1.0, top_n: int = 0) -> TokenLogprobs:
    """Log probabilities of token_ids (int64 [B], or [B, K] for several of a row)
    under softmax(logits / temperature) over each row's legal tokens.

    logits [B, V] (or [V] with one row of tokens) float16 / bfloat16 / float32:
    what any route of the head writes (-inf on illegal tokens), or any logits
    with their bitmask; NaN counts as illegal, as in sample_logits. The rows may
    have any stride. temperature: a number, or a float32 tensor with one value
    per row (a row whose value is not positive and finite reports NaN). A token
    that is not legal has -inf; a negative id stands for no token (padding) and
    reports 0. top_n (at most 64): alternatives by falling logit, ties to the
    lowest id. A row without a legal token reports -inf, entropy 0, ids -1.

    logprobs, entropy and logsumexp carry gradients to the logits when these
    require them (backward, once; not to the temperature); top_logprobs does not: pass the
    ids as token_ids for that. A token that is not legal counts in them as one of
    probability 0 (as with logits filled with -inf); a row whose temperature is
    not valid has NaN on its legal tokens. Sums are fp32 and in a fixed order, so
    equal calls give equal bits. Asynchronous on the current stream, capturable.
    """
    if not logits.is_cuda:
        raise ValueError("logits must be a CUDA tensor")
    rows = logits.unsqueeze(0) if logits.dim() == 1 else logits
    if rows.dim() != 2 or rows.shape[0] < 1 or rows.shape[1] < 1:
        raise ValueError("logits must have shape [V] or [B, V]")
    batch, vocab = rows.shape
    if batch > 2 ** 26 or vocab > 2 ** 30:  # (the C entries take 32-bit sizes)
        raise ValueError("logits may hold up to 2^26 rows of 2^30 tokens")
    if vocab > 1 and rows.stride(1) != 1:
        raise ValueError("logits must be contiguous along the vocabulary")
    _native.dtype_code(rows.dtype)
    if _native.has_tangent(rows):
        raise ValueError("there is no forward-mode gradient")
    tokens = _check_tokens(token_ids, batch, rows.device, temperature, top_n)
    mask = bitmask_gpu
    if mask is not None:
        if mask.device != rows.device or mask.dtype != torch.int32:
            raise ValueError("bitmask_gpu must be CUDA int32")
        if mask.dim() == 1:
            mask = mask.reshape(1, -1)
        if mask.dim() != 2 or mask.shape[0] != batch or mask.shape[1] < (vocab + 31) // 32:
            raise ValueError("bitmask shape does not match logits")
        if not mask.is_contiguous():
            raise ValueError("bitmask must be contiguous")
    if rows.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs(*_Differentiable.apply(rows, token_ids, tokens, mask, temperature, top_n))
    out = _outputs(token_ids, batch, top_n, rows.device)
    _native.token_logprobs(rows, mask, temperature, token_ids, tokens, top_n, *out)
    return out


def compact_token_logprobs(packed_ids: torch.Tensor, logits: torch.Tensor, offsets: torch.Tensor,
                           token_ids: torch.Tensor, *, temperature=1.0, top_n: int = 0,
                           max_len: int | None = None) -> TokenLogprobs:
    """token_logprobs on packed legal rows: (packed_ids int64 [N], logits [N],
    offsets int64 [B+1]) as bitmask_compact_logits and int8_compact_logits return
    them, ids rising in a row; token_ids are vocabulary ids, and so are the
    alternatives'. max_len, the longest row expected (default: twice the mean),
    only picks the launch shape. Positions past the end of the arrays, or past a
    row's 2^30th, are not read, whatever the offsets say. No gradient: the packed projections have none."""
    if not logits.is_cuda:
        raise ValueError("logits must be a CUDA tensor")
    if (logits.requires_grad and torch.is_grad_enabled()) or _native.has_tangent(logits):
        raise ValueError("packed logits have no gradient: take token_logprobs on vocabulary-shaped ones")
    if logits.dim() != 1 or packed_ids.shape != logits.shape:
        raise ValueError("packed_ids and logits must have shape [N]")
    if packed_ids.dtype != torch.int64 or offsets.dtype != torch.int64:
        raise ValueError("packed_ids and offsets must be int64")
    if packed_ids.device != logits.device or offsets.device != logits.device:
        raise ValueError("packed_ids, logits and offsets must be on one device")
    if not (packed_ids.is_contiguous() and logits.is_contiguous() and offsets.is_contiguous()):
        raise ValueError("packed_ids, logits and offsets must be contiguous")
    if offsets.dim() != 1 or offsets.shape[0] < 2:
        raise ValueError("offsets must have shape [B + 1]")
    _native.dtype_code(logits.dtype)
    batch = offsets.shape[0] - 1
    if batch > 2 ** 26:
        raise ValueError("offsets may name up to 2^26 rows")
    tokens = _check_tokens(token_ids, batch, logits.device, temperature, top_n)
    if max_len is None:
        max_len = min(logits.numel(), 2 * logits.numel() // batch)
    elif max_len < 0:
        raise ValueError("max_len must not be negative")
    out = _outputs(token_ids, batch, top_n, logits.device)
    _native.token_logprobs_compact(logits, packed_ids, offsets, min(max_len, 2 ** 31 - 1), temperature, token_ids,
                                   tokens, top_n, *out)
    return out
