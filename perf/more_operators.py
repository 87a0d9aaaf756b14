"""Operators around the LM head as they are measured: cases, inputs, plain forms.

  norm      the final norm before a head: the residual's addition, the
            root-mean-square norm, and its output in the input's type, in int8
            rows with one scale each, or in e4m3 with a scale per 128 columns;
  project   the LM head in 8-bit floating point: weight in e4m3 with a scale per
            128 x 128 block, hidden states in e4m3 with a scale per 128 columns,
            masked, on the three routes;
  logprobs  log probabilities of given tokens with the entropy, the logsumexp
            and the top alternatives, from masked logits;
  gradient  the same without alternatives, forward and backward.

Sizes are those of the head benchmark of this repository (vocabularies of
248,320, 151,936 and 262,144 tokens; hidden sizes 1,024 to 8,192; batches 1 to
128), prompts of up to 2,048 positions, and generic ones between them.
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # a decode step of 64 requests before the fp8 head
        {"name": "norm-step", "op": "norm", "rows": 64, "hidden": 2048, "dtype": "bf16", "out": "fp8", "residual": True},
        # every position of a batch of prompts, the widest model
        {"name": "norm-prompt", "op": "norm", "rows": 16384, "hidden": 8192, "dtype": "bf16", "out": "fp8",
         "residual": True},
        # one request under a grammar that leaves 1% of the vocabulary
        {"name": "project-one", "op": "project", "route": "row-sparse", "batch": 1, "vocab": 248320, "hidden": 2048,
         "dtype": "fp16", "density": 0.01, "clustered": False, "quantized": False},
        # a batch under grammars whose legal tokens lie in runs
        {"name": "project-block", "op": "project", "route": "block-sparse", "batch": 32, "vocab": 248320, "hidden": 2048,
         "dtype": "bf16", "density": 0.05, "clustered": True, "quantized": False},
        # a batch of free text
        {"name": "project-dense", "op": "project", "route": "dense-mask", "batch": 64, "vocab": 151936, "hidden": 1024,
         "dtype": "bf16", "density": 0.9, "clustered": False, "quantized": True},
        # the widest head of the benchmark, a full batch
        {"name": "project-wide", "op": "project", "route": "dense-mask", "batch": 128, "vocab": 262144, "hidden": 8192,
         "dtype": "bf16", "density": 1.0, "clustered": False, "quantized": False},
        # every position of a prompt, to score it
        {"name": "project-prompt", "op": "project", "route": "dense-mask", "batch": 2048, "vocab": 151936, "hidden": 1024,
         "dtype": "bf16", "density": 1.0, "clustered": False, "quantized": True},
        # what one request's drawn token was worth, with 20 alternatives
        {"name": "logprobs-one", "op": "logprobs", "form": "masked", "batch": 1, "vocab": 248320, "dtype": "fp16",
         "density": 0.01, "tokens": 1, "top_n": 20, "temperature": 0.8, "mixed": False},
        # a full batch of free text, five alternatives
        {"name": "logprobs-batch", "op": "logprobs", "form": "bits", "batch": 128, "vocab": 248320, "dtype": "bf16",
         "density": 0.95, "tokens": 1, "top_n": 5, "temperature": 1.0, "mixed": True},
        # four candidate answers compared at each position of a prompt
        {"name": "logprobs-score", "op": "logprobs", "form": "free", "batch": 1999, "vocab": 151936, "dtype": "bf16",
         "density": 1.0, "tokens": 4, "top_n": 0, "temperature": 1.0, "mixed": False},
        # a policy update on a few positions in 32 bits, a vocabulary of odd rows
        {"name": "gradient-small", "op": "gradient", "form": "masked", "batch": 12, "vocab": 50257, "dtype": "fp32",
         "density": 0.3, "tokens": 1, "top_n": 0, "temperature": 0.7, "mixed": False},
        # a policy update: the drawn tokens' log probabilities and the entropy
        {"name": "gradient-policy", "op": "gradient", "form": "bits", "batch": 2048, "vocab": 151936, "dtype": "bf16",
         "density": 0.9, "tokens": 1, "top_n": 0, "temperature": 1.0, "mixed": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "project", "project", "logprobs", "gradient"))
    if op == "norm":
        out = rng.choice(("same", "int8", "fp8"))
        hidden = _log(rng, 64, 16384)
        rows = _log(rng, 1, min(32768, 16384 * 8192 // hidden))
        # (8-bit values of 32-bit rows are no question of this comparison: a border that a
        # sum's last bit moves is one whole step)
        dtype = rng.choice(("fp16", "bf16", "fp32")) if out == "same" else rng.choice(("fp16", "bf16"))
        return {"op": op, "rows": rows, "hidden": hidden, "dtype": dtype, "out": out, "residual": rng.random() < 0.7}
    if op == "project":
        vocab, hidden = _log(rng, 1000, 262144), _log(rng, 64, 8192)
        if rng.random() < 0.75:
            hidden = (hidden + 15) // 16 * 16  # whole 16-byte vectors, as nearly every model has them
        route = rng.choice(("row-sparse", "block-sparse", "dense-mask"))
        if hidden % 16 or route == "row-sparse":
            batch, density = _log(rng, 1, 128), math.exp(rng.uniform(math.log(0.0005), math.log(0.05)))
        elif route == "block-sparse":
            batch, density = _log(rng, 1, 256), math.exp(rng.uniform(math.log(0.002), 0.0))
        else:
            batch, density = _log(rng, 1, 2048), rng.choice((1.0, 0.9))
            batch = max(1, min(batch, 2048 * 151936 * 1024 // (vocab * hidden)))
        return {"op": op, "route": route, "batch": batch, "vocab": vocab, "hidden": hidden,
                "dtype": rng.choice(("fp16", "bf16", "fp32")), "density": round(density, 5),
                "clustered": rng.random() < 0.5, "quantized": rng.random() < 0.5}
    form = rng.choice(("masked", "bits", "free") if op == "gradient" else ("masked", "bits", "free", "packed"))
    density = 1.0 if form == "free" else math.exp(rng.uniform(math.log(0.001), 0.0))
    top_n = rng.choice((0, 1, 5, 20, 64)) if op == "logprobs" else 0
    vocab = _log(rng, 1000, 262144)
    most = 128 if top_n or form == "packed" else 2048
    batch = max(1, min(_log(rng, 1, most), (most * 151936) // vocab))
    return {"op": op, "form": form, "batch": batch, "vocab": vocab, "dtype": rng.choice(("fp16", "bf16", "fp32")),
            "density": round(density, 5), "tokens": rng.choice((1, 1, 2, 8)), "top_n": top_n,
            "temperature": round(rng.uniform(0.5, 1.5), 3), "mixed": rng.random() < 0.3}


def work(case):
    """Each input read once and each output written once."""
    size = TYPES[case["dtype"]].itemsize
    if case["op"] == "norm":
        rows, hidden = case["rows"], case["hidden"]
        n, moved = rows * hidden, size * (1 + 2 * case["residual"])
        out, scales = {"same": (size, 0), "int8": (1, 1), "fp8": (1, (hidden + 127) // 128)}[case["out"]]
        return {"bytes": n * (moved + out) + 4 * rows * scales + size * hidden, "flops": 6 * n}
    batch, vocab, density = case["batch"], case["vocab"], case["density"]
    legal = batch * vocab * density
    mask = batch * vocab / 8
    if case["op"] == "project":
        hidden, route = case["hidden"], case["route"]
        rows = vocab if route == "dense-mask" else vocab * (1.0 - (1.0 - density) ** batch)
        states = batch * (hidden + 4 * ((hidden + 127) // 128)) if case["quantized"] else batch * hidden * size
        return {"bytes": rows * hidden * (1 + 4 / 16384) + states + (mask if density < 1.0 else 0) + batch * vocab * size,
                "flops": 2 * hidden * (batch * vocab if route == "dense-mask" else legal)}
    read = {"masked": batch * vocab * size, "free": batch * vocab * size,
            "bits": batch * vocab * size + mask, "packed": legal * size}[case["form"]]
    small = batch * (12 * case["tokens"] + 12 * case["top_n"] + 8)
    if case["op"] == "gradient":
        return {"bytes": read + batch * vocab * size * 2 + 2 * small, "flops": 14 * batch * vocab}
    return {"bytes": read + small, "flops": 6 * (legal if case["form"] == "packed" else batch * vocab)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _legal(g, batch, vocab, density, clustered):
    """[B, V] truth values, the same number for each request: single tokens anywhere, or up to 16 runs of tokens.
    Each run starts at a random place of its own part of the vocabulary."""
    count = min(vocab, max(1, round(vocab * density)))
    runs = min(16, count) if clustered else count
    length = count // runs
    first = torch.arange(runs, device=DEVICE) * vocab // runs
    room = (torch.arange(1, runs + 1, device=DEVICE) * vocab // runs - first - length + 1).clamp_(min=1)
    legal = torch.empty(batch, vocab, dtype=torch.bool, device=DEVICE)
    for b0 in range(0, batch, 256):
        n = min(256, batch - b0)
        start = first + (torch.rand(n, runs, generator=g, device=DEVICE) * room).long().minimum(room - 1)
        edge = torch.zeros(n, vocab + 1, dtype=torch.int32, device=DEVICE)
        one = torch.ones_like(start, dtype=torch.int32)
        edge.scatter_add_(1, start, one)
        edge.scatter_add_(1, start + length, -one)
        torch.gt(edge[:, :vocab].cumsum(1, dtype=torch.int32), 0, out=legal[b0:b0 + n])
    return legal


def _pack(legal):
    """[B, V] truth values -> [B, ceil(V / 32)] int32, lowest bit first."""
    batch, vocab = legal.shape
    words = (vocab + 31) // 32
    bits = torch.zeros(batch, words * 32, dtype=torch.bool, device=legal.device)
    bits[:, :vocab] = legal
    bits = bits.view(batch, words, 32)
    packed = torch.zeros(batch, words, dtype=torch.int64, device=legal.device)
    for k in range(32):
        packed |= bits[:, :, k].long() << k
    return torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).to(torch.int32)


def _pad_blocks(x, rows):
    """x [N, H] with N and H filled up to whole blocks, as [N / rows, rows, H / 128, 128]."""
    n, h = x.shape
    x = torch.nn.functional.pad(x, (0, -h % 128, 0, -n % rows))
    return x.view(x.shape[0] // rows, rows, x.shape[1] // 128, 128)


def _e4m3_blocks(x, rows):
    """The definition of the quantisers: blocks of `rows` x 128 (fp32 x [N, H]); scale = max |x| / 448, value = x / scale
    to the nearest e4m3 (ties to even). A block of zeros has scale 0."""
    n, h = x.shape
    blocks = _pad_blocks(x, rows)
    scales = blocks.abs().amax((1, 3)) / torch.full((), 448.0, device=x.device)  # (a true division, no reciprocal)
    by = scales[:, None, :, None]
    values = torch.where(by > 0, blocks / by, torch.zeros_like(blocks)).clamp_(-448, 448).to(torch.float8_e4m3fn)
    values = values.view(blocks.shape[0] * rows, -1)[:n, :h].contiguous()
    return values, scales


def _logits(g, batch, vocab, dtype):
    """Logits as a head writes them: a broad bell and a few tokens that stand out."""
    x = torch.empty(batch, vocab, dtype=dtype, device=DEVICE)
    for b0 in range(0, batch, 512):
        n = min(512, batch - b0)
        part = torch.randn(n, vocab, generator=g, device=DEVICE).mul_(2.2)
        at = torch.randint(0, vocab, (n, 24), generator=g, device=DEVICE)
        part.scatter_(1, at, 6.0 + 2.5 * torch.randn(n, 24, generator=g, device=DEVICE))
        x[b0:b0 + n] = part
    return x


def _drawn(g, x, legal, tokens):
    """Tokens drawn from softmax(x) over the legal ones, `tokens` for each row: the largest of x + Gumbel noise."""
    ids = torch.empty(x.shape[0], tokens, dtype=torch.int64, device=DEVICE)
    for b0 in range(0, x.shape[0], 256):
        part = x[b0:b0 + 256].float()
        if legal is not None:
            part.masked_fill_(~legal[b0:b0 + 256], float("-inf"))
        for k in range(tokens):
            noise = torch.empty_like(part).exponential_(generator=g).log_()
            ids[b0:b0 + 256, k] = (part - noise).argmax(1)
    return ids


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dtype = TYPES[case["dtype"]]
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE)  # noqa: E731
    if case["op"] == "norm":
        rows, hidden = case["rows"], case["hidden"]
        return {"op": "norm", "out": case["out"], "x": randn(rows, hidden).mul_(0.5).to(dtype),
                "residual": randn(rows, hidden).mul_(3.0).to(dtype) if case["residual"] else None,
                "weight": randn(hidden).mul_(0.2).add_(1.0).to(dtype)}
    batch, vocab = case["batch"], case["vocab"]
    if case["op"] == "project":
        hidden = case["hidden"]
        values = torch.empty(vocab, hidden, dtype=torch.float8_e4m3fn, device=DEVICE)
        scales = torch.empty((vocab + 127) // 128, (hidden + 127) // 128, device=DEVICE)
        for v0 in range(0, vocab, 65536):
            q, s = _e4m3_blocks(randn(min(65536, vocab - v0), hidden).mul_(0.02), 128)
            values[v0:v0 + 65536], scales[v0 // 128:(v0 + 65536) // 128] = q, s
        state = {"op": "project", "route": case["route"], "dtype": dtype, "w": values, "ws": scales, "mask": None}
        if case["density"] < 1.0:
            state["mask"] = _pack(_legal(g, batch, vocab, case["density"], case["clustered"]))
        elif case["route"] != "dense-mask":
            state["mask"] = torch.full((batch, (vocab + 31) // 32), -1, dtype=torch.int32, device=DEVICE)
        h = randn(batch, hidden).to(dtype)
        if case["quantized"]:  # as the norm before the head leaves them
            state["h"], state["hs"] = _e4m3_blocks(h.float(), 1)
        else:
            state["h"], state["hs"] = h, None
        return state
    x = _logits(g, batch, vocab, dtype)
    form = case["form"]
    legal = _legal(g, batch, vocab, case["density"], False) if form != "free" else None
    state = {"op": case["op"], "form": form, "top_n": case["top_n"], "mask": None}
    ids = _drawn(g, x, legal, case["tokens"])
    state["ids"] = ids[:, 0].contiguous() if case["tokens"] == 1 else ids
    if form == "masked":
        x.masked_fill_(~legal, float("-inf"))
    elif form == "bits":
        state["mask"] = _pack(legal)
    elif form == "packed":
        where = legal.nonzero()
        counts = legal.sum(1)
        state.update(packed_ids=where[:, 1].contiguous(), offsets=torch.cat([counts.new_zeros(1), counts.cumsum(0)]),
                     max_len=int(counts.max()))
        x = x[legal]
    state["x"] = x
    state["temperature"] = case["temperature"]
    if case["mixed"]:
        state["temperature"] = 0.5 + torch.rand(batch, generator=g, device=DEVICE)
    if case["op"] == "gradient":
        state["x"].requires_grad_(True)
        state["grad_logprobs"] = torch.randn(state["ids"].shape, generator=g, device=DEVICE)  # advantages
        state["grad_entropy"] = torch.full((batch,), 0.01, device=DEVICE)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _run_plain(state)


def _run_own(state):
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "grammar-sparse-projection_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from gsp import fp8_head, logprobs, norm
    if state["op"] == "norm":
        quantize = None if state["out"] == "same" else state["out"]
        r = norm.rms_norm(state["x"], state["weight"], residual=state["residual"], eps=EPS, quantize=quantize)
        return _norm_outputs(state, *((r.output, None) if quantize is None else r.output), r.residual)
    if state["op"] == "project":
        weight = fp8_head.Fp8Weight(state["w"], state["ws"])
        hidden = state["h"] if state["hs"] is None else fp8_head.Fp8Rows(state["h"], state["hs"])
        # (the top-1 comes with it; which of two logits next to a rounding border is the larger is no
        # question of this comparison)
        logits, _, _ = fp8_head.fp8_grammar_logits(hidden, weight, state["mask"], route=state["route"],
                                                   out_dtype=state["dtype"])
        return {"logits": logits}
    if state["form"] == "packed":
        r = logprobs.compact_token_logprobs(state["packed_ids"], state["x"], state["offsets"], state["ids"],
                                            temperature=state["temperature"], top_n=state["top_n"],
                                            max_len=state["max_len"])
    else:
        r = logprobs.token_logprobs(state["x"], state["ids"], bitmask_gpu=state["mask"],
                                    temperature=state["temperature"], top_n=state["top_n"])
    if state["op"] == "logprobs":
        return {"logprobs": r.logprobs, "entropy": r.entropy, "logsumexp": r.logsumexp, "top_ids": r.top_ids,
                "top_logprobs": r.top_logprobs}
    (grad,) = torch.autograd.grad((r.logprobs, r.entropy), state["x"], (state["grad_logprobs"], state["grad_entropy"]))
    return {"logprobs": r.logprobs.detach(), "entropy": r.entropy.detach(), "grad": grad}


def _norm_outputs(state, values, scales, residual):
    """8-bit values beside their scales: e4m3 ones as they are, integers as numbers of the input's type."""
    return {"values": values.to(state["x"].dtype) if state["out"] == "int8" else values, "scales": scales,
            "residual": residual if state["residual"] is not None else None}


def _unpack(mask, vocab):
    v = torch.arange(vocab, device=mask.device)
    return ((mask[:, v >> 5] >> (v & 31)) & 1).bool()


def _run_plain(state):
    if state["op"] == "norm":
        h = state["x"].float()
        if state["residual"] is not None:
            h = (h + state["residual"].float()).to(state["x"].dtype)
        residual, h = h, h.float()
        y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * state["weight"].float()
        if state["out"] == "same":
            return _norm_outputs(state, y.to(state["x"].dtype), None, residual)
        if state["out"] == "fp8":
            return _norm_outputs(state, *_e4m3_blocks(y, 1), residual)
        scales = y.abs().amax(1) / torch.full((), 127.0, device=y.device)
        by = scales.unsqueeze(1)
        values = torch.where(by > 0, torch.round(y / by), torch.zeros_like(y)).clamp_(-127, 127).to(torch.int8)
        return _norm_outputs(state, values, scales, residual)
    if state["op"] == "project":
        h, hs = (state["h"], state["hs"]) if state["hs"] is not None else _e4m3_blocks(state["h"].float(), 1)
        vocab, hidden = state["w"].shape
        h = h.float() * hs.repeat_interleave(128, 1)[:, :hidden]
        w = state["w"].float()
        w *= state["ws"].repeat_interleave(128, 0)[:vocab].repeat_interleave(128, 1)[:, :hidden]
        y = (h @ w.T).to(state["dtype"])
        if state["mask"] is not None:
            y.masked_fill_(~_unpack(state["mask"], vocab), float("-inf"))
        return {"logits": y}
    x, ids, n = state["x"], state["ids"], state["top_n"]
    if state["form"] == "packed":
        col = torch.arange(state["max_len"], device=x.device)
        inside = col < state["offsets"].diff().unsqueeze(1)
        place = (state["offsets"][:-1].unsqueeze(1) + col).clamp_(max=x.numel() - 1)
        rows = torch.where(inside, x[place].float(), float("-inf"))
        names = torch.where(inside, state["packed_ids"][place], 2 ** 40)
        at = torch.searchsorted(names, ids.view(ids.shape[0], -1))
    else:
        rows = x.float()
        if state["mask"] is not None:
            rows = rows.masked_fill(~_unpack(state["mask"], rows.shape[1]), float("-inf"))
        names, at = None, ids.view(ids.shape[0], -1)
    t = state["temperature"]
    t = t.unsqueeze(1) if isinstance(t, torch.Tensor) else t
    top = rows.amax(1, keepdim=True)
    z = (rows - top) / t
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    lse = torch.log(total)
    entropy = lse - torch.where(e > 0, e * z, 0.0).sum(1, keepdim=True) / total
    out = {"logprobs": (z.gather(1, at) - lse).view(ids.shape), "entropy": entropy.squeeze(1)}
    if state["op"] == "gradient":
        logp = z - lse
        g = state["grad_logprobs"].view(at.shape)
        p = e / total
        grad = torch.where(p > 0, -p * (g.sum(1, keepdim=True) + state["grad_entropy"].unsqueeze(1) * (logp + entropy)),
                           0.0)
        grad.scatter_add_(1, at, g)
        return {**out, "grad": (grad / t).to(x.dtype)}
    out["logsumexp"] = (top / t + lse).squeeze(1)
    # alternatives by falling logit, then rising id: whole numbers that sort this way
    bits = (rows + 0.0).view(torch.int32)
    rank = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long() << 32
    rank -= torch.arange(rows.shape[1], device=x.device)
    best = torch.topk(rank, min(n, rows.shape[1]), dim=1).indices
    best_logp = z.gather(1, best) - lse
    best_ids = best if names is None else names.gather(1, best)
    best_ids = torch.where(best_logp > float("-inf"), best_ids, -1)
    short = n - best.shape[1]
    out["top_ids"] = torch.nn.functional.pad(best_ids, (0, short), value=-1)
    out["top_logprobs"] = torch.nn.functional.pad(best_logp, (0, short), value=float("-inf"))
    return out


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_e4m3(x):
    """x [N, H] in 64 bits -> its e4m3 values and scales, both in 64 bits, rounded as they are held."""
    n, h = x.shape
    out, scales = torch.zeros_like(x), []
    for k0 in range(0, h, 128):
        part = x[:, k0:k0 + 128]
        s = (part.abs().max(dim=1).values.float().double() / 448.0).float().double()
        q = (part / s.clamp(min=1e-300).unsqueeze(1)).clamp(-448, 448).float().to(torch.float8_e4m3fn).double()
        out[:, k0:k0 + 128] = torch.where(s.unsqueeze(1) > 0, q, torch.zeros_like(q))
        scales.append(s)
    return out, torch.stack(scales, 1)


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return _exact(state)


def _exact(state):
    if state["op"] == "norm":
        h = state["x"].double()
        if state["residual"] is not None:
            h = (h + state["residual"].double()).to(state["x"].dtype).double()
        rms = ((h ** 2).sum(1) / h.shape[1] + EPS) ** 0.5
        y = h / rms.unsqueeze(1) * state["weight"].double()
        residual = h if state["residual"] is not None else None
        if state["out"] == "same":
            return {"values": y, "scales": None, "residual": residual}
        if state["out"] == "int8":
            s = y.abs().max(dim=1).values / 127.0
            return {"values": (y / s.unsqueeze(1)).round(), "scales": s, "residual": residual}
        values, scales = _exact_e4m3(y)
        return {"values": values, "scales": scales, "residual": residual}
    if state["op"] == "project":
        vocab, hidden = state["w"].shape
        if state["hs"] is None:
            h, hs = _exact_e4m3(state["h"].double())
        else:
            h, hs = state["h"].double(), state["hs"].double()
        h = h * hs[:, torch.arange(hidden, device=DEVICE) // 128]
        batch = h.shape[0]
        y = torch.empty(batch, vocab, dtype=torch.float64, device=DEVICE)
        block = torch.arange(hidden, device=DEVICE) // 128
        for v0 in range(0, vocab, 16384):  # blocks of the vocabulary
            v1 = min(vocab, v0 + 16384)
            by = state["ws"].double()[torch.arange(v0, v1, device=DEVICE) // 128]
            y[:, v0:v1] = h @ (state["w"][v0:v1].double() * by[:, block]).T
            if state["mask"] is not None:
                v = torch.arange(v0, v1, device=DEVICE)
                bit = (state["mask"].long()[:, v // 32] >> (v % 32)) & 1
                y[:, v0:v1][bit == 0] = -math.inf
        return {"logits": y}
    ids = state["ids"].view(state["ids"].shape[0], -1)
    batch, parts = ids.shape[0], {k: [] for k in ("logprobs", "entropy", "logsumexp", "top_logprobs", "grad")}
    for b in range(batch):
        row = state["x"]
        if state["form"] == "packed":
            lo, hi = int(state["offsets"][b]), int(state["offsets"][b + 1])
            row, mine = row[lo:hi].double(), torch.searchsorted(state["packed_ids"][lo:hi], ids[b])
        else:
            row, mine = row[b].double(), ids[b]
            if state["mask"] is not None:
                v = torch.arange(row.numel(), device=DEVICE)
                row = torch.where(((state["mask"][b].long()[v // 32] >> (v % 32)) & 1) == 1, row, -math.inf)
        t = state["temperature"]
        z = row / (t[b].double() if isinstance(t, torch.Tensor) else t)
        lse = torch.logsumexp(z, 0)
        logp = z - lse
        p = logp.exp()
        entropy = -torch.special.xlogy(p, p).sum()
        parts["logprobs"].append(logp[mine])
        parts["entropy"].append(entropy)
        if state["op"] == "gradient":
            g = state["grad_logprobs"].view(ids.shape)[b].double()
            d = -p * g.sum() - state["grad_entropy"][b].double() * (torch.special.xlogy(p, p) + p * entropy)
            d.index_add_(0, mine, g)
            d /= t[b].double() if isinstance(t, torch.Tensor) else t
            parts["grad"].append(d)
        else:
            parts["logsumexp"].append(lse)
            n = state["top_n"]
            best = torch.sort(logp, descending=True).values[:n]
            parts["top_logprobs"].append(torch.nn.functional.pad(best, (0, n - best.numel()), value=-math.inf))
    out = {k: torch.stack(v) for k, v in parts.items() if v}
    out["logprobs"] = out["logprobs"].view(state["ids"].shape)
    if state["op"] == "logprobs":
        out["top_ids"] = None
    return out
