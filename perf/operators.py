"""The head's int8 and sampling operators as they are measured: cases, inputs, plain forms.

Three operators of the grammar-conditioned LM head:

  quantize  rows (hidden states of a step, or the head's weight once) to int8
            with one scale per row;
  project   the LM head on int8 weights: quantise the step's hidden states,
            multiply in 8-bit integers, scale per token and channel, mask, and
            take the greedy top-1, on one of the three routes; or the legal
            tokens' logits alone, packed request by request;
  sample    temperature, top-k, min-p and top-p on masked logits and one draw
            per request from given uniform numbers, on vocabulary-shaped rows
            or on packed legal rows.

Sizes are those of the head benchmark of this repository (vocabularies of
248,320, 151,936 and 262,144 tokens; hidden sizes 1,024 to 8,192; batches 1 to
128) and generic ones between them.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DEVICE = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # the hidden states of one decode step of 64 requests
        {"name": "quantize-step", "op": "quantize", "rows": 64, "hidden": 2048, "dtype": "bf16"},
        # a whole head, once when a model is loaded
        {"name": "quantize-head", "op": "quantize", "rows": 248320, "hidden": 2048, "dtype": "fp16"},
        # one request under a grammar that leaves 1% of the vocabulary
        {"name": "project-one", "op": "project", "route": "row-sparse", "batch": 1, "vocab": 248320, "hidden": 2048,
         "dtype": "fp16", "density": 0.01, "clustered": False},
        # the packed legal logits of a few requests, for a sampler that follows
        {"name": "project-packed", "op": "project", "route": "packed", "batch": 8, "vocab": 248320, "hidden": 2048,
         "dtype": "bf16", "density": 0.005, "clustered": True},
        # batched decode, each request in a few runs of the vocabulary
        {"name": "project-block", "op": "project", "route": "block-sparse", "batch": 32, "vocab": 248320,
         "hidden": 2048, "dtype": "fp16", "density": 0.005, "clustered": True},
        # batched decode with free text among the requests
        {"name": "project-dense", "op": "project", "route": "dense-mask", "batch": 64, "vocab": 151936,
         "hidden": 1024, "dtype": "bf16", "density": 0.95, "clustered": False},
        # a wide head for a full batch
        {"name": "project-wide", "op": "project", "route": "dense-mask", "batch": 128, "vocab": 262144,
         "hidden": 8192, "dtype": "bf16", "density": 0.5, "clustered": True},
        # one request's step with all four filters
        {"name": "sample-one", "op": "sample", "form": "masked", "batch": 1, "vocab": 248320, "dtype": "fp16",
         "density": 0.01, "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.02, "mixed": False},
        # packed legal rows of a batch (1% of the vocabulary each)
        {"name": "sample-packed", "op": "sample", "form": "packed", "batch": 32, "vocab": 248320, "dtype": "fp16",
         "density": 0.01, "temperature": 0.7, "top_k": 0, "top_p": 0.9, "min_p": 0.0, "mixed": False},
        # free text, nucleus only, each request with settings of its own
        {"name": "sample-mixed", "op": "sample", "form": "bits", "batch": 64, "vocab": 151936, "dtype": "bf16",
         "density": 0.95, "temperature": 1.0, "top_k": 40, "top_p": 0.95, "min_p": 0.05, "mixed": True},
        # a full batch of unmasked rows in half precision, nucleus only
        {"name": "sample-batch", "op": "sample", "form": "free", "batch": 128, "vocab": 248320, "dtype": "bf16",
         "density": 1.0, "temperature": 0.9, "top_k": 0, "top_p": 0.9, "min_p": 0.0, "mixed": False},
        # 32-bit logits of the widest vocabulary, no filter but the temperature
        {"name": "sample-fp32", "op": "sample", "form": "free", "batch": 48, "vocab": 262144, "dtype": "fp32",
         "density": 1.0, "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "mixed": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("quantize", "project", "project", "sample", "sample"))
    dtype = rng.choice(("fp16", "bf16", "fp32"))
    if op == "quantize":
        hidden = _log(rng, 16, 8192)
        rows = _log(rng, 1, 248320 * 1024 // max(hidden, 1024))
        return {"op": op, "rows": rows, "hidden": hidden, "dtype": dtype}
    batch = _log(rng, 1, 128)
    if op == "project":
        vocab, hidden = _log(rng, 1000, 262144), _log(rng, 64, 8192)
        if rng.random() < 0.75:
            hidden = (hidden + 15) // 16 * 16  # whole 16-byte vectors, as nearly every model has them
        route = rng.choice(("row-sparse", "packed", "block-sparse", "dense-mask"))
        if hidden % 16 or route in ("row-sparse", "packed"):
            density = math.exp(rng.uniform(math.log(0.0005), math.log(0.05)))
        else:
            density = math.exp(rng.uniform(math.log(0.002), 0.0))
        return {"op": op, "route": route, "batch": batch, "vocab": vocab, "hidden": hidden, "dtype": dtype,
                "density": round(density, 5), "clustered": rng.random() < 0.5}
    form = rng.choice(("masked", "bits", "packed", "free"))
    density = 1.0 if form == "free" else math.exp(rng.uniform(math.log(0.001), 0.0))
    return {"op": op, "form": form, "batch": min(batch, 64), "vocab": _log(rng, 1000, 262144), "dtype": dtype,
            "density": round(density, 5), "temperature": round(rng.uniform(0.4, 1.5), 3),
            "top_k": rng.choice((0, 0, 1, 20, 50, 1000)), "top_p": rng.choice((1.0, 0.99, 0.95, 0.9, 0.8, 0.5)),
            "min_p": rng.choice((0.0, 0.0, 0.02, 0.1)), "mixed": rng.random() < 0.3}


def work(case):
    """Each input read once and each output written once."""
    size = TYPES[case["dtype"]].itemsize
    if case["op"] == "quantize":
        n = case["rows"] * case["hidden"]
        return {"bytes": n * (size + 1) + 4 * case["rows"], "flops": 3 * n}
    batch, vocab, density = case["batch"], case["vocab"], case["density"]
    legal = batch * vocab * density
    mask = batch * vocab / 8
    if case["op"] == "project":
        hidden, route = case["hidden"], case["route"]
        rows = vocab if route == "dense-mask" else vocab * (1.0 - (1.0 - density) ** batch)
        out = legal * (size + 8) if route == "packed" else batch * vocab * size
        return {"bytes": rows * (hidden + 4) + batch * hidden * size + mask + out + 12 * batch,
                "flops": 2 * hidden * (batch * vocab if route == "dense-mask" else legal)}
    read = {"masked": batch * vocab * size, "free": batch * vocab * size,
            "bits": batch * vocab * size + mask, "packed": legal * (size + 8) + 8 * batch}[case["form"]]
    return {"bytes": read + 20 * batch, "flops": 4 * (legal if case["form"] == "packed" else batch * vocab)}


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
    start = first + (torch.rand(batch, runs, generator=g, device=DEVICE) * room).long().minimum(room - 1)
    edge = torch.zeros(batch, vocab + 1, dtype=torch.int32, device=DEVICE)
    one = torch.ones_like(start, dtype=torch.int32)
    edge.scatter_add_(1, start, one)
    edge.scatter_add_(1, start + length, -one)
    return edge[:, :vocab].cumsum(1) > 0


def _pack(legal):
    """[B, V] truth values -> [B, ceil(V / 32)] int32, lowest bit first."""
    batch, vocab = legal.shape
    words = (vocab + 31) // 32
    bits = torch.zeros(batch, words * 32, dtype=torch.int64, device=legal.device)
    bits[:, :vocab] = legal
    word = (bits.view(batch, words, 32) << torch.arange(32, device=legal.device)).sum(2)
    return torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(torch.int32)


def _int8_rows(x):
    """The definition of quantize: scale = max |x| / 127, value = x / scale to the nearest (ties to even)."""
    x = x.float()
    scale = x.abs().amax(1) / 127.0
    q = torch.round(x / scale.unsqueeze(1))
    return torch.where(scale.unsqueeze(1) > 0, q, torch.zeros_like(q)).clamp_(-127, 127).to(torch.int8), scale


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dtype = TYPES[case["dtype"]]
    if case["op"] == "quantize":
        x = torch.randn(case["rows"], case["hidden"], generator=g, device=DEVICE)
        return {"op": "quantize", "x": x.mul_(0.02 if case["rows"] > 4096 else 1.0).to(dtype)}
    batch, vocab = case["batch"], case["vocab"]
    if case["op"] == "project":
        hidden = case["hidden"]
        values = torch.randn(vocab, hidden, generator=g, device=DEVICE)
        values, scales = _int8_rows(values.mul_(0.02))
        legal = _legal(g, batch, vocab, case["density"], case["clustered"])
        return {"op": "project", "route": case["route"],
                "h": torch.randn(batch, hidden, generator=g, device=DEVICE).to(dtype),
                "w": values, "ws": scales, "mask": _pack(legal), "legal_count": int(legal.sum())}
    # logits as a head writes them: a broad bell and a few tokens that stand out
    x = torch.randn(batch, vocab, generator=g, device=DEVICE).mul_(2.2)
    at = torch.randint(0, vocab, (batch, 24), generator=g, device=DEVICE)
    x.scatter_(1, at, 6.0 + 2.5 * torch.randn(batch, 24, generator=g, device=DEVICE))
    x = x.to(dtype)
    form = case["form"]
    state = {"op": "sample", "form": form, "u": torch.rand(batch, generator=g, device=DEVICE)}
    legal = _legal(g, batch, vocab, case["density"], False)
    if form == "masked":
        state["x"] = x.masked_fill_(~legal, float("-inf"))
    elif form == "packed":
        ids = legal.nonzero()
        counts = legal.sum(1)
        state.update(x=x[legal], ids=ids[:, 1].contiguous(), max_len=int(counts.max()),
                     offsets=torch.cat([counts.new_zeros(1), counts.cumsum(0)]))
    else:
        state.update(x=x, mask=_pack(legal) if form == "bits" else None)
    settings = {k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")}
    if case["mixed"]:  # every third request greedy, every third with one filter fewer
        i = torch.arange(batch, device=DEVICE)
        t = 0.5 + torch.rand(batch, generator=g, device=DEVICE)
        settings["temperature"] = torch.where(i % 3 == 2, torch.zeros_like(t), t)
        settings["top_k"] = torch.where(i % 3 == 1, 0, case["top_k"]).to(torch.int32)
        settings["top_p"] = torch.where(i % 2 == 0, case["top_p"], 1.0).to(torch.float32)
        settings["min_p"] = torch.where(i % 5 == 0, case["min_p"], 0.0).to(torch.float32)
    state["settings"] = settings
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "grammar-sparse-projection_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from gsp import int8_head, triton_runtime
    if state["op"] == "quantize":
        q = int8_head.quantize_rows_int8(state["x"], reciprocal=True)  # as torch takes amax / 127.0 on the GPU
        return {"values": q.values, "scales": q.scales}
    if state["op"] == "project":
        weight = int8_head.QuantizedRows(state["w"], state["ws"])
        if state["route"] == "packed":
            ids, logits, offsets = int8_head.int8_compact_logits(state["h"], weight, state["mask"],
                                                                 capacity=state["legal_count"], reciprocal=True)
            return {"ids": ids, "logits": logits, "offsets": offsets}
        logits, top, at = int8_head.int8_grammar_logits(state["h"], weight, state["mask"], route=state["route"],
                                                        reciprocal=True)
        return {"logits": logits, "top": top, "at": at}
    if state["form"] == "packed":
        r = triton_runtime.sample_compact_logits(state["ids"], state["x"], state["offsets"], uniforms=state["u"],
                                                 max_len=state["max_len"], **state["settings"])
    else:
        r = triton_runtime.sample_logits(state["x"], uniforms=state["u"], bitmask_gpu=state.get("mask"),
                                         **state["settings"])
    return {"token": r.token_ids, "logprob": r.logprobs, "kept": r.kept}


def _unpack(mask, vocab):
    v = torch.arange(vocab, device=mask.device)
    return ((mask[:, v >> 5] >> (v & 31)) & 1).bool()


def _run_plain(state):
    if state["op"] == "quantize":
        values, scales = _int8_rows(state["x"])
        return {"values": values, "scales": scales}
    if state["op"] == "project":
        h, w = state["h"], state["w"]
        batch, vocab = h.shape[0], w.shape[0]
        q, hs = _int8_rows(h)
        total = q.double() @ w.double().T  # whole numbers beyond 24 bits: exact in 64
        y = (total.float() * hs.unsqueeze(1) * state["ws"].unsqueeze(0)).to(h.dtype)
        legal = _unpack(state["mask"], vocab)
        if state["route"] == "packed":
            at = legal.nonzero()
            counts = legal.sum(1)
            return {"ids": at[:, 1].contiguous(), "logits": y[legal],
                    "offsets": torch.cat([counts.new_zeros(1), counts.cumsum(0)])}
        y = y.masked_fill(~legal, float("-inf"))
        top = y.amax(1, keepdim=True)
        v = torch.arange(vocab, device=h.device).expand(batch, vocab)
        at = torch.where(legal & (y == top), v, vocab).amin(1)
        return {"logits": y, "top": top.squeeze(1).float(), "at": torch.where(at < vocab, at, 0)}
    x, settings = state["x"], state["settings"]
    batch = state["u"].shape[0]
    if state["form"] == "packed":
        lengths = state["offsets"].diff()
        col = torch.arange(max(1, state["max_len"]), device=x.device)
        inside = col < lengths.unsqueeze(1)
        place = (state["offsets"][:-1].unsqueeze(1) + col).clamp_(max=max(0, x.numel() - 1))
        rows = torch.where(inside, x[place].float(), float("-inf"))
        at, logprob, kept = _filtered(rows, state["u"], **settings)
        token = state["ids"][place.gather(1, at.unsqueeze(1)).squeeze(1)]
        return {"token": torch.where(kept > 0, token, 0), "logprob": logprob, "kept": kept}
    rows = x.float()
    if state.get("mask") is not None:
        rows = rows.masked_fill(~_unpack(state["mask"], rows.shape[1]), float("-inf"))
    token, logprob, kept = _filtered(rows, state["u"], **settings)
    return {"token": token, "logprob": logprob, "kept": kept}


def _column(v, like):
    v = v if isinstance(v, torch.Tensor) else torch.full(like.shape, v, device=like.device, dtype=torch.float32)
    return v.double().unsqueeze(1)


def _filtered(x, u, temperature, top_k, top_p, min_p):
    """Place, log-probability and number of the tokens left, for rows x [B, N] in
    32 bits (-inf: not to be drawn). Sums and comparisons are in 64 bits: a
    border that 32 bits move by one token gives another token."""
    t, k, p, m, r = (_column(v, u) for v in (temperature, top_k, top_p, min_p, u))
    k = torch.where(t > 0, k, torch.ones_like(k))  # temperature 0 takes the first token
    t = torch.where(t > 0, t, torch.ones_like(t))
    x = torch.where(x.isnan(), float("-inf"), x)
    xs, order = torch.sort(x, dim=1, descending=True, stable=True)
    rank = torch.arange(x.shape[1], device=x.device)
    legal = xs > float("-inf")
    score = (xs.double() - xs[:, :1].double()) / t
    w = torch.where(xs == xs[:, :1], 1.0, torch.exp(score))
    keep = legal & ((k <= 0) | (rank < k)) & (w >= m)
    w = torch.where(keep, w, 0.0)
    upto = w.cumsum(1)
    keep &= (p >= 1) | (upto - w < p * upto[:, -1:]) | (rank == 0)
    w = torch.where(keep, w, 0.0)
    upto = w.cumsum(1)
    kept = keep.sum(1)
    at = (upto <= r * upto[:, -1:]).sum(1).clamp(max=x.shape[1] - 1).minimum((kept - 1).clamp(min=0)).unsqueeze(1)
    logprob = score.gather(1, at) - upto[:, -1:].log()
    some = kept > 0
    token = torch.where(some, order.gather(1, at).squeeze(1), 0)
    return token, torch.where(some, logprob.squeeze(1), float("-inf")).float(), kept.to(torch.int32)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if state["op"] == "quantize":
        if state["x"].numel() > 2 ** 28:
            rows = state["x"].double()
            scales = rows.abs().max(dim=1).values / 127
            return {"values": None, "scales": scales}
        x = state["x"].double().cpu().numpy()
        scales = np.abs(x).max(axis=1) / 127.0
        return {"values": None, "scales": scales}
    if state["op"] == "project":
        h = state["h"].double()
        scale = (h.abs().max(dim=1, keepdim=True).values.float() / 127.0).double()
        q = torch.where(scale > 0, (h / scale).round(), torch.zeros_like(h))
        vocab = state["w"].shape[0]
        words = state["mask"].cpu().numpy().view(np.uint32)
        legal = np.unpackbits(words.view(np.uint8), axis=1, bitorder="little")[:, :vocab].astype(bool)
        y = np.empty((h.shape[0], vocab))
        for v0 in range(0, vocab, 16384):  # blocks of the vocabulary
            w = state["w"][v0:v0 + 16384].double() * state["ws"][v0:v0 + 16384].double().unsqueeze(1)
            y[:, v0:v0 + 16384] = ((q * scale) @ w.T).cpu().numpy()
        if state["route"] == "packed":
            return {"ids": None, "logits": y[legal], "offsets": None}
        y[~legal] = -np.inf
        # the top-1 value is one of the rounded logits themselves: which one is no question of 64 bits
        return {"logits": y, "top": None, "at": None}
    x = state["x"].float().cpu().numpy().astype(np.float64)
    u = state["u"].cpu().numpy().astype(np.float64)
    batch = u.shape[0]
    if state["form"] == "packed":
        offsets = state["offsets"].cpu().numpy()
        rows = [x[offsets[b]:offsets[b + 1]] for b in range(batch)]
    else:
        if state.get("mask") is not None:
            words = state["mask"].cpu().numpy().view(np.uint32)
            legal = np.unpackbits(words.view(np.uint8), axis=1, bitorder="little")[:, :x.shape[1]].astype(bool)
            x = np.where(legal, x, -np.inf)
        rows = list(x)

    def setting(name, b):
        v = state["settings"][name]
        return float(v[b]) if isinstance(v, torch.Tensor) else float(np.float32(v))

    logprob = np.empty(batch)
    for b, row in enumerate(rows):
        t, k = setting("temperature", b), int(setting("top_k", b))
        row = np.sort(row[row > -np.inf])[::-1]
        if row.size == 0:
            logprob[b] = -np.inf
            continue
        if t == 0.0:
            logprob[b] = 0.0
            continue
        score = (row - row[0]) / t
        if k > 0:
            score = score[:k]
        weight = np.exp(score)
        weight = weight[weight >= setting("min_p", b)]
        if setting("top_p", b) < 1.0:
            reach = np.cumsum(weight)
            weight = weight[:1 + int(np.searchsorted(reach, setting("top_p", b) * reach[-1], side="left"))]
        reach = np.cumsum(weight)
        at = min(int(np.searchsorted(reach, u[b] * reach[-1], side="right")), weight.size - 1)
        logprob[b] = score[at] - math.log(reach[-1])
    return {"token": None, "logprob": logprob, "kept": None}
