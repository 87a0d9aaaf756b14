"""GPU tests of the norm, the fp8 head, the sampler and the log probabilities
together, as a decode step and a policy update use them, and of the decode loop
with them.

The step's logits are checked against 64-bit sums of the 8-bit operands the norm
wrote (the bound of the head's own tests: (264 + blocks + 16) * 2^-24 of the sum of
magnitudes, then half a step of the logits' type); the log probabilities against
64-bit ones of those very logits, to (V / 512 + 128 + 4 |logprob|) * 2^-24.
"""
import json
import math

import numpy as np
import pytest
import torch

from gsp import _native
from gsp import fp8_head as F
from gsp import int8_head as I
from gsp import logprobs as L
from gsp import norm
from gsp import triton_runtime as tr
from oracle import gsp_oracle as O

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -24


def _reference_logprobs(logits, ids, temperature):
    z = logits.double().cpu() / float(np.float32(temperature))
    return (z - torch.logsumexp(z, 1, keepdim=True)).gather(1, ids.cpu().view(-1, 1)).squeeze(1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_steps(cuda_device, dtype):
    dev, vocab, hidden, batch = cuda_device, 20_011, 512, 7
    g = torch.Generator().manual_seed(1)
    head = (torch.randn(vocab, hidden, generator=g) * 0.1).to(dtype).to(dev)
    weight, weight8 = F.quantize_weight_fp8(head), I.quantize_rows_int8(head)
    gain = (1 + 0.2 * torch.randn(hidden, generator=g)).to(dtype).to(dev)
    stream = torch.randn(batch, hidden, generator=g).to(dtype).to(dev)
    rng = np.random.default_rng(2)
    w64 = weight.values.double() * weight.scales.double().repeat_interleave(128, 0)[:vocab].repeat_interleave(128, 1)
    for step, counts in enumerate(([200] * batch, [0, 1, 5, vocab, 3000, 40, 2], [vocab] * batch)):
        mask_np = O.make_batch_mask(rng, batch, vocab, counts, clustered=step % 2 == 1, max_runs=6)
        mask, legal = torch.from_numpy(mask_np).to(dev), torch.from_numpy(O.unpack_bitmask(mask_np, vocab))
        x = torch.randn(batch, hidden, generator=g).to(dtype).to(dev)
        rows, after = norm.rms_norm(x, gain, residual=stream, quantize="fp8")
        assert torch.equal(after, (x.float() + stream.float()).to(dtype))
        h64 = rows.values.double() * rows.scales.double().repeat_interleave(128, 1)
        exact, size = (h64 @ w64.T).cpu(), (h64.abs() @ w64.abs().T).cpu()
        bound = size * (264 + 4 + 16) * STEP
        bound = bound + (exact.abs() + bound) * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).tiny
        u = torch.rand(batch, generator=g).to(dev)
        for route in tr.ROUTES:
            logits, _, greedy = F.fp8_grammar_logits(rows, weight, mask, route=route, out_dtype=dtype)
            got = logits.cpu().double()
            assert (got[~legal] == -math.inf).all() and ((got - exact).abs() <= bound)[legal].all()
            drawn = tr.sample_logits(logits, uniforms=u, temperature=0.8, top_p=0.95)
            r = L.token_logprobs(logits, drawn.token_ids, temperature=0.8, top_n=4)
            want = _reference_logprobs(logits, drawn.token_ids, 0.8)
            some = legal.any(1)
            off = (r.logprobs.double().cpu() - want).abs()[some]
            assert (off <= (vocab / 512 + 128 + 4 * want[some].abs()) * STEP).all()
            assert torch.equal(r.top_ids[some.to(dev), 0], greedy[some.to(dev)])
            assert (r.logprobs.cpu()[~some] == -math.inf).all()
        # the int8 head takes the norm's int8 rows, to the bits of its own quantiser on the same values
        rows8 = norm.rms_norm(x, gain, residual=stream, quantize="int8").output
        first, _, _ = I.int8_grammar_logits(rows8, weight8, mask, route="row-sparse", out_dtype=dtype)
        assert torch.equal(first, I.int8_grammar_logits(rows8, weight8, mask, route="dense-mask", out_dtype=dtype)[0])
        stream = after
    assert _native.workspace_error(dev) == 0


def test_step_captured_and_replayed(cuda_device):
    """Norm, projection, draw and log probabilities in one CUDA graph, new inputs at every replay."""
    dev, vocab, hidden, batch = cuda_device, 9_001, 256, 5
    g = torch.Generator().manual_seed(3)
    weight = F.quantize_weight_fp8((torch.randn(vocab, hidden, generator=g) * 0.1).to(dev))
    rng = np.random.default_rng(4)

    def inputs():
        mask = torch.from_numpy(O.make_batch_mask(rng, batch, vocab, [50, 900, 4000, 0, vocab])).to(dev)
        return [torch.randn(batch, hidden, generator=g).half().to(dev), torch.randn(batch, hidden, generator=g).half().to(dev),
                mask, torch.rand(batch, generator=g).to(dev)]

    def step(x, stream, mask, u):
        rows, after = norm.rms_norm(x, residual=stream, quantize="fp8")
        logits, _, greedy = F.fp8_grammar_logits(rows, weight, mask, route="block-sparse", out_dtype=torch.float16)
        drawn = tr.sample_logits(logits, uniforms=u, top_p=0.9, temperature=0.7)
        return (after, logits, greedy, drawn.token_ids, *L.token_logprobs(logits, drawn.token_ids, temperature=0.7, top_n=3))

    static = inputs()
    step(*static)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for _ in range(4):
        new = inputs()
        want = step(*new)
        for s, n in zip(static, new):
            s.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_policy_update_through_the_head(cuda_device):
    """Logits of a plain fp16 head, scored and pushed back to the hidden states: the gradient of the logits reaches
    them through torch's own product, and matches the formula's in 64 bits."""
    dev, vocab, hidden, batch = cuda_device, 5003, 128, 6
    g = torch.Generator().manual_seed(5)
    head = (torch.randn(vocab, hidden, generator=g) * 0.1).to(dev)
    h = torch.randn(batch, hidden, generator=g).to(dev).requires_grad_(True)
    ids = torch.randint(0, vocab, (batch,), generator=g).to(dev)
    advantage = torch.randn(batch, generator=g).to(dev)
    r = L.token_logprobs(h @ head.T, ids, temperature=0.9)
    (-(r.logprobs * advantage).mean() - 0.01 * r.entropy.mean()).backward()
    h64 = h.detach().double().requires_grad_(True)
    lp = torch.log_softmax(h64 @ head.double().T / float(np.float32(0.9)), 1)
    loss = -(lp.gather(1, ids.view(-1, 1)).squeeze(1) * advantage.double()).mean() - 0.01 * -(lp.exp() * lp).sum(1).mean()
    loss.backward()
    # the product's own rounding: 128 terms of the logits, 5,003 of the gradient, in fp32
    bound = (h64.grad.abs().max() + head.abs().max()) * (5003 + 2 * 300) * STEP
    assert (h.grad.double() - h64.grad).abs().max() <= bound


SCHEMAS = [
    {"type": "object",
     "properties": {"unit": {"enum": ["kg", "lb", "oz"]}, "fragile": {"type": "boolean"}},
     "required": ["unit", "fragile"], "additionalProperties": False},
    {"type": "object",
     "properties": {"op": {"const": "resize"}, "count": {"type": "integer", "minimum": 0, "maximum": 99}},
     "required": ["op", "count"], "additionalProperties": False},
]


@pytest.mark.parametrize("head,fused", [("fp8", False), ("fp8", True), ("int8", True)])
def test_decode_loop(cuda_device, head, fused):
    from gsp.decode_loop import GrammarDecodeLoop, SyntheticVocabulary, TinyDecoder
    size, hidden = 32_768, 512
    vocab = SyntheticVocabulary(size, extra_pieces=("unit", "count", "fragile", "resize"))
    g = torch.Generator().manual_seed(11)
    w = (torch.randn(size, hidden, generator=g) * 0.02).half().to(cuda_device)
    loop = GrammarDecodeLoop(TinyDecoder(size, hidden, seed=3, device=cuda_device), w, vocab, head=head, fused_norm=fused)
    seen = []

    def on_step(step, hidden, mask, logits, greedy, route):
        seen.append((hidden, logits.clone()))

    gen = torch.Generator(device=cuda_device).manual_seed(5)
    out, records = loop.run(SCHEMAS, max_steps=40, sampling=dict(temperature=1.2, top_k=50), generator=gen, logprobs=3,
                            on_step=on_step)
    kind = {"fp8": F.Fp8Rows, "int8": I.QuantizedRows}[head]
    for record, (h, logits) in zip(records, seen):
        assert isinstance(h, kind) == fused
        ids = torch.tensor(record.tokens)
        want = _reference_logprobs(logits, ids, 1.2)
        for b, worth in enumerate(record.logprobs):
            assert abs(worth["logprob"] - want[b].item()) <= (size / 512 + 128 + 4 * abs(want[b].item())) * STEP
            assert worth["entropy"] >= 0 and len(worth["top"]) <= 3
            assert worth["top"][0][0] == int(logits[b].argmax())
    for b, schema in enumerate(SCHEMAS):
        if out[b] and out[b][-1] == vocab.stop_id:
            assert set(json.loads(vocab.decode(out[b]))) == set(schema["required"])
    greedy, records = loop.run(SCHEMAS, max_steps=4)
    assert all(r.logprobs is None for r in records)


def test_decode_loop_refuses_a_fused_norm_for_other_heads(cuda_device):
    from gsp.decode_loop import GrammarDecodeLoop
    with pytest.raises(ValueError, match="fused_norm"):
        GrammarDecodeLoop(None, None, None, head="dense", fused_norm=True)
