"""GPU test of the int8 head and the filtered sampler together, as a decode
step uses them: quantise the weight once; per step quantise the hidden states,
project under the grammar mask, draw.

One step by step against 64-bit oracles with masks of every kind, whole and
packed rows; then the decode loop with xgrammar matchers, which must accept
every drawn token.
"""
import json

import numpy as np
import pytest
import torch

from gsp import _native
from gsp import int8_head as I
from gsp import triton_runtime as tr
from oracle import gsp_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_steps_against_oracles(cuda_device, dtype):
    dev = cuda_device
    vocab, hidden, batch = 20_011, 512, 7
    g = torch.Generator(device="cpu").manual_seed(1)
    head = (torch.randn(vocab, hidden, generator=g) * 0.1).to(dtype).to(dev)
    weight = I.quantize_rows_int8(head)
    w64 = weight.values.double().cpu().numpy().astype(np.int64)
    ws = weight.scales.cpu()
    rng = np.random.default_rng(2)
    settings = dict(temperature=0.8, top_k=60, top_p=0.95, min_p=0.01)
    for step, counts in enumerate(([200] * batch, [0, 1, 5, vocab, 3000, 40, 2], [vocab] * batch)):
        mask_np = O.make_batch_mask(rng, batch, vocab, counts, clustered=step % 2 == 1, max_runs=6)
        mask = torch.from_numpy(mask_np).to(dev)
        h = torch.randn(batch, hidden, generator=g).to(dtype).to(dev)
        u = torch.rand(batch, generator=g).to(dev)
        logits = None
        for route in tr.ROUTES:
            got, _, top = I.int8_grammar_logits(h, weight, mask, route=route)
            assert logits is None or torch.equal(got, logits)
            logits = got
        # the product's definition: exact sums, two fp32 products, one rounding
        q = I.quantize_rows_int8(h)
        total = torch.from_numpy(q.values.cpu().numpy().astype(np.int64) @ w64.T)
        legal = torch.from_numpy(O.unpack_bitmask(mask_np, vocab))
        want = (total.float() * q.scales.cpu().unsqueeze(1) * ws.unsqueeze(0)).to(dtype)
        assert torch.equal(logits.cpu(), want.masked_fill(~legal, float("-inf")))
        assert torch.equal(top, logits.argmax(-1))
        whole = tr.sample_logits(logits, uniforms=u, **settings)
        ids, packed, offsets = I.int8_compact_logits(h, weight, mask)
        parts = tr.sample_compact_logits(ids, packed, offsets, uniforms=u, **settings)
        assert torch.equal(whole.token_ids, parts.token_ids) and torch.equal(whole.kept, parts.kept)
        for b in range(batch):
            at, logprob, kept = O.filtered_sample_reference(logits[b].double().cpu().numpy(), u[b].item(), **settings)
            assert whole.token_ids[b].item() == at and whole.kept[b].item() == kept, (step, b)
            if kept:
                assert legal[b, at]
                assert abs(whole.logprobs[b].item() - logprob) <= abs(logprob) * 2.0 ** -24 + 1e-11
    assert _native.workspace_error(dev) == 0


def test_step_captured_and_replayed(cuda_device):
    """The whole step in one CUDA graph: new hidden states, mask and uniform numbers at every replay."""
    dev = cuda_device
    vocab, hidden, batch = 9_001, 256, 3
    g = torch.Generator(device="cpu").manual_seed(3)
    weight = I.quantize_rows_int8((torch.randn(vocab, hidden, generator=g) * 0.1).half().to(dev))
    rng = np.random.default_rng(4)

    def inputs():
        mask = torch.from_numpy(O.make_batch_mask(rng, batch, vocab, [50, 900, 4000])).to(dev)
        return (torch.randn(batch, hidden, generator=g).half().to(dev), mask, torch.rand(batch, generator=g).to(dev))

    def step(h, mask, u):
        logits, _, _ = I.int8_grammar_logits(h, weight, mask, route="block-sparse")
        return tr.sample_logits(logits, uniforms=u, top_p=0.9, temperature=0.7)

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


SCHEMAS = [
    {"type": "object",
     "properties": {"unit": {"enum": ["kg", "lb", "oz"]}, "fragile": {"type": "boolean"}},
     "required": ["unit", "fragile"], "additionalProperties": False},
    {"type": "object",
     "properties": {"op": {"const": "resize"}, "count": {"type": "integer", "minimum": 0, "maximum": 99}},
     "required": ["op", "count"], "additionalProperties": False},
]


@pytest.mark.parametrize("head", ["int8", "adaptive", "graphed"])
def test_decode_loop_draws_what_the_grammar_allows(cuda_device, head):
    from gsp.decode_loop import GrammarDecodeLoop, SyntheticVocabulary, TinyDecoder
    size, hidden = 32_768, 512
    vocab = SyntheticVocabulary(size, extra_pieces=("unit", "count", "fragile", "resize"))
    g = torch.Generator(device="cpu").manual_seed(11)
    w = (torch.randn(size, hidden, generator=g) * 0.02).half().to(cuda_device)
    loop = GrammarDecodeLoop(TinyDecoder(size, hidden, seed=3, device=cuda_device), w, vocab, head=head)
    settings = dict(temperature=1.2, top_k=50, top_p=0.98)

    def run(seed):
        seen = []
        gen = torch.Generator(device=cuda_device).manual_seed(seed)
        out, records = loop.run(SCHEMAS, max_steps=40, sampling=settings, generator=gen,
                                on_step=lambda step, h, m, logits, greedy, route: seen.append(logits.clone()))
        return out, records, seen

    out, records, seen = run(5)
    # the same generator gives the same text; the tokens are sample_logits' own
    again, _, _ = run(5)
    assert out == again
    gen = torch.Generator(device=cuda_device).manual_seed(5)
    for record, logits in zip(records, seen):
        u = torch.rand(len(SCHEMAS), device=cuda_device, generator=gen)
        assert tr.sample_logits(logits, uniforms=u, **settings).token_ids.tolist() == record.tokens
    for b, schema in enumerate(SCHEMAS):
        text = vocab.decode(out[b])
        if len(out[b]) and out[b][-1] == vocab.stop_id:
            assert set(json.loads(text)) == set(schema["required"])
    with pytest.raises(ValueError, match="teacher-forced"):
        loop.run(SCHEMAS, targets=[[0], [0]], sampling=settings)
