"""GPU test that the decode loop with the 8-bit heads decodes whole documents, and that its greedy tokens are the
largest of the logits it reports."""
import json

import pytest
import torch

from test_gpu_norm_fp8_logprobs_loop import SCHEMAS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("head,fused", [("fp8", False), ("fp8", True), ("int8", True)])
def test_requests_finish(cuda_device, head, fused):
    from gsp.decode_loop import GrammarDecodeLoop, SyntheticVocabulary, TinyDecoder
    size, hidden = 32_768, 512
    vocab = SyntheticVocabulary(size, extra_pieces=("unit", "count", "fragile", "resize"))
    g = torch.Generator().manual_seed(11)
    w = (torch.randn(size, hidden, generator=g) * 0.02).half().to(cuda_device)
    loop = GrammarDecodeLoop(TinyDecoder(size, hidden, seed=3, device=cuda_device), w, vocab, head=head, fused_norm=fused)
    steps = []
    gen = torch.Generator(device=cuda_device).manual_seed(5)
    out, records = loop.run(SCHEMAS, max_steps=400, sampling=dict(temperature=1.2, top_k=50), generator=gen, logprobs=3,
                            on_step=lambda step, *_: steps.append(step))
    assert steps == list(range(len(records))) and records and all(out)
    assert all(len(r.logprobs) == len(SCHEMAS) for r in records)
    finished = 0
    for tokens, schema in zip(out, SCHEMAS):
        if tokens[-1] == vocab.stop_id:
            assert set(json.loads(vocab.decode(tokens))) == set(schema["required"])
            finished += 1
    assert finished > 0
    taken = []
    out, records = loop.run(SCHEMAS, max_steps=6, on_step=lambda step, h, mask, logits, greedy, route:
                            taken.append((logits.float().cpu().argmax(1).tolist(), [int(t) for t in greedy])))
    assert len(taken) == len(records) > 0
    for record, (largest, greedy) in zip(records, taken):
        assert record.tokens == largest == greedy and record.logprobs is None
