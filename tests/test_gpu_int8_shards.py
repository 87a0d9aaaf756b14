"""GPU tests of the int8 head's top-1 keys and vocabulary offset (a weight that
is one row shard of a larger vocabulary), and of its top-1 on rows whose logits
are NaN. Integers and copies of logits: no tolerance."""
import numpy as np
import pytest
import torch

from gsp import _native
from gsp import int8_head as I
from gsp import triton_runtime as tr
from oracle import gsp_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _case(dev, dtype, batch, vocab, hidden):
    g = torch.Generator(device=dev).manual_seed(vocab)
    weight = I.QuantizedRows(torch.randint(-127, 128, (vocab, hidden), generator=g, device=dev, dtype=torch.int8),
                             torch.rand(vocab, generator=g, device=dev) * 2e-3 + 1e-4)
    h = torch.randn(batch, hidden, generator=g, device=dev).to(dtype)
    counts = [vocab // 7] * (batch - 1) + [0]
    mask = torch.from_numpy(O.make_batch_mask(np.random.default_rng(vocab), batch, vocab, counts)).to(dev)
    return h, weight, mask


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [(5, 6016, 64), (40, 4000, 30)])
def test_shards_merge_to_the_whole(cuda_device, dtype, case):
    batch, vocab, hidden = case
    dev = cuda_device
    h, weight, mask = _case(dev, dtype, *case)
    q = I.quantize_rows_int8(h)
    cut = 2048  # whole mask words
    for route in tr.ROUTES:
        logits, value, token = I.int8_grammar_logits(h, weight, mask, route=route)
        keys, parts = [], []
        for lo, hi in ((0, cut), (cut, vocab)):
            key = torch.empty(batch, dtype=torch.int64, device=dev)
            part = torch.empty(batch, hi - lo, dtype=dtype, device=dev)
            words = mask[:, lo // 32:(hi + 31) // 32].contiguous()
            _native.int8_logits(route, q.values, q.scales, weight.values[lo:hi], weight.scales[lo:hi], words, dtype,
                                logits=part, top_key=key, vocab_offset=lo)
            keys.append(key)
            parts.append(part)
        assert torch.equal(torch.cat(parts, 1), logits)
        merged_value = torch.empty(batch, device=dev)
        merged_token = torch.empty(batch, dtype=torch.int64, device=dev)
        _native.top1_from_keys(torch.maximum(*keys), merged_value, merged_token)
        assert torch.equal(merged_value, value) and torch.equal(merged_token, token)
    # packed: the shard's ids are the whole vocabulary's, and so are a sampler's
    words = mask[:, cut // 32:].contiguous()
    capacity = batch * (vocab - cut)
    ids = torch.full((capacity,), -1, dtype=torch.int64, device=dev)
    packed = torch.empty(capacity, dtype=dtype, device=dev)
    offsets = torch.empty(batch + 1, dtype=torch.int64, device=dev)
    key = torch.empty(batch, dtype=torch.int64, device=dev)
    _native.int8_compact(q.values, q.scales, weight.values[cut:], weight.scales[cut:], words, dtype, packed, ids,
                         offsets, top_key=key, vocab_offset=cut)
    n = int(offsets[-1])
    part = logits[:, cut:]
    legal = ~part.isneginf()
    assert torch.equal(ids[:n], legal.nonzero()[:, 1] + cut) and torch.equal(packed[:n], part[legal])
    assert (ids[n:] == -1).all() and torch.equal(key, keys[1])
    u = torch.rand(batch, device=dev)
    drawn = tr.sample_compact_logits(ids, packed, offsets, uniforms=u, top_k=9)
    token = torch.empty(batch, dtype=torch.int64, device=dev)
    logprob, kept = torch.empty(batch, device=dev), torch.empty(batch, dtype=torch.int32, device=dev)
    _native.sample_logits(part, None, (1.0, 9, 1.0, 0.0), u, token, logprob, kept, vocab_offset=cut)
    some = kept > 0
    assert torch.equal(token[some], drawn.token_ids[some]) and torch.equal(kept, drawn.kept)
    assert torch.equal(logprob, drawn.logprobs)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch", [2, 37])
def test_top1_of_rows_that_are_nan(cuda_device, dtype, batch):
    """As logits.argmax(-1): the first NaN, and NaN as the value."""
    dev = cuda_device
    h, weight, mask = _case(dev, dtype, batch, 3001, 128)
    h[0, 77] = float("nan")
    weight.scales[500:] = torch.where(torch.arange(2501, device=dev) % 3 == 0, float("nan"), weight.scales[500:])
    for route in tr.ROUTES:
        for words in (mask, None):
            logits, value, token = I.int8_grammar_logits(h, weight, words, route=route)
            at = logits.argmax(-1)
            assert torch.equal(token, at)
            assert torch.equal(value.isnan(), logits.gather(1, at.unsqueeze(1)).squeeze(1).isnan())
