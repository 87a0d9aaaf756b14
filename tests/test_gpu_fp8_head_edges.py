"""GPU tests of the fp8 head's top-1 keys and vocabulary offset (a weight that is one row shard of a larger
vocabulary), of its top-1 where every legal logit rounds to -inf, and of the number of logits. Integers and copies
of logits: no tolerance."""
import math

import numpy as np
import pytest
import torch

from gsp import _native
from gsp import fp8_head as F
from gsp import triton_runtime as tr
from oracle import gsp_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [(5, 6016, 64), (40, 4000, 30), (200, 4000, 256)])
def test_shards_merge_to_the_whole(cuda_device, dtype, case):
    batch, vocab, hidden = case
    dev, cut = cuda_device, 2048  # whole mask words and blocks
    g = torch.Generator().manual_seed(vocab)
    w = (torch.randn(vocab, hidden, generator=g) * 0.02)
    w[cut:cut + 128] = w[cut - 128:cut] * 8  # the largest logits, the same on both sides of the border
    w[cut - 128:cut] *= 8
    weight = F.quantize_weight_fp8(w.to(dev))
    rows = F.quantize_rows_fp8(torch.randn(batch, hidden, generator=g).to(dev))
    counts = [vocab // 7] * (batch - 2) + [0, vocab]
    mask = torch.from_numpy(O.make_batch_mask(np.random.default_rng(vocab), batch, vocab, counts)).to(dev)
    mask[:batch - 2, (cut - 128) // 32:(cut + 128) // 32] = -1
    for route in tr.ROUTES:
        for words in (mask, None):
            logits, value, token = F.fp8_grammar_logits(rows, weight, words, route=route, out_dtype=dtype)
            keys, parts = [], []
            for lo, hi in ((0, cut), (cut, vocab)):
                key = torch.empty(batch, dtype=torch.int64, device=dev)
                part = torch.empty(batch, hi - lo, dtype=dtype, device=dev)
                some = None if words is None else words[:, lo // 32:(hi + 31) // 32].contiguous()
                _native.fp8_logits(route, rows.values, rows.scales, weight.values[lo:hi],
                                   weight.scales[lo // 128:(hi + 127) // 128], some, dtype, logits=part, top_key=key,
                                   vocab_offset=lo)
                keys.append(key)
                parts.append(part)
            assert torch.equal(torch.cat(parts, 1), logits)
            merged_value = torch.empty(batch, device=dev)
            merged_token = torch.empty(batch, dtype=torch.int64, device=dev)
            _native.top1_from_keys(torch.maximum(*keys), merged_value, merged_token)
            assert torch.equal(merged_value, value) and torch.equal(merged_token, token)
            assert torch.equal(token.cpu(), logits.float().cpu().argmax(1))
    assert _native.workspace_error(dev) == 0


@pytest.mark.parametrize("batch", [4, 150])
def test_top1_where_legal_logits_round_to_minus_infinity(cuda_device, batch):
    """As logits.argmax(-1): token 0 where every logit is -inf, on every route, with one key for all."""
    vocab, hidden, dev = 700, 256, cuda_device
    weight = F.quantize_weight_fp8(torch.where(torch.arange(vocab, device=dev) == 650, 1.0, -10.0).unsqueeze(1).expand(vocab, hidden).contiguous())
    h = torch.full((batch, hidden), 40.0, device=dev)  # logits -102,400 (fp16: -inf), token 650's 10,240
    legal = np.zeros((batch, (vocab + 31) // 32 * 32), dtype=np.uint8)
    legal[0, 77] = 1
    legal[1, 77:690] = 1
    legal[1, 650] = 0
    legal[2, 77:690] = 1
    legal[3:, :vocab] = np.random.default_rng(1).random((batch - 3, vocab)) < 0.1
    mask = torch.from_numpy(np.packbits(legal, axis=1, bitorder="little").view(np.int32).copy()).to(dev)
    found = []
    for route in tr.ROUTES:
        for dtype in DTYPES:
            logits, value, token = F.fp8_grammar_logits(h, weight, mask, route=route, out_dtype=dtype)
            first = logits.float().cpu().argmax(1)
            assert torch.equal(token.cpu(), first), (route, dtype)
            assert torch.equal(value.cpu(), logits.float().cpu().gather(1, first.unsqueeze(1)).squeeze(1))
            if dtype == torch.float16:
                assert (logits[:2] == -math.inf).all() and token[:3].tolist() == [0, 0, 650]
        key = torch.empty(batch, dtype=torch.int64, device=dev)
        _native.fp8_logits(route, h.half(), None, weight.values, weight.scales, mask, torch.float16, top_key=key)
        found.append(key)
    assert torch.equal(found[0], found[1]) and torch.equal(found[0], found[2])


def test_logits_past_the_limit_are_refused(cuda_device):
    """More than 2^32 - 1 logits, whole mask words counted."""
    dev = cuda_device
    h = torch.zeros(65536, 1, device=dev)
    for vocab in (65536, 65505):
        weight = F.Fp8Weight(torch.zeros(vocab, 1, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn),
                             torch.zeros(512, 1, device=dev))
        before = torch.cuda.memory_allocated()
        with pytest.raises(ValueError, match="2\\^32"):
            F.fp8_grammar_logits(h, weight, None, route="dense-mask")
        assert torch.cuda.memory_allocated() == before
