"""GPU tests of the fp8 head's top-1 where every legal logit rounds to -inf. Integers and copies of logits: no
tolerance."""
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
