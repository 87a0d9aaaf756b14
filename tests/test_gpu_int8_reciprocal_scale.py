"""GPU tests of the int8 head's scales by the reciprocal (reciprocal=True):
scale = max |x| * fp32(1 / 127), value = x / scale to the nearest. Bit for bit
what torch computes on the GPU for amax / 127.0 and x / scale, and what numpy's
fp32 product gives; no tolerance."""
import ctypes

import numpy as np
import pytest
import torch

from gsp import _native
from gsp import int8_head as I
from gsp import triton_runtime as tr
from oracle import gsp_oracle as O

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _torch_rows(x):
    """Rows to int8 by torch expressions."""
    x = x.float()
    scale = x.abs().amax(1) / 127.0
    q = torch.round(x / scale.unsqueeze(1))
    return torch.where(scale.unsqueeze(1) > 0, q, torch.zeros_like(q)).clamp_(-127, 127).to(torch.int8), scale


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (64, 2048), (4097, 512), (1500, 1023), (2, 40000), (30000, 96), (7, 24)])
def test_rows_match_torch_and_numpy(cuda_device, dtype, shape):
    g = torch.Generator(device=cuda_device).manual_seed(sum(shape))
    x = torch.randn(*shape, generator=g, device=cuda_device).mul_(0.02).to(dtype)
    x[shape[0] // 2] = 0.0
    got = I.quantize_rows_int8(x, reciprocal=True)
    values, scales = _torch_rows(x)
    assert torch.equal(got.scales, scales) and torch.equal(got.values, values)
    amax = x.float().abs().amax(1).cpu().numpy()
    assert np.array_equal(got.scales.cpu().numpy(), amax * (np.float32(1) / np.float32(127)))
    # the division's scales are within one step of the product's, and the default
    step = np.spacing(amax / np.float32(127))
    divided = I.quantize_rows_int8(x).scales.cpu().numpy()
    assert np.array_equal(divided, amax / np.float32(127)) and (np.abs(divided - got.scales.cpu().numpy()) <= step).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [(1, 5000, 2048), (4, 3000, 48), (33, 2500, 1040), (16, 40000, 128), (3, 777, 31)])
def test_projections_quantise_their_hidden_states_so(cuda_device, dtype, case):
    """Every route and the packed logits: the bits of rows quantised before the call."""
    batch, vocab, hidden = case
    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(vocab)
    weight = I.QuantizedRows(torch.randint(-127, 128, (vocab, hidden), generator=g, device=dev, dtype=torch.int8),
                             torch.rand(vocab, generator=g, device=dev) * 2e-3 + 1e-4)
    h = torch.randn(batch, hidden, generator=g, device=dev).to(dtype)
    mask = torch.from_numpy(O.make_batch_mask(np.random.default_rng(batch), batch, vocab, [vocab // 9] * batch)).to(dev)
    q = I.QuantizedRows(*_torch_rows(h))
    for route in tr.ROUTES:
        want = I.int8_grammar_logits(q, weight, mask, route=route, out_dtype=dtype)
        got = I.int8_grammar_logits(h, weight, mask, route=route, reciprocal=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    want = I.int8_compact_logits(q, weight, mask, out_dtype=dtype)
    got = I.int8_compact_logits(h, weight, mask, reciprocal=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(ValueError, match="reciprocal"):
        I.int8_grammar_logits(q, weight, mask, out_dtype=dtype, reciprocal=True)


def test_refusals():
    """At the C ABI, before any device work (no kernel is launched)."""
    lib, fake = _native.load(), ctypes.c_void_p(4096)
    q = lib.gsp_quantize_rows_int8
    for dtype in (_native.SCALE_RECIPROCAL + 3, 2 * _native.SCALE_RECIPROCAL, -1):
        assert q(fake, 8, 4, 8, dtype, fake, 8, fake, None) == _native.GSP_ERR_UNSUPPORTED
    assert q(None, 8, 0, 8, _native.SCALE_RECIPROCAL + 1, None, 8, None, None) == _native.GSP_OK  # no rows
    for dtype in (_native.SCALE_RECIPROCAL + _native.DTYPE_I8, _native.SCALE_RECIPROCAL + 4):
        assert lib.gsp_int8_logits(0, fake, 64, dtype, fake, fake, 64, fake, None, 0, 2, 64, 64, 0, 0, None, 64, None,
                                   None, None, fake, 1 << 20, fake, 1 << 30, None) == _native.GSP_ERR_UNSUPPORTED
        assert b"hidden_dtype" in lib.gsp_last_error()
