"""GPU test: calls that need no workspace (row-sparse, no top-1) but are given
one too small for their sizes leave it alone. The sizes are those of the
cooperative kernel, which a workspace of full size would choose."""
import ctypes

import numpy as np
import pytest
import torch

from gsp import _native
from gsp import int8_head as I
from gsp import triton_runtime as tr
from oracle import gsp_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("offered", [0, 4096, "one less"])
def test_a_workspace_too_small_is_not_used(cuda_device, int8, offered):
    dev = cuda_device
    batch, vocab, hidden = 16, 40000, 128
    g = torch.Generator(device=dev).manual_seed(1)
    mask = torch.from_numpy(O.make_batch_mask(np.random.default_rng(1), batch, vocab, [300] * batch)).to(dev)
    h = torch.randn(batch, hidden, generator=g, device=dev).half()
    lib = _native.load()
    need = _native._workspace_bytes(batch, vocab)
    space = torch.full((2 * need,), 0xAB, dtype=torch.uint8, device=dev)
    stream = ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)
    logits = torch.empty(batch, vocab, dtype=torch.float16, device=dev)
    p = lambda t: ctypes.c_void_p(t.data_ptr())
    if offered == "one less":  # than the row-sparse part of it
        offered = _row_sparse_bytes(batch, vocab) - 1
    if int8:
        weight = I.quantize_rows_int8(torch.randn(vocab, hidden, generator=g, device=dev))
        want = I.int8_grammar_logits(h, weight, mask)[0]
        q = I.quantize_rows_int8(h)
        status = lib.gsp_int8_logits(0, p(q.values), hidden, _native.DTYPE_I8, p(q.scales), p(weight.values), hidden,
                                     p(weight.scales), p(mask), mask.stride(0), batch, vocab, hidden, 0, 0, p(logits),
                                     vocab, None, None, None, None, 0, p(space), offered, stream)
    else:
        weight = torch.randn(vocab, hidden, generator=g, device=dev).half()
        want = tr.grammar_logits_with_top1(h, weight, mask, route="row-sparse")[0]
        status = lib.gsp_row_sparse_logits(p(h), hidden, p(weight), hidden, p(mask), mask.stride(0), batch, vocab,
                                           hidden, 0, 0, p(logits), vocab, None, None, None, p(space), offered, stream)
    assert status == _native.GSP_OK
    torch.cuda.synchronize()
    assert torch.equal(logits.isneginf(), want.isneginf())
    legal = ~want.isneginf()
    if int8:
        assert torch.equal(logits, want)
    else:  # fp32 sums of 128 products in any order, then half a step of fp16 (129: their product)
        exact = (h.double() @ weight.double().T)[legal]
        bound = exact.abs() * 2.0 ** -11 + 129 * 2.0 ** -24 * (h.double().abs() @ weight.double().abs().T)[legal]
        assert ((logits.double()[legal] - exact).abs() <= bound + 2.0 ** -25).all()
    assert (space == 0xAB).all()


def _row_sparse_bytes(batch, vocab):
    """The least size that such a call with a top-1 accepts (refusals launch nothing)."""
    lib, fake = _native.load(), ctypes.c_void_p(4096)
    refused = lib.gsp_row_sparse_logits(fake, 64, fake, 64, None, 0, batch, vocab, 64, 0, 0, None, 0, fake, None, None,
                                        fake, 1, None)
    assert refused == _native.GSP_ERR_WORKSPACE
    return int(lib.gsp_last_error().split(b"needs ")[1])
