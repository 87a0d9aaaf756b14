"""GPU tests of what the norm and the quantisers write into tensors that the caller gives: overlaps that would be read
after they are written, and the tensors' versions, which autograd goes by. And that forward-mode gradients, which the norm and
the log probabilities do not have, are refused."""
import pytest
import torch

from gsp import fp8_head as F
from gsp import int8_head as I
from gsp import logprobs as L
from gsp import norm

pytestmark = pytest.mark.gpu


def test_residual_out_may_be_an_input_but_not_a_part_of_one(cuda_device):
    n, h = 9, 256
    buffer = torch.randn(n, 3 * h + 8, generator=torch.Generator().manual_seed(1)).to(cuda_device)
    x, residual = buffer[:, :h], buffer[:, h:2 * h]
    want = norm.rms_norm(x.clone(), residual=residual.clone())
    for out in (residual, x, buffer[:, 2 * h:3 * h]):  # rows between the inputs' rows share no element with them
        kept = buffer.clone()
        r = norm.rms_norm(x, residual=residual, residual_out=out)
        assert r.residual.data_ptr() == out.data_ptr()
        assert torch.equal(r.residual, want.residual) and torch.equal(r.output, want.output)
        buffer.copy_(kept)
    flat = buffer.view(-1)
    weight = flat[5:5 + h]
    with pytest.raises(ValueError, match="overlap"):
        norm.rms_norm(torch.zeros(n, h, device=cuda_device), weight, residual=torch.zeros(n, h, device=cuda_device),
                      residual_out=flat[:n * h].view(n, h))
    for out in (buffer[:, 8:h + 8], buffer[:, h - 1:2 * h - 1], flat[:n * h].view(n, h), flat[h:h + n * h].view(n, h),
                flat[1:1 + n * (2 * h)].view(n, 2 * h)[:, :h]):
        with pytest.raises(ValueError, match="overlap"):
            norm.rms_norm(x, residual=residual, residual_out=out)
    one = torch.zeros(2 * h, device=cuda_device)
    with pytest.raises(ValueError, match="overlap"):
        norm.rms_norm(one[:h], residual=one[h:], residual_out=one[1:h + 1])
    norm.rms_norm(one[:h], residual=one[h:], residual_out=one[:h])
    norm.rms_norm(one.view(2, h)[:1], residual=one.view(2, h)[1:], residual_out=one.view(1, 2 * h)[:, :h])
    assert torch.equal(buffer, kept)


def test_quantised_outputs_must_not_overlap(cuda_device):
    n, h = 64, 256
    raw = torch.zeros(4 * n * h, dtype=torch.uint8, device=cuda_device)
    x = raw[:2 * n * h].view(torch.float16).view(n, h)
    values = torch.empty(n, h, dtype=torch.float8_e4m3fn, device=cuda_device)
    scales = torch.empty(n, 2, device=cuda_device)
    inside = raw[n * h:2 * n * h].view(torch.float8_e4m3fn).view(n, h)
    beside = raw[2 * n * h:3 * n * h].view(torch.float8_e4m3fn).view(n, h)
    for bad in (F.Fp8Rows(inside, scales), F.Fp8Rows(values, raw[:n * 8].view(torch.float32).view(n, 2)),
                F.Fp8Rows(beside, raw[2 * n * h:2 * n * h + n * 8].view(torch.float32).view(n, 2))):
        with pytest.raises(ValueError, match="overlap"):
            F.quantize_rows_fp8(x, out=bad)
    F.quantize_rows_fp8(x, out=F.Fp8Rows(beside, scales))


def test_versions_of_written_tensors(cuda_device):
    """A graph that saved a tensor which a call writes into refuses to go backward with the changed values."""
    x = torch.randn(4, 256, device=cuda_device)
    leaf = torch.randn(4, 256, device=cuda_device, requires_grad=True)
    stream = leaf * 2
    loss = (stream * stream).sum()  # saves the stream
    with torch.no_grad():
        norm.rms_norm(x, residual=stream, residual_out=stream)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    for quantise in (F.quantize_rows_fp8, F.quantize_weight_fp8, I.quantize_rows_int8):
        out = quantise(x)
        before = [t._version for t in out]
        quantise(x, out=out)
        assert all(t._version > v for t, v in zip(out, before))
    with torch.inference_mode():  # (tensors without a version)
        stream = torch.randn(4, 256, device=cuda_device)
        norm.rms_norm(x, residual=stream, residual_out=stream)
        F.quantize_rows_fp8(x, out=F.quantize_rows_fp8(x))
    with pytest.raises(ValueError, match="gradient"):
        norm.rms_norm(x, residual=x, residual_out=leaf * 2)


def test_forward_mode_gradients_are_refused(cuda_device):
    x = torch.randn(2, 64, device=cuda_device)
    ids = torch.zeros(2, dtype=torch.int64, device=cuda_device)
    offsets = torch.tensor([0, 30, 64], device=cuda_device)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: norm.rms_norm(dual), lambda: norm.rms_norm(x, dual[0]), lambda: norm.rms_norm(x, residual=dual),
                     lambda: L.token_logprobs(dual, ids), lambda: L.compact_token_logprobs(torch.arange(64, device=cuda_device), dual[0], offsets, ids),
                     lambda: L.token_logprobs(x, ids, temperature=dual[0, :2])):
            with pytest.raises(ValueError, match="gradient"):
                call()
        norm.rms_norm(x)  # (no dual among its tensors)
        L.token_logprobs(x, ids)
