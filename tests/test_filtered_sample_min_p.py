"""A min_p above 1 counts as 1: the largest logit and its ties are kept. On the
oracle by hand, and the kernels (clusters, counted rows, packed rows) against it."""
import numpy as np
import pytest
import torch

from gsp import triton_runtime as tr
from oracle import gsp_oracle as O

ABOVE = (1.0, 1.0000001, 2.0, float("inf"))


@pytest.mark.parametrize("min_p", ABOVE)
def test_oracle(min_p):
    row = [1.0, 3.0, -np.inf, 3.0, 2.0]
    assert O.filtered_sample_reference(row, 0.2, min_p=min_p) == (1, -np.log(2.0), 2)
    assert O.filtered_sample_reference(row, 0.7, min_p=min_p) == (3, -np.log(2.0), 2)
    assert O.filtered_sample_reference(row, 0.7, min_p=min_p, top_k=1) == (1, 0.0, 1)
    assert O.filtered_sample_reference([-np.inf], 0.7, min_p=min_p) == (0, -np.inf, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 5000), (200, 9001)])  # (16-bit: 200 rows are counted, unless a scalar min_p says few)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_kernels(cuda_device, dtype, shape):
    """Log-probabilities are -log of a count: one rounding to fp32."""
    batch, vocab = shape
    g = torch.Generator(device=cuda_device).manual_seed(vocab)
    x = torch.randn(batch, vocab, generator=g, device=cuda_device).to(dtype)
    top = x.float().amax(1)
    for ties in (1, 3):  # the largest again at places before and behind
        x[:, 7 * ties] = x.amax(1)
    u = torch.rand(batch, generator=g, device=cuda_device)
    ids = torch.arange(vocab, device=cuda_device).repeat(batch)
    offsets = torch.arange(batch + 1, device=cuda_device) * vocab
    rows = x.float().cpu().numpy()
    for top_k in (0, 2):
        want = [O.filtered_sample_reference(rows[b], u[b].item(), min_p=2.0, top_k=top_k) for b in range(batch)]
        for min_p in ABOVE:
            for p in (min_p, torch.full((batch,), min_p, device=cuda_device)):
                for r in (tr.sample_logits(x, uniforms=u, min_p=p, top_k=top_k),
                          tr.sample_compact_logits(ids, x.reshape(-1), offsets, uniforms=u, min_p=p, top_k=top_k)):
                    assert r.token_ids.tolist() == [w[0] for w in want] and r.kept.tolist() == [w[2] for w in want]
                    for got, w in zip(r.logprobs.tolist(), want):
                        assert abs(got - w[1]) <= abs(w[1]) * 2.0 ** -24 + 1e-11
    assert torch.equal(top, x.float().amax(1))
