"""GPU tests of the filtered sampler on long flat rows, whose border and draw
bins hold more tokens than a cluster lists, so that the search goes on in the
whole row; against the oracle's float64 sort and running sums.

Tokens and counts are equal: the weights are integers in units of 2^-43 of the
largest (2^18 tokens), together at most 2^18 * 2^-44 = 2^-26 off a sum of at
least 256 (the rows here), 6e-11 relative, and a token differs only where its
border lies that near a target: of 2^18 borders, 3e-5 a row at the very worst,
and the inputs are fixed. Log-probabilities: one rounding to fp32, the same
6e-11, 3e-11 for the oracle's running sum (2^18 * 2^-53) and 2e-13 for the
exponential's polynomial."""
import pytest
import torch

from gsp import triton_runtime as tr
from oracle import gsp_oracle as O

pytestmark = pytest.mark.gpu

SETTINGS = [dict(), dict(top_p=0.9), dict(top_p=0.999, temperature=1.5), dict(top_k=30000, top_p=0.8),
            dict(min_p=0.05, top_p=0.95)]


@pytest.mark.parametrize("spread", [1.0, 0.05])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("batch", [2, 7])
def test_long_flat_rows(cuda_device, batch, dtype, spread):
    vocab = 262144
    g = torch.Generator(device=cuda_device).manual_seed(batch)
    x = (torch.randn(batch, vocab, generator=g, device=cuda_device) * spread).to(dtype)
    u = torch.rand(batch, generator=g, device=cuda_device)
    rows = x.float().cpu().numpy()
    for settings in SETTINGS:
        got = tr.sample_logits(x, uniforms=u, **settings)
        again = tr.sample_logits(x, uniforms=u, **settings)
        assert all(torch.equal(a, b) for a, b in zip(got, again))
        for b in range(batch):
            token, logprob, kept = O.filtered_sample_reference(rows[b], u[b].item(), **settings)
            assert (got.token_ids[b].item(), got.kept[b].item()) == (token, kept)
            assert abs(got.logprobs[b].item() - logprob) <= abs(logprob) * 2.0 ** -24 + 1e-10
