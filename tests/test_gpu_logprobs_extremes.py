"""GPU tests of the log probabilities and their gradient on rows with the largest and lowest values of their type, at
temperatures down to 1e-37, against the 64-bit restatement of test_gpu_logprobs (and within its bounds).

Beyond those bounds a gradient's weight 2^d below 2^-126 is taken as 0, so a probability may be off by 2^-126 more;
what rounds past the largest number of the output's type is infinite.
"""
import math

import pytest
import torch

from gsp import logprobs as L
from test_gpu_logprobs import DTYPES, STEP, _check, _error, _logits, _pack, _reference

pytestmark = pytest.mark.gpu

VOCAB = 20011


def _rows(dtype):
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    every = torch.arange(VOCAB)
    bell = lambda seed: _logits(seed, 1, VOCAB, torch.float32)[0]  # noqa: E731
    rows = [
        torch.where(every % 3 == 0, high, low),                           # extremes, side by side
        bell(1).index_fill_(0, torch.tensor([77]), high),                 # a forced token among ordinary logits
        bell(2).index_fill_(0, torch.tensor([5, 77, VOCAB - 1]), high),   # several
        torch.full((VOCAB,), low).index_fill_(0, torch.tensor([VOCAB - 2]), 1.0),
        torch.full((VOCAB,), low),
        torch.full((VOCAB,), high),
        bell(3).index_fill_(0, torch.tensor([77]), high / 4).index_fill_(0, every[::5], math.nan),
        bell(4).index_fill_(0, every[::2], -math.inf).index_fill_(0, torch.tensor([4001]), high / 64),
        torch.where(every % 7 == 0, 0.0, -0.0),
        torch.full((VOCAB,), -math.inf),
        bell(5).index_fill_(0, torch.tensor([77, 78]), math.inf),
        torch.linspace(-40.0, 40.0, VOCAB),
    ]
    return torch.stack(rows).to(dtype)


def _ids(batch):
    return torch.stack([torch.full((batch,), i) for i in (0, 77, VOCAB - 2, VOCAB - 1)], 1).contiguous()


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 0.05, 1e-3, 1e-6, 1e-37])
@pytest.mark.parametrize("dtype", DTYPES)
def test_forward(cuda_device, dtype, temperature, masked):
    x = _rows(dtype)
    ids = _ids(len(x))
    legal = torch.rand(x.shape, generator=torch.Generator().manual_seed(9)) < 0.6 if masked else None
    mask = _pack(legal).to(cuda_device) if masked else None
    r = L.token_logprobs(x.to(cuda_device), ids.to(cuda_device), bitmask_gpu=mask, temperature=temperature, top_n=5)
    _check(r, x, ids, temperature, 5, legal)


@pytest.mark.parametrize("temperature", [1.5, 5.0, 1e3, 1e30])
@pytest.mark.parametrize("dtype", DTYPES)
def test_lowest_beside_largest_values_at_high_temperatures(cuda_device, dtype, temperature):
    """A difference that passes fp32 before it is divided, and not afterwards."""
    x = _rows(dtype)
    ids = _ids(len(x))
    ids[:, 1] = 1  # (the lowest value of the first row)
    r = L.token_logprobs(x.to(cuda_device), ids.to(cuda_device), temperature=temperature, top_n=5)
    _check(r, x, ids, temperature, 5)


def test_entropy_of_tied_largest_values(cuda_device):
    """ln of their number, however large they are and however low the temperature."""
    for dtype in DTYPES:
        x = _rows(dtype)[[0, 2, 5]]
        ids = torch.zeros(3, dtype=torch.int64, device=cuda_device)
        for temperature in (0.005, 1e-6, 1e-37):
            r = L.token_logprobs(x.to(cuda_device), ids, temperature=temperature)
            want = torch.tensor([(VOCAB + 2) // 3, 3, VOCAB], dtype=torch.float64).log()
            assert (r.entropy.double().cpu() - want).abs().max() <= 2 * _error(VOCAB) * (1 + math.log(VOCAB) + 1)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 0.05, 0.005, 1e-3, 1e-6, 1e-37])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient(cuda_device, dtype, temperature, masked):
    x = _rows(dtype)
    batch = len(x)
    ids = _ids(batch)
    legal = torch.ones(x.shape, dtype=torch.bool)
    mask = None
    if masked:
        legal = torch.rand(x.shape, generator=torch.Generator().manual_seed(9)) < 0.6
        mask = _pack(legal).to(cuda_device)
    g = torch.Generator().manual_seed(6)
    gp, gh, gl = torch.randn(batch, 4, generator=g), torch.ones(batch), torch.randn(batch, generator=g)
    _, entropy, _, _, _, p = _reference(x, ids, temperature, 0, legal)
    own = torch.zeros_like(p).scatter_add_(1, ids, gp.double())
    absolute = torch.zeros_like(p).scatter_add_(1, ids, gp.double().abs())
    lnp = torch.where(p > 0, p.log(), 0.0)
    there = legal & (x > -math.inf)  # (NaN is not)
    info, t = torch.finfo(dtype), float(torch.tensor(temperature, dtype=torch.float32))
    for gh_, gl_ in ((gh.double(), gl.double()), (torch.zeros(batch).double(), torch.zeros(batch).double())):
        leaf = x.to(cuda_device).requires_grad_(True)
        r = L.token_logprobs(leaf, ids.to(cuda_device), bitmask_gpu=mask, temperature=temperature)
        if gh_.any():
            (grad,) = torch.autograd.grad((r.logprobs, r.entropy, r.logsumexp), leaf,
                                          [v.to(cuda_device) for v in (gp, gh, gl)])
        else:  # (the log probabilities' alone)
            (grad,) = torch.autograd.grad(r.logprobs, leaf, gp.to(cuda_device))
        got = grad.double().cpu()
        want = p * (gl_.unsqueeze(1) - gp.double().sum(1, keepdim=True) - gh_.unsqueeze(1) * (lnp + entropy.unsqueeze(1))) + own
        want = torch.where(there, want, 0.0) / t
        size = (p + 2.0 ** -126) * (gl_.abs().unsqueeze(1) + gp.double().abs().sum(1, keepdim=True)
                                    + gh_.unsqueeze(1) * (lnp.abs() + entropy.unsqueeze(1) + 1))
        flushed = 2.0 ** -126 * (size / (p + 2.0 ** -126))
        bound = (size * 4 * _error(VOCAB) + flushed + absolute * 8 * STEP) / t + want.abs() * info.eps / 2 + info.tiny * info.eps
        assert not got.isnan().any()
        assert (got[~there] == 0).all()
        past = want.abs() + bound >= info.max  # may have rounded to infinity
        assert ((got - want).abs() <= bound)[~past].all(), ((got - want).abs() / bound)[~past].max()
        assert (got * want.sign() >= info.max * (1 - 2 * info.eps))[want.abs() - bound >= info.max].all()


def test_gradient_of_rows_whose_temperature_is_not_valid(cuda_device):
    """NaN like what they report, and 0 on illegal tokens."""
    x = _logits(1, 5, 300, torch.float32)
    legal = torch.rand(5, 300, generator=torch.Generator().manual_seed(2)) < 0.5
    legal[:, 0] = True
    t = torch.tensor([1.0, 0.0, -1.0, math.nan, math.inf], device=cuda_device)
    for dtype in DTYPES:
        leaf = x.to(dtype).to(cuda_device).requires_grad_(True)
        r = L.token_logprobs(leaf, torch.zeros(5, dtype=torch.int64, device=cuda_device), temperature=t,
                             bitmask_gpu=_pack(legal).to(cuda_device))
        for loss in (r.logprobs.sum(), r.entropy.sum()):
            (grad,) = torch.autograd.grad(loss, leaf, retain_graph=True)
            grad = grad.cpu()
            assert torch.isfinite(grad[0]).all() and (grad[~legal] == 0).all()
            assert grad[1:][legal[1:]].isnan().all()
