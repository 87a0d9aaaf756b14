"""GPU tests of token_logprobs / compact_token_logprobs and their gradient
against a 64-bit restatement.

Tolerances, in units of 2^-24 (half a step of fp32). S, a sum of up to V / 512
terms per thread and then a tree of at most 20, of terms whose exponent carries
two roundings of at most 60 (smaller terms weigh nothing) and whose power is good
to 2 steps: e(V) = V / 512 + 20 + 60 + 20, rounded up to V / 512 + 128. ln S is
then off by e(V), a log probability by that and four roundings of itself. The
entropy ln S - A / S: A's terms carry one rounding more, and |A / S| <= ln S + 1.
A gradient's probability is off by e(V) for S and the same 128 for its exponent;
its factor by four roundings; then half a step of the output's type (and of its
smallest number). Ids are equal.
"""
import math

import numpy as np
import pytest
import torch

from gsp import logprobs as L
from gsp import triton_runtime as tr

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
SHAPES = [(1, 1), (2, 2), (3, 7), (5, 33), (1, 1000), (4, 4097), (2, 50257), (1, 248320), (150, 3001), (61, 70001)]
STEP = 2.0 ** -24


def _error(vocab):
    return STEP * (vocab / 512 + 128)


def _logits(seed, batch, vocab, dtype, density=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(batch, vocab, generator=g) * 2.2
    x[torch.arange(batch), torch.randint(0, vocab, (batch,), generator=g)] += 6.0
    if density < 1.0:
        x.masked_fill_(torch.rand(batch, vocab, generator=g) >= density, -math.inf)
    return x.to(dtype)


def _pack(legal):
    batch, vocab = legal.shape
    words = (vocab + 31) // 32
    bits = np.zeros((batch, words * 32), dtype=np.uint8)
    bits[:, :vocab] = legal.numpy()
    return torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32).copy())


def _reference(x, ids, temperature, top_n, legal=None):
    """(logprobs [B, K], entropy, logsumexp, top ids, top logprobs, p) in 64 bits; x [B, V] on the CPU."""
    x = x.double()
    x = torch.where(x.isnan(), -math.inf, x)
    if legal is not None:
        x = x.masked_fill(~legal, -math.inf)
    batch, vocab = x.shape
    t = temperature.double().unsqueeze(1) if isinstance(temperature, torch.Tensor) else float(np.float32(temperature))
    m = x.amax(1, keepdim=True)
    z = torch.where(x == m, 0.0, (x - m) / t)
    z = torch.where(x > -math.inf, z, -math.inf)
    w = z.exp()
    total = w.sum(1, keepdim=True)
    some = total > 0
    lp = torch.where(some, z - total.log(), -math.inf)
    p = torch.where(some, w / total, 0.0)
    entropy = -torch.special.xlogy(p, p).sum(1)
    lse = torch.where(some, m / t + total.log(), -math.inf).squeeze(1)
    ids2 = ids.view(batch, -1)
    given = lp.gather(1, ids2.clamp(0, vocab - 1))
    given = torch.where(ids2 < 0, 0.0, torch.where(ids2 >= vocab, -math.inf, given))
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top_n]
    top = lp.gather(1, order)
    order = torch.where(x.gather(1, order) > -math.inf, order, -1)
    short = top_n - order.shape[1]
    return (given.view(ids.shape), entropy, lse, torch.nn.functional.pad(order, (0, short), value=-1),
            torch.nn.functional.pad(top, (0, short), value=-math.inf), p)


def _near(got, want, tol, what):
    got = got.detach().double().cpu()
    # outputs are fp32: what lies past its largest number, (1 - 2^-25) 2^128, rounds to infinity
    # (the lowest bf16 less the highest is -1.992 * 2^128)
    want = torch.where(want.abs() >= (1 - 2.0 ** -25) * 2.0 ** 128, want * math.inf, want)
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine], want[~fine]), what
    off = (got - want).abs()[fine]
    bound = (tol if isinstance(tol, torch.Tensor) else torch.full_like(want, tol))[fine]
    assert (off <= bound).all(), (what, (off / bound).max().item())


def _check(r, x, ids, temperature, top_n, legal=None):
    vocab = x.shape[1]
    lp, entropy, lse, top_ids, top_lp, _ = _reference(x, ids, temperature, top_n, legal)
    e = _error(vocab)
    assert r.logprobs.shape == ids.shape and r.top_ids.shape == (x.shape[0], top_n)
    _near(r.logprobs, lp, e + 4 * STEP * lp.abs(), "logprobs")
    ln_s = math.log(vocab) + 1
    _near(r.entropy, entropy, 2 * e * (1 + ln_s), "entropy")
    _near(r.logsumexp, lse, e + 4 * STEP * (lse.abs() + ln_s), "logsumexp")
    assert torch.equal(r.top_ids.cpu(), top_ids)
    _near(r.top_logprobs, top_lp, e + 4 * STEP * top_lp.abs(), "top_logprobs")


def _some_ids(seed, batch, vocab, k=None):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, vocab, (batch,) if k is None else (batch, k), generator=g)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_64_bits(cuda_device, shape, dtype):
    batch, vocab = shape
    for density, top_n, temperature in ((1.0, 0, 1.0), (1.0, 20, 0.7), (0.3, 64, 1.3), (0.002, 5, 1.0)):
        x = _logits(batch + vocab, batch, vocab, dtype, density)
        ids = _some_ids(vocab, batch, vocab)
        r = L.token_logprobs(x.to(cuda_device), ids.to(cuda_device), temperature=temperature, top_n=top_n)
        _check(r, x, ids, temperature, top_n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(3, 7), (5, 33), (4, 4097), (2, 50257), (61, 70001)])
def test_bitmask_and_several_tokens(cuda_device, shape, dtype):
    batch, vocab = shape
    x = _logits(7, batch, vocab, dtype)
    legal = torch.rand(batch, vocab, generator=torch.Generator().manual_seed(3)) < 0.4
    legal[0] = False                     # nothing legal
    legal[1] = False
    legal[1, vocab - 1] = True           # one token
    ids = _some_ids(5, batch, vocab, 6)
    ids[:, 1] = ids[:, 0]                # twice the same
    ids[:, 2], ids[:, 3] = -100, vocab   # none, and past the end
    temperature = torch.linspace(0.5, 2.0, batch)
    mask = torch.cat([_pack(legal), torch.full((batch, 2), -1, dtype=torch.int32)], 1)  # wider than needed
    r = L.token_logprobs(x.to(cuda_device), ids.to(cuda_device), bitmask_gpu=mask.to(cuda_device),
                         temperature=temperature.to(cuda_device), top_n=3)
    _check(r, x, ids, temperature, 3, legal)
    assert r.top_ids[0].tolist() == [-1] * 3 and r.entropy[:2].tolist() == [0.0, 0.0]


@pytest.mark.parametrize("dtype", DTYPES)
def test_extreme_rows(cuda_device, dtype):
    vocab = 20011
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    rows = {
        "zeros": torch.zeros(vocab),
        "signed zeros": torch.where(torch.arange(vocab) % 2 == 0, -0.0, 0.0),
        "lowest": torch.full((vocab,), low),
        "lowest but one": torch.full((vocab,), low).index_fill_(0, torch.tensor([vocab - 2]), 1.0),
        "rising": torch.linspace(-20.0, 20.0, vocab),
        "falling": torch.linspace(20.0, -20.0, vocab),
        "extremes": torch.where(torch.arange(vocab) % 3 == 0, high, low),
        "nan": _logits(1, 1, vocab, torch.float32)[0].index_fill_(0, torch.arange(0, vocab, 5), math.nan),
        "all nan": torch.full((vocab,), math.nan),
        "nothing": torch.full((vocab,), -math.inf),
        "one infinite": _logits(2, 1, vocab, torch.float32)[0].index_fill_(0, torch.tensor([77]), math.inf),
        "infinite ones": _logits(3, 1, vocab, torch.float32)[0].index_fill_(0, torch.arange(0, vocab, 7), math.inf),
        "late largest": _logits(4, 1, vocab, torch.float32)[0].index_fill_(0, torch.tensor([vocab - 1]), 40.0),
    }
    x = torch.stack(list(rows.values())).to(dtype)
    ids = torch.stack([torch.full((len(rows),), i) for i in (0, 77, vocab - 2, vocab - 1)], 1).contiguous()
    for temperature in (1.0, 0.05):
        r = L.token_logprobs(x.to(cuda_device), ids.to(cuda_device), temperature=temperature, top_n=64)
        _check(r, x, ids, temperature, 64)


def test_temperatures_that_are_not_valid(cuda_device):
    x = _logits(1, 5, 300, torch.float32).to(cuda_device)
    t = torch.tensor([1.0, 0.0, -1.0, math.nan, math.inf], device=cuda_device)
    r = L.token_logprobs(x, torch.zeros(5, dtype=torch.int64, device=cuda_device), temperature=t, top_n=2)
    assert r.logprobs.isnan().tolist() == r.entropy.isnan().tolist() == [False] + [True] * 4
    assert r.logsumexp.isnan().tolist() == r.top_logprobs[:, 0].isnan().tolist() == [False] + [True] * 4
    assert (r.top_ids[1:] == -1).all() and (r.top_ids[0] >= 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(cuda_device, dtype):
    batch, vocab = 6, 9001
    wide = _logits(9, batch, vocab + 40, dtype)
    legal = torch.rand(batch, vocab, generator=torch.Generator().manual_seed(4)) < 0.5
    ids = _some_ids(6, batch, vocab)
    dev, mask = wide.to(cuda_device), _pack(legal).to(cuda_device)
    for first in (0, 1, 3, 8, 13):
        x = wide[:, first:first + vocab]
        xd = dev[:, first:first + vocab]
        _check(L.token_logprobs(xd, ids.to(cuda_device), top_n=10), x, ids, 1.0, 10)
        _check(L.token_logprobs(xd, ids.to(cuda_device), bitmask_gpu=mask, top_n=10), x, ids, 1.0, 10, legal)
    shared = wide[2, 5:5 + vocab].expand(batch, vocab)  # one row for all
    _check(L.token_logprobs(dev[2, 5:5 + vocab].expand(batch, vocab), ids.to(cuda_device)), shared, ids, 1.0, 0)
    one = L.token_logprobs(dev[0, 1:1 + vocab], ids[:1].to(cuda_device), top_n=1)
    _check(one, wide[:1, 1:1 + vocab], ids[:1], 1.0, 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch", [300, 700])
def test_many_rows_with_lists_that_overflow(cuda_device, batch, dtype):
    """Rows in rising order and of equal values among ordinary ones, a CTA each (of 512 and of 256 threads)."""
    vocab = 16411
    x = _logits(61, batch, vocab, dtype)
    x[5] = torch.linspace(-30, 30, vocab).to(dtype)
    x[7] = 1.5
    x[9, ::2] = -math.inf
    ids = _some_ids(3, batch, vocab, 2)
    for top_n in (0, 64):
        r = L.token_logprobs(x.to(cuda_device), ids.to(cuda_device), temperature=0.9, top_n=top_n)
        _check(r, x, ids, 0.9, top_n)


def test_no_given_tokens(cuda_device):
    x = _logits(3, 4, 5000, torch.bfloat16)
    ids = torch.empty(4, 0, dtype=torch.int64)
    _check(L.token_logprobs(x.to(cuda_device), ids.to(cuda_device), top_n=2), x, ids, 1.0, 2)


@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_rows(cuda_device, dtype):
    batch, vocab = 9, 30011
    x = _logits(11, batch, vocab, dtype)
    legal = torch.rand(batch, vocab, generator=torch.Generator().manual_seed(8)) < 0.1
    legal[3] = False
    legal[4] = True
    ids = _some_ids(2, batch, vocab, 4)
    ids[:, 0] = torch.where(legal.any(1), legal.to(torch.int8).argmax(1), 0)
    ids[0, 3], ids[1, 3] = -1, vocab + 5
    at, counts = legal.nonzero(), legal.sum(1)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    args = [t.to(cuda_device) for t in (at[:, 1].contiguous(), x[legal], offsets, ids)]
    for max_len in (None, 0, vocab):
        r = L.compact_token_logprobs(*args, temperature=0.8, top_n=7, max_len=max_len)
        _check(r, x, ids, 0.8, 7, legal)
    # offsets past the end of the arrays, and falling ones, read nothing there
    bad = offsets.clone()
    bad[-1], bad[2] = 10 ** 12, offsets[-1] + 5
    r = L.compact_token_logprobs(args[0], args[1], bad.to(cuda_device), args[3], top_n=2)
    assert r.logprobs.shape == ids.shape and (r.logprobs[2] == -math.inf).all()


def _grad_bound(p, ids, g, gh, gl, t, want, dtype, entropy):
    lnp = torch.where(p > 0, p.log(), 0.0).abs()
    size = p * (gl.abs().unsqueeze(1) + g.abs().sum(1, keepdim=True) + gh.abs().unsqueeze(1) * (lnp + entropy.unsqueeze(1) + 1))
    own = torch.zeros_like(p).scatter_add_(1, ids.clamp(0, p.shape[1] - 1), g.abs())
    e = 2 * _error(p.shape[1])
    return (size * e * 2 + own * 8 * STEP) / t + want.abs() * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).tiny * torch.finfo(dtype).eps


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (2, 7), (3, 1000), (5, 8193), (2, 50257)])
def test_gradient_formula(cuda_device, shape, dtype):
    batch, vocab = shape
    x = _logits(21, batch, vocab, dtype)
    legal = torch.rand(batch, vocab, generator=torch.Generator().manual_seed(5)) < 0.6
    if batch > 1:
        legal[0] = False
    ids = _some_ids(3, batch, vocab, 4)
    ids[:, 1] = ids[:, 0]
    if batch > 1:
        ids[1, 2] = -1
    g = torch.Generator().manual_seed(6)
    gp, gh, gl = torch.randn(batch, 4, generator=g), torch.randn(batch, generator=g), torch.randn(batch, generator=g)
    temperature = torch.linspace(0.6, 1.7, batch)
    xd = x.to(cuda_device).requires_grad_(True)
    r = L.token_logprobs(xd, ids.to(cuda_device), bitmask_gpu=_pack(legal).to(cuda_device),
                         temperature=temperature.to(cuda_device), top_n=2)
    assert not r.top_logprobs.requires_grad and r.logprobs.requires_grad
    (grad,) = torch.autograd.grad((r.logprobs, r.entropy, r.logsumexp), xd, [t.to(cuda_device) for t in (gp, gh, gl)])
    assert grad.dtype == dtype and grad.shape == x.shape
    _, entropy, _, _, _, p = _reference(x, ids, temperature, 0, legal)
    given = torch.where(ids >= 0, gp, torch.zeros_like(gp)).double()
    t = temperature.double().unsqueeze(1)
    lnp = torch.where(p > 0, p.log(), 0.0)
    want = p * (gl.double().unsqueeze(1) - given.sum(1, keepdim=True) - gh.double().unsqueeze(1) * (lnp + entropy.unsqueeze(1)))
    want.scatter_add_(1, ids.clamp(min=0), given)
    want = torch.where(legal, want, 0.0) / t
    if batch > 1:
        want[0] = 0.0
    _near(grad, want, _grad_bound(p, ids, given, gh.double(), gl.double(), t, want, dtype, entropy), "gradient")
    again = torch.autograd.grad(L.token_logprobs(xd, ids.to(cuda_device), bitmask_gpu=_pack(legal).to(cuda_device),
                                                 temperature=temperature.to(cuda_device)).logprobs.sum(), xd)[0]
    assert torch.isfinite(again).all()


def test_gradient_against_differences(cuda_device):
    vocab, h = 301, 2.0 ** -6
    x = _logits(2, 1, vocab, torch.float32)
    ids = torch.tensor([[5, 17]])
    xd = x.to(cuda_device).requires_grad_(True)

    def loss64(y):  # the 64-bit restatement: its differences, and the kernel's gradient
        lp, entropy, lse, _, _, _ = _reference(y, ids, 0.9, 0)
        return (lp.sum() + 0.3 * entropy.sum() - 0.2 * lse.sum()).item()

    r = L.token_logprobs(xd, ids.to(cuda_device), temperature=0.9)
    (r.logprobs.sum() + 0.3 * r.entropy.sum() - 0.2 * r.logsumexp.sum()).backward()
    for j in list(range(0, vocab, 23)) + [5, 17, int(x.argmax())]:
        up, down = x.double(), x.double()
        up, down = up.clone(), down.clone()
        up[0, j] += h
        down[0, j] -= h
        slope = (loss64(up) - loss64(down)) / (2 * h)
        # third derivatives are at most a few units: h^2 of them, and the gradient's own bound
        assert abs(slope - xd.grad[0, j].item()) <= 4 * h * h + 1e-4


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_strides_infinities_and_broadcast(cuda_device, dtype):
    batch, vocab = 4, 5003
    wide = _logits(31, batch, vocab + 9, dtype)
    wide[1, 40], wide[1, 50] = math.inf, math.inf
    wide[2, 60:90] = math.nan
    wide[3] = -math.inf
    ids = _some_ids(1, batch, vocab)
    ids[1] = 40 - 3
    leaf = wide.to(cuda_device).requires_grad_(True)
    r = L.token_logprobs(leaf[:, 3:3 + vocab], ids.to(cuda_device))
    r.logprobs[:3].sum().backward()
    inner = wide[:, 3:3 + vocab]
    p = _reference(inner, ids, 1.0, 0)[-1]
    want = torch.zeros_like(wide, dtype=torch.float64)
    want[:3, 3:3 + vocab] = -p[:3]
    for b in range(3):
        if inner[b, ids[b]] > -math.inf:
            want[b, 3 + ids[b]] += 1.0
    got = leaf.grad.double().cpu()
    assert (got - want).abs().max() <= torch.finfo(dtype).eps / 2 + 2 * _error(vocab)
    # one row shared by all: its gradient is the sum (torch adds the rows in the rows' type)
    row = wide[0, :vocab].to(cuda_device).requires_grad_(True)
    L.token_logprobs(row.expand(batch, vocab), ids.to(cuda_device)).logprobs.sum().backward()
    p = _reference(wide[:1, :vocab], ids[:1], 1.0, 0)[-1][0]
    want = -batch * p
    want.index_add_(0, ids, torch.ones(batch, dtype=torch.float64))
    assert (row.grad.double().cpu() - want).abs().max() <= batch * 4 * (torch.finfo(dtype).eps / 2 + 2 * _error(vocab))


def test_repeated_streams_and_captured(cuda_device):
    batch, vocab = 7, 40009
    x = _logits(41, batch, vocab, torch.bfloat16).to(cuda_device)
    ids = _some_ids(4, batch, vocab).to(cuda_device)
    first = L.token_logprobs(x, ids, top_n=20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = L.token_logprobs(x, ids, top_n=20)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    buffer = x.clone().requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):  # forward and backward
        r = L.token_logprobs(buffer, ids, top_n=20)
        (grad,) = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), buffer)
    for seed in (42, 43):
        new = _logits(seed, batch, vocab, torch.bfloat16).to(cuda_device)
        with torch.no_grad():
            buffer.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        eager = new.clone().requires_grad_(True)
        want = L.token_logprobs(eager, ids, top_n=20)
        assert all(torch.equal(a, b) for a, b in zip(r, want))
        assert torch.equal(grad, torch.autograd.grad(want.logprobs.sum() + want.entropy.sum(), eager)[0])


def test_agrees_with_the_samplers_log_probability(cuda_device):
    """Drawn without a filter, a token's log-probability is the sampler's (exact sums there, fp32 here)."""
    batch, vocab = 16, 50257
    x = _logits(51, batch, vocab, torch.float16).to(cuda_device)
    drawn = tr.sample_logits(x, uniforms=torch.rand(batch, device=cuda_device), temperature=0.8)
    r = L.token_logprobs(x, drawn.token_ids, temperature=0.8)
    bound = _error(vocab) + 5 * STEP * drawn.logprobs.abs()
    assert ((r.logprobs - drawn.logprobs).abs() <= bound).all()


def test_refusals(cuda_device):
    x = torch.zeros(2, 64, device=cuda_device)
    ids = torch.zeros(2, dtype=torch.int64, device=cuda_device)
    for kw, word in ((dict(temperature=0.0), "temperature"), (dict(temperature=math.nan), "temperature"),
                     (dict(temperature=torch.ones(3, device=cuda_device)), "temperature"), (dict(top_n=65), "top_n"),
                     (dict(top_n=-1), "top_n"), (dict(bitmask_gpu=torch.zeros(2, 1, dtype=torch.int32, device=cuda_device)), "bitmask"),
                     (dict(temperature=torch.ones(2, device=cuda_device, requires_grad=True)), "gradient")):
        with pytest.raises(ValueError, match=word):
            L.token_logprobs(x, ids, **kw)
    for bad in (ids.cpu(), ids.int(), ids[:1], torch.zeros(2, 2048, dtype=torch.int64, device=cuda_device)[:, ::2],
                torch.zeros(2, 1025, dtype=torch.int64, device=cuda_device)):
        with pytest.raises(ValueError, match="token_ids"):
            L.token_logprobs(x, bad)
    with pytest.raises(ValueError, match="contiguous"):
        L.token_logprobs(torch.zeros(64, 2, device=cuda_device).T, ids)
    with pytest.raises(ValueError, match="gradient"):
        L.compact_token_logprobs(ids, torch.zeros(2, device=cuda_device, requires_grad=True), torch.tensor([0, 1, 2], device=cuda_device), ids)
