"""GPU tests of sample_logits / sample_compact_logits against the oracle's
float64 restatement (sort, cumulative sums).

Tokens and counts are equal: the kernel's sums are exact integers of weights
rounded to 2^-44 or finer, so a token could differ only where a border lies
within about 1e-11 of the target; the inputs here are fixed and hold none.
Log-probabilities: one rounding to fp32, |want| * 2^-24, and 1e-11 for the
weights' rounding and the two logarithms.
"""
import numpy as np
import pytest
import torch

from gsp import _native
from gsp import triton_runtime as tr
from oracle import gsp_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
SETTINGS = [
    dict(),
    dict(temperature=0.7),
    dict(top_k=1),
    dict(top_k=20),
    dict(top_k=500, temperature=1.3),
    dict(top_p=0.9),
    dict(top_p=0.5, temperature=0.6),
    dict(top_p=0.0),
    dict(min_p=0.05),
    dict(min_p=1.0),
    dict(top_k=40, top_p=0.95, min_p=0.02, temperature=0.8),
    dict(top_k=3, top_p=0.99, min_p=0.5, temperature=2.0),
    dict(temperature=0.0, top_k=5),
    dict(temperature=0.02, top_p=0.95),
    dict(temperature=50.0, top_p=0.75),
    dict(top_k=10 ** 6, top_p=2.0, min_p=-1.0),
]


def _logits(seed, batch, vocab, dtype, dev, density=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    x = torch.randn(batch, vocab, generator=g) * 2.2
    x[torch.arange(batch), torch.randint(0, vocab, (batch,), generator=g)] += 6.0
    if density < 1.0:
        x.masked_fill_(torch.rand(batch, vocab, generator=g) >= density, float("-inf"))
    return x.to(dtype).to(dev)


def _uniforms(seed, batch, dev):
    return torch.rand(batch, generator=torch.Generator(device="cpu").manual_seed(seed)).to(dev)


def _at(settings, b):
    return {k: (v[b].item() if isinstance(v, torch.Tensor) else v) for k, v in settings.items()}


def _check(got, rows, uniforms, settings, ids=None):
    assert got.token_ids.dtype == torch.int64 and got.logprobs.dtype == torch.float32 and got.kept.dtype == torch.int32
    for b, row in enumerate(rows):
        at, logprob, kept = O.filtered_sample_reference(row.double().cpu().numpy(), uniforms[b].item(),
                                                        **_at(settings, b))
        token = at if ids is None else (int(ids[b][at]) if kept else 0)
        where = (b, settings, got.token_ids[b].item(), token, got.kept[b].item(), kept)
        assert got.kept[b].item() == kept, where
        assert got.token_ids[b].item() == token, where
        value = got.logprobs[b].item()
        if kept == 0:
            assert value == -np.inf
        else:
            assert abs(value - logprob) <= abs(logprob) * 2.0 ** -24 + 1e-11, (where, value, logprob)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (2, 2), (3, 7), (5, 33), (1, 1000), (4, 4097), (2, 50257), (1, 248320),
                                   (150, 3001), (61, 70001)])
def test_matches_oracle(cuda_device, shape, dtype):
    batch, vocab = shape
    x = _logits(batch + vocab, batch, vocab, dtype, cuda_device)
    for i, settings in enumerate(SETTINGS):
        u = _uniforms(i, batch, cuda_device)
        _check(tr.sample_logits(x, uniforms=u, **settings), x, u, settings)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(6, 20011), (3, 140001), (60, 140001)])
@pytest.mark.parametrize("form", ["equal", "two", "coarse"])
def test_ties_go_to_the_lowest_id(cuda_device, form, shape, dtype):
    """Every logit equal, two values, a few values: borders fall inside ties.
    (Over 65,535 tokens of one value, in few rows and in many.)"""
    batch, vocab = shape
    g = torch.Generator(device="cpu").manual_seed(3)
    if form == "equal":
        x = torch.full((batch, vocab), -1.5)
    elif form == "two":
        x = torch.where(torch.rand(batch, vocab, generator=g) < 0.3, 0.5, 0.25)
    else:
        x = (torch.randn(batch, vocab, generator=g) * 2).round() / 2
    x = x.to(dtype).to(cuda_device)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 0.5, 0.25, 0.123, 0.987] * 10, device=cuda_device)[:batch].contiguous()
    for settings in SETTINGS + [dict(top_k=7001, top_p=0.3), dict(top_k=100, min_p=1.0), dict(top_k=9000, min_p=0.9)]:
        _check(tr.sample_logits(x, uniforms=u, **settings), x, u, settings)


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_nan_and_empty_rows(cuda_device, dtype):
    dev = cuda_device
    vocab = 3000
    x = _logits(1, 8, vocab, dtype, dev)
    inf, nan = float("inf"), float("nan")
    x[0] = -inf
    x[1] = nan
    x[2, ::3] = nan
    x[3, 5], x[3, 700] = inf, inf            # only these have weight
    x[4] = -inf
    x[4, 2999] = torch.finfo(dtype).min      # one legal token, the lowest value
    x[5, :] = torch.finfo(dtype).max
    x[6, 1:] = torch.finfo(dtype).min
    x[7, ::2] = -0.0
    x[7, 1::2] = 0.0
    u = _uniforms(9, 8, dev)
    for settings in SETTINGS:
        got = tr.sample_logits(x, uniforms=u, **settings)
        for b in (0, 1, 2, 4, 5, 6, 7):
            _check(tr.FilteredSample(*(t[b:b + 1] for t in got)), x[b:b + 1], u[b:b + 1], settings)
        assert got.token_ids[3].item() in (5, 700)
    # values in masked places do not matter
    legal = torch.rand(8, vocab, generator=torch.Generator().manual_seed(2)) < 0.1
    mask = torch.from_numpy(O.pack_bitmask(legal.numpy())).to(dev)
    y = _logits(4, 8, vocab, dtype, dev)
    z = y.clone()
    z[~legal.to(dev)] = nan
    z[0][~legal[0].to(dev)] = inf
    want = y.masked_fill(~legal.to(dev), -inf)
    for settings in SETTINGS:
        got = tr.sample_logits(z, uniforms=u, bitmask_gpu=mask, **settings)
        _check(got, want, u, settings)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("density", [0.0005, 0.03, 0.9])
def test_mask_masked_logits_and_packed_rows_agree(cuda_device, dtype, density):
    dev = cuda_device
    batch, vocab = 9, 30011
    x = _logits(5, batch, vocab, dtype, dev)
    g = torch.Generator(device="cpu").manual_seed(6)
    legal = torch.rand(batch, vocab, generator=g) < density
    legal[3] = False
    mask_np = O.pack_bitmask(legal.numpy())
    wide = np.full((batch, mask_np.shape[1] + 2), -1, dtype=np.int32)  # set bits past the vocabulary
    wide[:, :mask_np.shape[1]] = mask_np
    wide[:, mask_np.shape[1] - 1] |= np.int32(-1) << np.int32(vocab % 32)
    mask, legal = torch.from_numpy(wide).to(dev), legal.to(dev)
    masked = x.masked_fill(~legal, float("-inf"))
    counts = legal.sum(1)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    ids = legal.nonzero()[:, 1].contiguous()
    packed = x[legal]
    u = _uniforms(7, batch, dev)
    for settings in SETTINGS:
        a = tr.sample_logits(masked, uniforms=u, **settings)
        _check(a, masked, u, settings)
        b = tr.sample_logits(x, uniforms=u, bitmask_gpu=mask, **settings)
        for max_len in (None, int(counts.max()), 1):
            c = tr.sample_compact_logits(ids, packed, offsets, uniforms=u, max_len=max_len, **settings)
            # (packed rows are shorter: their weights have a finer unit)
            assert torch.equal(a.token_ids, c.token_ids) and torch.equal(a.kept, c.kept)
            assert torch.allclose(a.logprobs, c.logprobs, rtol=2.0 ** -23, atol=1e-11)
        assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_rows_longer_than_shared_memory(cuda_device):
    """1,000,003 fp32 logits: part of the row is read from global memory in every pass."""
    x = _logits(8, 2, 1_000_003, torch.float32, cuda_device)
    u = _uniforms(8, 2, cuda_device)
    for settings in SETTINGS[:12]:
        _check(tr.sample_logits(x, uniforms=u, **settings), x, u, settings)
    packed = x.reshape(-1)
    ids = torch.arange(1_000_003, device=cuda_device).repeat(2)
    offsets = torch.tensor([0, 1_000_003, 2_000_006], device=cuda_device)
    a = tr.sample_compact_logits(ids, packed, offsets, uniforms=u, top_p=0.9, max_len=10)  # an expectation far too low
    b = tr.sample_logits(x, uniforms=u, top_p=0.9)
    assert all(torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_alignment_and_one_row(cuda_device, dtype):
    dev = cuda_device
    base = _logits(11, 7, 5003, dtype, dev)
    u = _uniforms(12, 7, dev)
    for view in (base[:, 1:4000], base[:, 3:], base[::1, :17], base[:1].expand(7, 5003), base.flip(0)):
        got = tr.sample_logits(view, uniforms=u, top_p=0.9, top_k=300)
        _check(got, view, u, dict(top_p=0.9, top_k=300))
    one = tr.sample_logits(base[2], uniforms=u[:1], top_k=10)
    assert one.token_ids.shape == (1,)
    _check(one, base[2:3], u[:1], dict(top_k=10))


def test_settings_per_request_and_invalid_ones(cuda_device):
    dev = cuda_device
    batch, vocab = 12, 9001
    x = _logits(13, batch, vocab, torch.bfloat16, dev)
    u = _uniforms(14, batch, dev)
    settings = dict(
        temperature=torch.tensor([0.0, 0.3, 0.7, 1.0, 1.5, 0.0, 0.9, 1.1, 2.0, 0.5, 1.0, 1.0], device=dev),
        top_k=torch.tensor([5, 0, 1, 50, -3, 9, 100, 0, 0, 20, 3, 7], dtype=torch.int32, device=dev),
        top_p=torch.tensor([0.5, 0.9, 1.0, 0.95, 0.1, 0.0, 0.99, 0.8, 1.0, 0.7, -1.0, 3.0], device=dev),
        min_p=torch.tensor([0.0, 0.1, 0.0, 0.02, 0.0, 0.5, 0.0, 1.0, 0.001, 0.0, 0.0, 2.0], device=dev))
    # a min_p above 1 would keep nothing: it counts as 1
    like = dict(settings, min_p=settings["min_p"].clamp(max=1.0))
    _check(tr.sample_logits(x, uniforms=u, **settings), x, u, like)
    bad = {k: v.clone() for k, v in settings.items()}
    bad["temperature"][1], bad["temperature"][2], bad["temperature"][3] = -1.0, float("nan"), float("inf")
    bad["top_p"][4], bad["min_p"][6] = float("nan"), float("nan")
    v = u.clone()
    v[7], v[8], v[9] = 1.0, -0.25, float("nan")
    got = tr.sample_logits(x, uniforms=v, **bad)
    wrong = [1, 2, 3, 4, 6, 7, 8, 9]
    assert (got.token_ids[wrong] == -1).all() and got.logprobs[wrong].isnan().all() and (got.kept[wrong] == 0).all()
    fine = [0, 5, 10, 11]
    want = tr.sample_logits(x, uniforms=u, **settings)
    assert all(torch.equal(a[fine], b[fine]) for a, b in zip(got, want))


def test_packed_rows_never_read_past_the_arrays(cuda_device):
    """Offsets past the capacity (a truncated compact output), falling ones, empty rows, no rows at all."""
    dev = cuda_device
    x = _logits(15, 1, 100, torch.float16, dev)[0]
    ids = torch.arange(1000, 1100, device=dev)
    offsets = torch.tensor([0, 60, 60, 130, 500, 400], device=dev)
    u = _uniforms(16, 5, dev)
    got = tr.sample_compact_logits(ids, x, offsets, uniforms=u, top_p=0.9)
    rows = [x[:60], x[60:60], x[60:100], x[100:], x[100:]]
    _check(got, rows, u, dict(top_p=0.9), ids=[ids[:60], ids[60:60], ids[60:], ids, ids])
    none = tr.sample_compact_logits(ids[:0], x[:0], torch.zeros(3, dtype=torch.int64, device=dev), uniforms=u[:2])
    assert none.token_ids.tolist() == [0, 0] and none.kept.tolist() == [0, 0]


def test_vocab_offset(cuda_device):
    x = _logits(17, 3, 500, torch.float32, cuda_device)
    u = _uniforms(18, 3, cuda_device)
    want = tr.sample_logits(x, uniforms=u)
    out = tr._sample_outputs(3, cuda_device)
    _native.sample_logits(x, None, (1.0, 0, 1.0, 0.0), u, *out, vocab_offset=7000)
    assert torch.equal(out.token_ids, want.token_ids + 7000)


def test_repeatable_on_streams_and_in_graphs(cuda_device):
    dev = cuda_device
    x = _logits(19, 16, 40009, torch.float16, dev)
    u = _uniforms(20, 16, dev)
    want = tr.sample_logits(x, uniforms=u, top_p=0.95, temperature=1.5)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(tr.sample_logits(x, uniforms=u, top_p=0.95, temperature=1.5), want))
    streams = [torch.cuda.Stream(dev) for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for s in streams:  # at the same time: the call has no workspace
        with torch.cuda.stream(s):
            outs.append([tr.sample_logits(x, uniforms=u, top_p=0.95, temperature=1.5) for _ in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for r in o for a, b in zip(r, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = tr.sample_logits(x, uniforms=u, top_p=0.95, temperature=1.5)
    u2 = _uniforms(21, 16, dev)
    want2 = tr.sample_logits(x, uniforms=u2, top_p=0.95, temperature=1.5)
    u.copy_(u2)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want2))


def test_refusals_of_device_tensors(cuda_device):
    dev = cuda_device
    ids, x = torch.arange(8, device=dev), torch.zeros(8, device=dev)
    offsets = torch.tensor([0, 8], device=dev)
    for u in (torch.zeros((), device=dev), torch.zeros(2, device=dev), torch.zeros(1, 1, device=dev)):
        with pytest.raises(ValueError, match="uniforms"):
            tr.sample_compact_logits(ids, x, offsets, uniforms=u)
        with pytest.raises(ValueError, match="uniforms"):
            tr.sample_logits(x, uniforms=u)
    long = torch.empty(1, 2 ** 32 + 32, dtype=torch.float16, device=dev)  # (32 tokens, cut to 32 bits)
    with pytest.raises(ValueError, match="2\\^30 tokens"):
        tr.sample_logits(long, uniforms=torch.zeros(1, device=dev))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_packed_rows_of_very_different_lengths(cuda_device, dtype):
    """The launch shape follows the mean length: rows far longer and shorter than it, and any stated length, agree."""
    dev = cuda_device
    lengths = [1, 90000, 0, 3, 700, 20]
    x = _logits(23, 1, sum(lengths), dtype, dev)[0]
    ids = torch.arange(x.numel(), device=dev)
    offsets = torch.tensor([0, *np.cumsum(lengths)], device=dev)
    u = _uniforms(24, len(lengths), dev)
    got = tr.sample_compact_logits(ids, x, offsets, uniforms=u, top_p=0.9)
    at = offsets.tolist()
    rows = [x[at[i]:at[i + 1]] for i in range(len(lengths))]
    _check(got, rows, u, dict(top_p=0.9), ids=[ids[at[i]:at[i + 1]] for i in range(len(lengths))])
    for max_len in (0, 1, 5000, 2 ** 40):
        again = tr.sample_compact_logits(ids, x, offsets, uniforms=u, top_p=0.9, max_len=max_len)
        assert all(torch.equal(a, b) for a, b in zip(again, got))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_long_rows_of_a_full_batch(cuda_device, dtype):
    """148 rows of 70,000 tokens with settings per request (counted, one CTA
    per row): every combination of filters, greedy, and rows of one value or
    two, more of it than 16 bits count; then settings known at the call (rows
    split over clusters)."""
    dev = cuda_device
    batch, vocab = 148, 70000
    x = _logits(31, batch, vocab, dtype, dev)
    x[5] = 1.5
    x[6] = -0.75
    x[7, ::2], x[7, 1::2] = 0.0, -0.0
    x[8, 100:], x[8, :100] = -2.0, 2.0
    x[9] = float("-inf")
    x[10, 3::7] = float("nan")
    x[11, 50000:50003] = float("inf")
    u = _uniforms(32, batch, dev)
    at = [SETTINGS[(b * 7) % len(SETTINGS)] for b in range(batch)]
    full = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    types = dict(temperature=torch.float32, top_k=torch.int32, top_p=torch.float32, min_p=torch.float32)
    settings = {k: torch.tensor([{**full, **s}[k] for s in at], dtype=types[k], device=dev) for k in full}
    got = tr.sample_logits(x, uniforms=u, **settings)
    _check(got, x, u, settings)
    for one in (dict(top_k=20), dict(min_p=0.05, temperature=0.9), dict(temperature=0.0), dict(top_k=700, top_p=0.9)):
        _check(tr.sample_logits(x, uniforms=u, **one), x, u, one)
