"""GPU tests of the int8 head: quantize_rows_int8, int8_grammar_logits on its
three routes, int8_compact_logits.

The oracle is 64-bit: integer sums in int64, scales and products in float64.
Bounds, derived from the definition (gsp/int8_head.py):
  scale   one fp32 division: half a step, 2^-24 relative;
  value   rint of one fp32 division: the 64-bit quotient is within
          0.5 + 127.5 * 2^-24 of the integer;
  logit   float(sum), two products: three roundings, (1 + 2^-24)^3 - 1 < 3.01 * 2^-24
          relative, then one to the output type, eps / 2 relative or half the
          smallest subnormal absolute.
The product has one definition in fp32, so the routes agree bit for bit and
equal the same expression evaluated by torch.
"""
import threading

import numpy as np
import pytest
import torch

from gsp import _native
from gsp import int8_head as I
from gsp import triton_runtime as tr
from oracle import gsp_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _rows(seed, n, h, dtype, dev, scale=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(n, h, generator=g) * scale).to(dtype).to(dev)


def _int8_weight(seed, vocab, hidden, dev):
    g = torch.Generator(device="cpu").manual_seed(seed)
    values = torch.randint(-128, 128, (vocab, hidden), generator=g, dtype=torch.int8)
    scales = torch.rand(vocab, generator=g) * 2e-3 + 1e-4
    return I.QuantizedRows(values.to(dev), scales.to(dev))


def _legal(mask, vocab):
    return torch.from_numpy(O.unpack_bitmask(mask.cpu().numpy(), vocab))


# ---------------------------------------------------------------------------
# rows to int8
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (1, 16), (5, 2048), (64, 2064), (2, 8192), (700, 96), (1500, 1023),
                                   (2, 40000), (4097, 512)])
def test_quantize_matches_definition(cuda_device, dtype, shape):
    x = _rows(sum(shape), *shape, dtype, cuda_device)
    q = I.quantize_rows_int8(x)
    assert q.values.dtype == torch.int8 and q.scales.dtype == torch.float32
    x64 = x.double()
    amax = x64.abs().amax(1)
    assert ((q.scales.double() - amax / 127).abs() <= amax / 127 * 2.0 ** -24 * 1.001).all()
    quotient = x64 / q.scales.double().unsqueeze(1)
    assert ((quotient - q.values.double()).abs() <= 0.5 + 127.5 * 2.0 ** -24).all()
    # the same expression in numpy's fp32 (torch divides by a plain number as a product with its reciprocal)
    x32 = x.float().cpu().numpy()
    scale = np.abs(x32).max(axis=1) / np.float32(127)
    assert np.array_equal(q.scales.cpu().numpy(), scale)
    assert np.array_equal(q.values.cpu().numpy(), np.rint(x32 / scale[:, None]).astype(np.int8))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_ties_and_extremes(cuda_device, dtype):
    """Exact halves round to even; zeros, subnormals, the largest values, and rows that are not finite."""
    dev = cuda_device
    big = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # smallest subnormal
    rows = torch.zeros(8, 32, dtype=torch.float64)
    rows[0, :8] = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, -127.0])  # scale 1: exact ties
    rows[2, 0], rows[2, 1] = big, -big
    rows[3, 0], rows[3, 1] = tiny, -3 * tiny
    rows[4, 0], rows[4, 5] = float("inf"), 1.0
    rows[5, 31] = float("nan")
    rows[6, 3] = -0.0
    rows[7] = torch.linspace(-1, 1, 32, dtype=torch.float64)
    x = rows.to(dtype).to(dev)
    q = I.quantize_rows_int8(x)
    assert q.values[0, :8].tolist() == [127, 0, 2, 2, 0, -2, -2, -127]
    assert q.scales[1].item() == 0.0 and (q.values[1] == 0).all()
    assert q.values[2, :2].tolist() == [127, -127]
    x32 = x[3].float().cpu().numpy()
    scale = np.abs(x32).max() / np.float32(127)
    want = np.zeros(32) if scale == 0 else np.clip(np.rint(x32 / scale), -127, 127)
    assert np.array_equal(q.values[3].cpu().numpy(), want)
    for r in (4, 5):
        assert torch.isnan(q.scales[r]) and (q.values[r] == 0).all()
    assert q.scales[6].item() == 0.0 and (q.values[6] == 0).all()
    assert q.values[7, 0].item() == -127 and q.values[7, 31].item() == 127


def test_quantize_strided_rows_and_out(cuda_device):
    dev = cuda_device
    base = _rows(1, 40, 300, torch.bfloat16, dev)
    for view in (base[:, :256], base[:, 3:250], base[::2], base[:1].expand(7, 300)):
        got = I.quantize_rows_int8(view)
        want = I.quantize_rows_int8(view.contiguous())
        assert torch.equal(got.values, want.values) and torch.equal(got.scales, want.scales)
    out = I.QuantizedRows(torch.full((42, 300), 77, dtype=torch.int8, device=dev),
                          torch.full((42,), -1.0, device=dev))
    part = I.QuantizedRows(out.values[1:41], out.scales[1:41])
    assert I.quantize_rows_int8(base, out=part) is part
    assert (out.values[0] == 77).all() and (out.values[41] == 77).all()  # the rows around are left as they were
    assert out.scales[0].item() == -1.0 and out.scales[41].item() == -1.0
    assert I.quantize_rows_int8(base[:0]).values.shape == (0, 300)


# ---------------------------------------------------------------------------
# projection
# ---------------------------------------------------------------------------
def _check(h, weight, mask, dtype, got, legal):
    logits, top_value, top_index = got
    vocab = weight.values.shape[0]
    q = h if isinstance(h, I.QuantizedRows) else I.quantize_rows_int8(h)
    total = torch.from_numpy(q.values.cpu().numpy().astype(np.int64) @ weight.values.cpu().numpy().astype(np.int64).T)
    hs, ws = q.scales.cpu(), weight.scales.cpu()
    # the 64-bit value within the derived bound
    y64 = total.double() * hs.double().unsqueeze(1) * ws.double().unsqueeze(0)
    eps, sub = torch.finfo(dtype).eps, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    bound = y64.abs() * (3.01 * 2.0 ** -24 + eps / 2 * (1 + 2.0 ** -20)) + sub / 2
    out = logits.cpu()
    assert torch.equal(out.isneginf(), ~legal)
    assert ((out.double() - y64).abs()[legal] <= bound[legal]).all()
    # the definition's own bits
    want = (total.float() * hs.unsqueeze(1) * ws.unsqueeze(0)).to(dtype).masked_fill(~legal, float("-inf"))
    assert torch.equal(out, want)
    # the fused top-1: largest logit, lowest id
    top = want.amax(1)
    assert torch.equal(top_value.cpu(), top.float())
    first = torch.where(legal & (want == top.unsqueeze(1)), torch.arange(vocab), vocab).amin(1)
    assert torch.equal(top_index.cpu(), torch.where(first < vocab, first, 0))
    assert _native.workspace_error(logits.device) == 0


CASES = [
    # vocab, hidden, batch, legal tokens per request, clustered
    (1, 16, 1, [1], False),
    (33, 64, 1, [5], False),
    (4099, 256, 1, [41], True),
    (1000, 48, 2, [0, 999], False),           # a request without a legal token
    (5000, 1024, 3, [5000, 0, 17], True),
    (3001, 2064, 33, [60] * 33, False),       # K tail inside a stage, odd vocabulary
    (40000, 128, 16, [300] * 16, True),       # cooperative kernel (20,000 mask words)
    (2600, 100, 5, [130] * 5, False),         # rows without 16-byte alignment
    (777, 31, 40, [40] * 40, False),
    (1300, 64, 300, [13] * 300, True),        # two chunks of requests on the tensor cores
    (700, 320, 130, [699] * 130, False),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES)
def test_routes_match_definition(cuda_device, case, dtype):
    vocab, hidden, batch, counts, clustered = case
    rng = np.random.default_rng(vocab + batch)
    mask_np = O.make_batch_mask(rng, batch, vocab, counts, clustered=clustered, max_runs=5)
    mask = torch.from_numpy(mask_np).to(cuda_device)
    weight = _int8_weight(vocab, vocab, hidden, cuda_device)
    h = _rows(batch, batch, hidden, dtype, cuda_device)
    legal = _legal(mask, vocab)
    for route in tr.ROUTES:
        got = I.int8_grammar_logits(h, weight, mask, route=route)
        assert got[0].dtype == dtype and got[0].shape == (batch, vocab)
        _check(h, weight, mask, dtype, got, legal)


@pytest.mark.parametrize("route", tr.ROUTES)
def test_no_mask_wide_mask_and_quantised_hidden(cuda_device, route):
    vocab, hidden, batch = 2050, 512, 9
    weight = _int8_weight(2, vocab, hidden, cuda_device)
    h = _rows(3, batch, hidden, torch.float16, cuda_device)
    every = torch.ones(batch, vocab, dtype=torch.bool)
    _check(h, weight, None, torch.float16, I.int8_grammar_logits(h, weight, None, route=route), every)
    q = I.quantize_rows_int8(h)
    _check(q, weight, None, torch.float32, I.int8_grammar_logits(q, weight, None, route=route,
                                                                 out_dtype=torch.float32), every)
    # a mask with words past the vocabulary, all of whose bits are set
    rng = np.random.default_rng(5)
    narrow = O.make_batch_mask(rng, batch, vocab, [100] * batch)
    wide = np.full((batch, narrow.shape[1] + 3), -1, dtype=np.int32)
    wide[:, :narrow.shape[1]] = narrow
    wide[:, narrow.shape[1] - 1] |= np.int32(-1) << np.int32(vocab % 32)
    mask = torch.from_numpy(wide).to(cuda_device)
    legal = _legal(torch.from_numpy(narrow), vocab)
    _check(h, weight, mask, torch.float16, I.int8_grammar_logits(h, weight, mask, route=route), legal)
    no_logits = I.int8_grammar_logits(h, weight, mask, route=route, return_logits=False)
    assert no_logits[0] is None
    assert torch.equal(no_logits[2], I.int8_grammar_logits(h, weight, mask, route=route)[2])


@pytest.mark.parametrize("route", tr.ROUTES)
def test_extreme_sums_are_exact(cuda_device, route):
    """Every product at its largest: sums past 2^24 (fp32 would round them on
    the way) and, at the longest row, near 2^31."""
    for hidden in (4096, 131056):
        vocab, batch = 130, 3
        values = torch.full((vocab, hidden), -128, dtype=torch.int8, device=cuda_device)
        values[1] = 127
        values[2, ::2] = 127
        weight = I.QuantizedRows(values, torch.ones(vocab, device=cuda_device))
        q = I.QuantizedRows(torch.full((batch, hidden), -128, dtype=torch.int8, device=cuda_device),
                            torch.ones(batch, device=cuda_device))
        every = torch.ones(batch, vocab, dtype=torch.bool)
        got = I.int8_grammar_logits(q, weight, None, route=route, out_dtype=torch.float32)
        assert got[0][0, 0].item() == float(128 * 128 * hidden)
        _check(q, weight, None, torch.float32, got, every)


def test_nan_rows_show_in_the_logits(cuda_device):
    vocab, hidden = 300, 64
    weight = _int8_weight(7, vocab, hidden, cuda_device)
    h = _rows(8, 2, hidden, torch.float16, cuda_device)
    h[1, 5] = float("nan")
    for route in tr.ROUTES:
        logits, _, _ = I.int8_grammar_logits(h, weight, None, route=route)
        assert torch.isnan(logits[1]).all() and torch.isfinite(logits[0]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [(1, 4099, 256, [41]), (4, 3000, 48, [0, 500, 1, 3000]), (20, 30000, 96, [200] * 20),
                                  (3, 500, 30, [10, 0, 0])])
def test_compact_matches_full_logits(cuda_device, case, dtype):
    batch, vocab, hidden, counts = case
    rng = np.random.default_rng(vocab)
    mask = torch.from_numpy(O.make_batch_mask(rng, batch, vocab, counts)).to(cuda_device)
    weight = _int8_weight(11, vocab, hidden, cuda_device)
    h = _rows(12, batch, hidden, dtype, cuda_device)
    full, _, _ = I.int8_grammar_logits(h, weight, mask)
    legal = _legal(mask, vocab).to(cuda_device)
    ids, logits, offsets = I.int8_compact_logits(h, weight, mask)
    counts = legal.sum(1)
    assert torch.equal(offsets, torch.cat([counts.new_zeros(1), counts.cumsum(0)]))
    assert torch.equal(ids, legal.nonzero()[:, 1]) and torch.equal(logits, full[legal])
    # a capacity below the count writes that much, one above leaves the rest
    n = int(counts.sum())
    if n > 5:
        few = I.int8_compact_logits(h, weight, mask, capacity=5)
        assert torch.equal(few[0], ids[:5]) and torch.equal(few[1], logits[:5]) and torch.equal(few[2], offsets)
    more = I.int8_compact_logits(h, weight, mask, capacity=n + 9)
    assert torch.equal(more[0][:n], ids) and torch.equal(more[1][:n], logits)


@pytest.mark.parametrize("route", tr.ROUTES)
def test_streams_and_graphs(cuda_device, route):
    """On a side stream, and captured: two graphs replayed in turn and at the
    same time on two streams, each with a workspace of its own."""
    dev = cuda_device
    vocab, hidden, batch = 9000, 256, 4
    rng = np.random.default_rng(3)
    mask = torch.from_numpy(O.make_batch_mask(rng, batch, vocab, [90] * batch)).to(dev)
    weight = _int8_weight(21, vocab, hidden, dev)
    hs = [_rows(30 + i, batch, hidden, torch.bfloat16, dev) for i in range(2)]
    want = [I.int8_grammar_logits(h, weight, mask, route=route) for h in hs]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = I.int8_grammar_logits(hs[0], weight, mask, route=route)
    torch.cuda.current_stream(dev).wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graphs, outs = [], []
    for h in hs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(I.int8_grammar_logits(h, weight, mask, route=route))
        graphs.append(g)
    streams = [torch.cuda.Stream(dev) for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(o, w))


@pytest.mark.parametrize("route", tr.ROUTES)
@pytest.mark.parametrize("hidden", [31, 256])
def test_operands_at_odd_addresses(cuda_device, route, hidden):
    """Contiguous operands that begin in the middle of an allocation: bytes 3 and 5 off a 16-byte boundary."""
    vocab, batch = 517, 3
    dev = cuda_device
    w, q = _int8_weight(41, vocab, hidden, dev), I.quantize_rows_int8(_rows(42, batch, hidden, torch.float16, dev))
    values = torch.empty(vocab * hidden + 3, dtype=torch.int8, device=dev)[3:].view(vocab, hidden).copy_(w.values)
    states = torch.empty(batch * hidden + 5, dtype=torch.int8, device=dev)[5:].view(batch, hidden).copy_(q.values)
    mask = torch.from_numpy(O.make_batch_mask(np.random.default_rng(43), batch, vocab, [60, 0, 500])).to(dev)
    legal = _legal(mask, vocab)
    for weight, h in ((I.QuantizedRows(values, w.scales), q), (w, I.QuantizedRows(states, q.scales))):
        got = I.int8_grammar_logits(h, weight, mask, route=route, out_dtype=torch.float16)
        _check(h, weight, mask, torch.float16, got, legal)


def test_sizes_past_32_bits_are_refused(cuda_device):
    x = torch.empty(1, 2 ** 32 + 32, dtype=torch.float16, device=cuda_device)  # (32 columns, cut to 32 bits)
    with pytest.raises(ValueError, match="2\\^30 columns"):
        I.quantize_rows_int8(x)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [(5000, 2048, 1), (5000, 4096, 4), (2000, 48, 2), (900, 16400, 1), (900, 1040, 3)])
def test_hidden_states_of_few_requests(cuda_device, case, dtype):
    """Quantised inside the projection (or, past its limits, before it): the
    bits of the quantiser's values and scales, zeros and rows that are not
    finite among them, contiguous rows at any 16-byte address and others."""
    vocab, hidden, batch = case
    dev = cuda_device
    weight = _int8_weight(51, vocab, hidden, dev)
    mask = torch.from_numpy(O.make_batch_mask(np.random.default_rng(52), batch, vocab, [vocab // 9] * batch)).to(dev)
    legal = _legal(mask, vocab)
    h = _rows(53, batch, hidden, dtype, dev)
    h[batch - 1, hidden - 1] = -9.0  # the maximum in the last place
    _check(h, weight, mask, dtype, I.int8_grammar_logits(h, weight, mask), legal)
    space = torch.zeros(batch * hidden + 9, dtype=dtype, device=dev)
    for shift in (8, 1):  # 16 bytes (fp32: 32), and an odd address
        moved = space[shift:shift + batch * hidden].view(batch, hidden).copy_(h)
        _check(moved, weight, mask, dtype, I.int8_grammar_logits(moved, weight, mask), legal)
    ids, logits, offsets = I.int8_compact_logits(h, weight, mask)
    full = I.int8_grammar_logits(h, weight, mask)[0]
    assert torch.equal(logits, full[legal.to(dev)]) and offsets[-1].item() == int(legal.sum())
    h[0] = 0.0
    _check(h, weight, mask, dtype, I.int8_grammar_logits(h, weight, mask), legal)
    h[batch - 1, 3] = float("inf")
    out = I.int8_grammar_logits(h, weight, mask)[0]
    assert out[batch - 1][legal[batch - 1].to(dev)].isnan().all() and out[~legal.to(dev)].isneginf().all()


@pytest.mark.parametrize("route", tr.ROUTES)
def test_threads_on_one_stream(cuda_device, route):
    """Two threads' calls of two launches each, on the same stream: neither's
    scratch nor tile list is the other's."""
    dev = cuda_device
    vocab, hidden, batch, rounds = 6000, 128, 7, 60
    weight = _int8_weight(61, vocab, hidden, dev)
    hs = [_rows(62 + i, batch, hidden, torch.float16, dev) for i in range(2)]
    masks = [torch.from_numpy(O.make_batch_mask(np.random.default_rng(64 + i), batch, vocab, [9] * batch)).to(dev)
             for i in range(2)]
    want = [I.int8_grammar_logits(h, weight, m, route=route) for h, m in zip(hs, masks)]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        for _ in range(rounds):
            got[i].append(I.int8_grammar_logits(hs[i], weight, masks[i], route=route))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == rounds
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
    assert _native.workspace_error(dev) == 0
