"""GPU tests of the fp8 head against 64-bit sums of its quantised operands.

Tolerance: a block's 128 products are exact; a tensor-core instruction adds 32 of
them and the sum so far, each cut at worst at 2^-23 of the largest, four times over:
4 * 33 * 2 units of 2^-24. A block's scales multiply twice and add once per block
(the row-sparse kernel: one rounding per state, 16 products in a chain, then a tree
of 6). In all (264 + blocks + 16) * 2^-24 of the sum of magnitudes, then half a step
of the logits' type (and of its smallest number).
"""
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
SHAPES = [(1, 1, 16), (2, 33, 64), (3, 4099, 256), (32, 20000, 512), (33, 3001, 144), (64, 9000, 1024), (128, 5003, 384),
          (129, 4100, 1024), (300, 2500, 272), (5, 3000, 100), (7, 1000, 2048), (1, 50257, 768), (70, 257, 4096)]


def _case(seed, batch, vocab, hidden, dtype, dev):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(batch, hidden, generator=g).to(dtype).to(dev)
    w = (torch.randn(vocab, hidden, generator=g) * 0.02).to(dev)
    return h, F.quantize_weight_fp8(w)


def _mask(seed, batch, vocab, clustered):
    rng = np.random.default_rng(seed)
    counts = [min(vocab, c) for c in rng.choice([0, 1, max(1, vocab // 50), max(1, vocab // 3)], batch)]
    return torch.from_numpy(O.make_batch_mask(rng, batch, vocab, counts, clustered=clustered, max_runs=8))


def _legal(mask, vocab):
    v = torch.arange(vocab)
    return ((mask.cpu()[:, v >> 5] >> (v & 31)) & 1).bool()


def _exact(rows, weight):
    hidden = weight.values.shape[1]
    h = rows.values.double() * rows.scales.double().repeat_interleave(128, 1)[:, :hidden]
    w = weight.values.double() * weight.scales.double().repeat_interleave(128, 0)[:weight.values.shape[0]] \
        .repeat_interleave(128, 1)[:, :hidden]
    return (h @ w.T).cpu(), (h.abs() @ w.abs().T).cpu()


def _check(result, exact, size, legal, dtype, blocks):
    logits, value, index = result
    got = logits.cpu()
    assert got.dtype == dtype and got.shape == exact.shape
    assert (got[~legal] == -math.inf).all()
    info = torch.finfo(dtype)
    bound = size * (264 + blocks + 16) * 2.0 ** -24
    bound = bound + (exact.abs() + bound) * info.eps / 2 + info.tiny * info.eps
    off = (got.double() - exact).abs()
    assert (off[legal] <= bound[legal]).all(), (off[legal] / bound[legal]).max()
    first = got.float().argmax(1)  # (CPU: the first of equal ones)
    assert torch.equal(index.cpu(), first)
    assert torch.equal(value.cpu(), got.float().gather(1, first.unsqueeze(1)).squeeze(1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_routes_match_64_bits(cuda_device, shape, dtype):
    batch, vocab, hidden = shape
    h, weight = _case(sum(shape), batch, vocab, hidden, dtype, cuda_device)
    rows = F.quantize_rows_fp8(h)
    exact, size = _exact(rows, weight)
    for clustered in (False, True):
        mask = _mask(vocab, batch, vocab, clustered).to(cuda_device)
        legal = _legal(mask, vocab)
        for route in tr.ROUTES:
            for given in (h, rows):
                out = F.fp8_grammar_logits(given, weight, mask, route=route, out_dtype=dtype)
                _check(out, exact, size, legal, dtype, (hidden + 127) // 128)
    every = torch.ones(batch, vocab, dtype=torch.bool)
    for route in tr.ROUTES:
        _check(F.fp8_grammar_logits(rows, weight, None, route=route, out_dtype=dtype), exact, size, every, dtype,
               (hidden + 127) // 128)
    assert _native.workspace_error(cuda_device) == 0


@pytest.mark.parametrize("shape", [(2, 300, 32768), (3, 1048609, 16), (140, 1048609, 16), (1, 129, 33), (260, 40, 128)])
def test_largest_hidden_size_and_vocabularies_past_the_list(cuda_device, shape):
    """The widest hidden state that shared memory takes; vocabularies whose active groups are not listed (the block
    route then takes the legal rows); sizes below a vector, a block and a tile."""
    batch, vocab, hidden = shape
    h, weight = _case(7, batch, vocab, hidden, torch.bfloat16, cuda_device)
    rows = F.quantize_rows_fp8(h)
    exact, size = _exact(rows, weight)
    legal = torch.zeros(batch, vocab, dtype=torch.bool)
    legal[:, ::97], legal[0, -1] = True, True
    words = torch.zeros(batch, (vocab + 31) // 32 * 32, dtype=torch.uint8)
    words[:, :vocab] = legal
    mask = torch.from_numpy(np.packbits(words.numpy(), axis=1, bitorder="little").view(np.int32).copy()).to(cuda_device)
    for route in tr.ROUTES:
        _check(F.fp8_grammar_logits(h, weight, mask, route=route), exact, size, legal, torch.bfloat16, (hidden + 127) // 128)
    assert _native.workspace_error(cuda_device) == 0


@pytest.mark.parametrize("batch", [1, 17, 200])
@pytest.mark.parametrize("route", tr.ROUTES)
def test_masks_without_a_token_wide_masks_and_no_logits(cuda_device, route, batch):
    vocab, hidden = 5000, 256
    h, weight = _case(1, batch, vocab, hidden, torch.bfloat16, cuda_device)
    none = torch.zeros(batch, (vocab + 31) // 32, dtype=torch.int32, device=cuda_device)
    logits, value, index = F.fp8_grammar_logits(h, weight, none, route=route)
    assert (logits == -math.inf).all() and (value == -math.inf).all() and (index == 0).all()
    wide = torch.full((batch, (vocab + 31) // 32 + 3), -1, dtype=torch.int32, device=cuda_device)  # bits past the vocabulary too
    full = F.fp8_grammar_logits(h, weight, wide, route=route)
    free = F.fp8_grammar_logits(h, weight, None, route=route)
    assert all(torch.equal(a, b) for a, b in zip(full, free))
    _, value, index = F.fp8_grammar_logits(h, weight, wide, route=route, return_logits=False)
    assert torch.equal(value, full[1]) and torch.equal(index, full[2])
    last = none.clone()
    last[:, (vocab - 1) // 32] = 1 << ((vocab - 1) % 32)  # the last token alone
    _, _, index = F.fp8_grammar_logits(h, weight, last, route=route)
    assert (index == vocab - 1).all()


@pytest.mark.parametrize("route", tr.ROUTES)
def test_zeros_and_values_that_are_not_finite(cuda_device, route):
    vocab, hidden = 700, 384
    h, weight = _case(2, 4, vocab, hidden, torch.float16, cuda_device)
    h[0] = 0.0
    h[1, 130] = math.inf
    h[2, 5] = math.nan
    mask = torch.full((4, 22), -1, dtype=torch.int32, device=cuda_device)
    mask[:, 0] = -16  # tokens 0 to 3 are illegal
    logits, value, index = F.fp8_grammar_logits(h, weight, mask, route=route)
    assert (logits[:, :4] == -math.inf).all()
    assert (logits[0, 4:] == 0).all() and index[0] == 4
    assert logits[1:3, 4:].isnan().all() and (index[1:3] == 4).all() and value[1:3].isnan().all()
    assert torch.isfinite(logits[3, 4:]).all()


def test_streams_threads_and_captured_calls(cuda_device):
    import threading
    vocab, hidden, batch = 20011, 512, 24
    h, weight = _case(3, batch, vocab, hidden, torch.bfloat16, cuda_device)
    masks = [_mask(s, batch, vocab, True).to(cuda_device) for s in (1, 2)]
    want = {(r, i): F.fp8_grammar_logits(h, weight, masks[i], route=r) for r in tr.ROUTES for i in (0, 1)}
    torch.cuda.synchronize()
    failed = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(10):
                for route in tr.ROUTES:
                    got = F.fp8_grammar_logits(h, weight, masks[i], route=route)
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[route, i])):
                        failed.append((route, i))

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed
    # two graphs, replayed in turn and side by side: each has scratch of its own
    mask = masks[0].clone()
    graphs, outs = [], []
    for route in ("block-sparse", "row-sparse"):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(F.fp8_grammar_logits(h, weight, mask, route=route))
        graphs.append(g)
    for i in (1, 0, 1):
        mask.copy_(masks[i])
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for route, out in zip(("block-sparse", "row-sparse"), outs):
            assert all(torch.equal(a, b) for a, b in zip(out, want[route, i])), (route, i)
    assert _native.workspace_error(cuda_device) == 0


def test_refusals(cuda_device):
    h, weight = _case(4, 2, 300, 256, torch.float16, cuda_device)
    mask = torch.full((2, 10), -1, dtype=torch.int32, device=cuda_device)
    rows = F.quantize_rows_fp8(h)
    bad = (((h, weight, mask[:, :9].contiguous()), {}, "bitmask"), ((h, weight, mask.long()), {}, "int32"),
           ((h[:, :128].contiguous(), weight, mask), {}, "dimension"), ((rows, weight, mask), {}, "out_dtype"),
           ((h, weight, mask), {"route": "none"}, "route"), ((h, weight, mask), {"out_dtype": torch.int32}, "dtype"),
           ((h, F.Fp8Weight(weight.values, weight.scales[:2]), mask), {}, "scales"),
           ((h, F.Fp8Weight(weight.values.view(torch.uint8), weight.scales), mask), {}, "float8"),
           ((F.Fp8Rows(rows.values, rows.scales[:1]), weight, mask), {"out_dtype": torch.float16}, "scales"),
           ((h.T, weight, mask), {}, "contiguous"), ((h.cpu(), weight, mask), {}, "CUDA"))
    for args, kw, word in bad:
        with pytest.raises(ValueError, match=word):
            F.fp8_grammar_logits(*args, **kw)
    with pytest.raises(ValueError, match="32768"):
        wide = F.Fp8Weight(torch.zeros(128, 32896, dtype=torch.uint8, device=cuda_device).view(torch.float8_e4m3fn),
                           torch.ones(1, 257, device=cuda_device))
        F.fp8_grammar_logits(torch.zeros(1, 32896, device=cuda_device), wide, None)
