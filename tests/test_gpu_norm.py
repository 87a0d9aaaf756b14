"""GPU tests of rms_norm against a 64-bit restatement, and of the fp8 quantisers
against their definition.

Tolerances, in units of 2^-24 (half a step of fp32), with H columns: the squares'
sum has at most H / 32 terms per thread and a tree of at most 12; its root halves
that; division, eps, root, reciprocal and the two products add one each:
e(H) = H / 64 + 12, rounded up to H / 64 + 16. The output rounds once more (half a
step of its type). An 8-bit value is off by half of its step, and by the errors of
y and of the scale on the way there; the scale by y's error and its division. The
new residual is equal.
"""
import math

import pytest
import torch

from gsp import fp8_head as F
from gsp import int8_head, norm

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
SHAPES = [(1, 1), (3, 7), (2, 100), (5, 128), (9, 303), (64, 2048), (2, 4099), (7, 8192), (3, 16384), (2, 16390), (2, 20000),
          (1, 70000), (700, 1024)]
STEP = 2.0 ** -24


def _rows(seed, n, h, dtype, scale=1.0):
    return (torch.randn(n, h, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _reference(x, residual, weight, eps):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    d = h.double()
    y = d / (d.pow(2).mean(1, keepdim=True) + eps).sqrt()
    return h, y if weight is None else y * weight.double()


def _check(r, x, residual, weight, eps, quantize):
    h, y = _reference(x, residual, weight, eps)
    e = STEP * (x.shape[1] / 64 + 16)
    if residual is None:
        assert r.residual is None
    else:
        assert torch.equal(r.residual.cpu(), h)
    if quantize is None:
        got = r.output.double().cpu()
        info = torch.finfo(x.dtype)
        bound = y.abs() * (e + info.eps / 2) + info.tiny * info.eps
        assert r.output.dtype == x.dtype and ((got - y).abs() <= bound).all(), ((got - y).abs() / bound).max()
        return
    values, scales = r.output.values.double().cpu(), r.output.scales.double().cpu()
    if quantize == "int8":
        assert isinstance(r.output, int8_head.QuantizedRows) and r.output.values.dtype == torch.int8
        want = y.abs().amax(1) / 127
        by = scales.unsqueeze(1)
        half = by * 0.5
    else:
        assert isinstance(r.output, F.Fp8Rows) and r.output.values.dtype == torch.float8_e4m3fn
        pad = torch.nn.functional.pad(y, (0, -y.shape[1] % 128)).view(y.shape[0], -1, 128)
        want = pad.abs().amax(2) / 448
        by = scales.repeat_interleave(128, 1)[:, :y.shape[1]]
        half = torch.maximum(y.abs() * 2.0 ** -4, by * 2.0 ** -10)
    assert scales.shape == want.shape
    tiny = torch.finfo(torch.float32).tiny
    assert ((scales - want).abs() <= want * (e + 2 * STEP) + tiny).all()
    bound = half * (1 + 4 * e) + y.abs() * (4 * e + 4 * STEP) + tiny
    assert ((values * by - y).abs() <= bound).all(), ((values * by - y).abs() / bound).max()


@pytest.mark.parametrize("quantize", [None, "int8", "fp8"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_norm_matches_64_bits(cuda_device, shape, dtype, quantize):
    n, h = shape
    x, residual, weight = _rows(1, n, h, dtype, 0.5), _rows(2, n, h, dtype, 3.0), _rows(3, 1, h, dtype)[0]
    for res, w in ((residual, weight), (None, weight), (residual, None)):
        r = norm.rms_norm(x.to(cuda_device), None if w is None else w.to(cuda_device),
                          residual=None if res is None else res.to(cuda_device), eps=1e-6, quantize=quantize)
        _check(r, x, res, w, 1e-6, quantize)


@pytest.mark.parametrize("quantize", [None, "int8", "fp8"])
def test_norm_strides_in_place_and_one_row(cuda_device, quantize):
    wide, stream = _rows(4, 6, 1032, torch.bfloat16), _rows(5, 6, 1032, torch.bfloat16)
    weight = _rows(6, 1, 1024, torch.bfloat16)[0]
    for first in (0, 1, 8):
        x, res = wide[:, first:first + 1024], stream[:, 8 - first:8 - first + 1024]
        xd, rd = wide.to(cuda_device)[:, first:first + 1024], stream.to(cuda_device)
        rv = rd[:, 8 - first:8 - first + 1024]
        r = norm.rms_norm(xd, weight.to(cuda_device), residual=rv, quantize=quantize, residual_out=rv)
        assert r.residual.data_ptr() == rv.data_ptr()
        _check(r, x, res, weight, 1e-6, quantize)
        outside = torch.ones(1032, dtype=torch.bool)
        outside[8 - first:8 - first + 1024] = False
        assert torch.equal(rd.cpu()[:, outside], stream[:, outside])  # what is not the rows' stays
    shared = wide[:1, :1024].expand(6, 1024)
    _check(norm.rms_norm(wide.to(cuda_device)[:1, :1024].expand(6, 1024), quantize=quantize), shared, None, None, 1e-6, quantize)
    one = norm.rms_norm(wide.to(cuda_device)[0, :1024], weight.to(cuda_device), residual=stream.to(cuda_device)[0, :1024],
                        quantize=quantize)
    assert one.residual.shape == (1024,)
    h, y = _reference(wide[:1, :1024], stream[:1, :1024], weight, 1e-6)
    if quantize is None:
        assert one.output.shape == (1024,) and (one.output.double().cpu() - y[0]).abs().max() <= y.abs().max() * 2.0 ** -7
    else:
        assert one.output.values.shape == (1, 1024)


def test_norm_extremes(cuda_device):
    h = 512
    x = torch.zeros(6, h)
    x[1] = 1e-30                    # squares vanish beside eps
    x[2, 5] = math.inf
    x[3, 7] = math.nan
    x[4] = 1e18                     # squares up to 1e36 * 512
    x[5, 0] = 3.0                   # blocks of zeros beside one that is not
    for quantize in (None, "int8", "fp8"):
        r = norm.rms_norm(x.to(cuda_device), quantize=quantize)
        if quantize is None:
            out = r.output.cpu()
            assert (out[0] == 0).all() and torch.allclose(out[4], torch.ones(h), rtol=1e-5)
            assert out[2, 5].isnan() and out[3].isnan().all()
        else:
            scales = r.output.scales.cpu().view(6, -1)
            values = r.output.values.float().cpu()
            assert (scales[0] == 0).all() and (values[0] == 0).all()
            assert scales[2].isnan().any() and scales[3].isnan().all() and (values[3] == 0).all()
            if quantize == "fp8":
                assert (scales[5, 1:] == 0).all() and values[5, 0] == 448 and (values[5, 1:] == 0).all()
    empty = norm.rms_norm(torch.empty(0, h, device=cuda_device), quantize="fp8")
    assert empty.output.values.shape == (0, h) and empty.output.scales.shape == (0, 4)


def _blocks_reference(x, rows):
    n, h = x.shape
    f = x.float()
    pad = torch.nn.functional.pad(f, (0, -h % 128, 0, -n % rows))
    blocks = pad.view(pad.shape[0] // rows, rows, -1, 128)
    top = blocks.abs().amax((1, 3))
    scales = torch.where(torch.isfinite(top), top / torch.tensor(448.0), math.nan)
    by = scales[:, None, :, None]
    values = torch.where(by > 0, blocks / by, 0.0).clamp(-448, 448).to(torch.float8_e4m3fn)
    return values.view(pad.shape)[:n, :h], scales


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 100), (130, 264), (64, 2048), (257, 1000), (5, 4099), (300, 128)])
def test_quantisers_are_their_definition(cuda_device, shape, dtype):
    x = _rows(11, *shape, dtype, 0.02)
    x[0, 0] = 0.0
    if shape[0] > 2 and shape[1] >= 256:
        x[1, 128:256] = 0.0
        x[2, 3], x[2, 200] = math.inf, math.nan
        x[0, 128:256] = torch.finfo(dtype).tiny * torch.finfo(dtype).eps  # a scale that is denormal, or 0
    for quantise, rows in ((F.quantize_rows_fp8, 1), (F.quantize_weight_fp8, 128)):
        want, scales = _blocks_reference(x, rows)
        got = quantise(x.to(cuda_device))
        assert torch.equal(got.scales.cpu().isnan(), scales.isnan())
        assert torch.equal(got.scales.cpu().nan_to_num(-1), scales.nan_to_num(-1))
        assert torch.equal(got.values.cpu().view(torch.uint8), want.contiguous().view(torch.uint8))
        wide = torch.cat([x, x], 1).to(cuda_device)[:, 1:1 + shape[1]]  # rows of another stride, not aligned
        again = quantise(wide, out=got)
        assert again.values.data_ptr() == got.values.data_ptr()
        want, scales = _blocks_reference(torch.cat([x, x], 1)[:, 1:1 + shape[1]], rows)
        assert torch.equal(again.values.cpu().view(torch.uint8), want.contiguous().view(torch.uint8))


def test_fp8_norm_of_a_normed_row_is_the_quantisers(cuda_device):
    """With a root mean square of one, no weight and eps 0, y is x itself: the norm's 8-bit output is the quantiser's."""
    x = torch.where(torch.rand(64, 1024, generator=torch.Generator().manual_seed(1)) < 0.5, -1.0, 1.0).to(cuda_device)
    a, b = norm.rms_norm(x, eps=0.0, quantize="fp8").output, F.quantize_rows_fp8(x)
    assert torch.equal(a.values.view(torch.uint8), b.values.view(torch.uint8)) and torch.equal(a.scales, b.scales)


def test_norm_refusals(cuda_device):
    x = torch.zeros(2, 64, device=cuda_device)
    for kw, word in ((dict(quantize="int4"), "quantize"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"),
                     (dict(weight=torch.ones(32, device=cuda_device)), "weight"), (dict(residual=x[:1]), "residual"),
                     (dict(weight=torch.ones(64, device=cuda_device).half()), "weight"),
                     (dict(residual=x.half()), "residual"), (dict(residual_out=x), "residual_out"),
                     (dict(weight=torch.ones(64, device=cuda_device, requires_grad=True)), "gradient")):
        with pytest.raises(ValueError, match=word):
            norm.rms_norm(x, **kw)
    with pytest.raises(ValueError, match="overlap"):
        norm.rms_norm(x, residual=x, residual_out=x[:1].expand(2, 64))
    with pytest.raises(ValueError, match="contiguous"):
        norm.rms_norm(torch.zeros(64, 2, device=cuda_device).T)
