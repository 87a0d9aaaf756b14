"""The filtered sampler without a GPU: its oracle on rows small enough to
count by hand, and the refusals of the C ABI and of the Python entry points."""
import ctypes

import numpy as np
import pytest
import torch

from gsp import _native
from gsp import triton_runtime as tr
from oracle import gsp_oracle as O

FAKE = ctypes.c_void_p(4096)  # never dereferenced: every call below fails validation first


def test_oracle_counts_by_hand():
    row = np.log([0.1, 0.4, 0.2, 0.2, 0.1])  # order: 1, 2, 3, 0, 4
    draw = lambda u, **kw: O.filtered_sample_reference(row, u, **kw)
    assert [draw(u)[0] for u in (0.0, 0.39, 0.41, 0.59, 0.61, 0.85, 0.95)] == [1, 1, 2, 2, 3, 0, 4]
    assert draw(0.9, top_k=2)[0] == 2 and draw(0.9, top_k=2)[2] == 2
    assert abs(draw(0.9, top_k=2)[1] - np.log(0.2 / 0.6)) < 1e-12
    assert draw(0.99, top_p=0.55)[2] == 2 and draw(0.99, top_p=0.65)[2] == 3 and draw(0.5, top_p=0.0)[2] == 1
    assert draw(0.99, min_p=0.4)[2] == 3 and draw(0.99, min_p=0.6)[0] == 1
    assert draw(0.99, top_k=3, top_p=0.6)[2] == 2  # 0.4 / 0.8 and 0.6 / 0.8: the shortest prefix of at least 0.6 has two
    assert draw(0.7, temperature=0.0) == (1, 0.0, 1)
    assert O.filtered_sample_reference([-np.inf, np.nan], 0.3) == (0, -np.inf, 0)


def _sample(**kw):
    a = dict(x=FAKE, s=64, d=0, mask=None, ms=0, batch=2, vocab=64, off=0, t=1.0, ta=None, k=0, ka=None, p=1.0,
             pa=None, m=0.0, ma=None, u=FAKE, ids=FAKE, lp=None, kept=None)
    a.update(kw)
    return _native.load().gsp_sample_logits(*a.values(), None)


def test_sample_logits_refusals():
    lib = _native.load()
    nan = float("nan")
    for kw, word in (({"x": None}, b"logits"), ({"vocab": 0}, b"vocab"), ({"batch": 0}, b"batch"),
                     ({"s": -1}, b"logits_row_stride"), ({"mask": FAKE, "ms": 1}, b"bitmask_row_stride"),
                     ({"u": None}, b"uniforms"), ({"ids": None}, b"token_ids"), ({"t": -0.5}, b"temperature"),
                     ({"t": float("inf")}, b"temperature"), ({"t": nan}, b"temperature"), ({"p": nan}, b"top_p"),
                     ({"m": nan}, b"min_p")):
        assert _sample(**kw) == _native.GSP_ERR_INVALID_ARGUMENT, kw
        assert word in lib.gsp_last_error(), (kw, lib.gsp_last_error())
    assert _sample(d=7) == _native.GSP_ERR_UNSUPPORTED
    assert _sample(vocab=(1 << 30) + 1, s=1 << 31) == _native.GSP_ERR_UNSUPPORTED and b"2^30" in lib.gsp_last_error()


def test_sample_compact_refusals():
    lib = _native.load()
    a = [FAKE, FAKE, FAKE, 10, 10, 0, 2, 1.0, None, 0, None, 1.0, None, 0.0, None, FAKE, FAKE, None, None, None]
    for i, v, word in ((0, None, b"compact_logits"), (1, None, b"compact_ids"), (2, None, b"request_offsets"),
                       (3, -1, b"capacity"), (4, -1, b"max_len"), (6, 0, b"batch"), (15, None, b"uniforms")):
        b = list(a)
        b[i] = v
        assert lib.gsp_sample_compact(*b) == _native.GSP_ERR_INVALID_ARGUMENT, i
        assert word in lib.gsp_last_error(), (i, lib.gsp_last_error())


def test_python_refuses_cpu_tensors():
    x, u = torch.zeros(2, 64), torch.zeros(2)
    with pytest.raises(ValueError, match="CUDA"):
        tr.sample_logits(x, uniforms=u)
    with pytest.raises(ValueError, match="CUDA"):
        tr.sample_compact_logits(torch.zeros(4, dtype=torch.int64), torch.zeros(4), torch.tensor([0, 2, 4]), uniforms=u)


@pytest.mark.parametrize("values, word", [
    ((float("nan"), 0, 1.0, 0.0), "temperature"), ((-1.0, 0, 1.0, 0.0), "temperature"),
    ((float("inf"), 0, 1.0, 0.0), "temperature"), ((1.0, 2.5, 1.0, 0.0), "top_k"),
    ((1.0, float("inf"), 1.0, 0.0), "top_k"),
    ((1.0, 0, float("nan"), 0.0), "top_p"), ((1.0, 0, 1.0, float("nan")), "min_p"),
    ((torch.ones(3), 0, 1.0, 0.0), "temperature"), ((1.0, torch.ones(2), 1.0, 0.0), "top_k"),
    ((1.0, 0, torch.ones(4)[::2], 0.0), "top_p"),
])
def test_settings_refused(values, word):
    with pytest.raises(ValueError, match=word):
        tr._sample_settings(values, torch.zeros(2), torch.device("cpu"))


def test_uniforms_refused():
    for u in (torch.zeros(2, dtype=torch.float64), torch.zeros(2, 1), torch.zeros(4)[::2]):
        with pytest.raises(ValueError, match="uniforms"):
            tr._sample_settings((1.0, 0, 1.0, 0.0), u, torch.device("cpu"))
