"""Refusals of token_logprobs, at the C ABI and in Python, before any device work (no kernel is launched)."""
import ctypes

import pytest
import torch

from gsp import _native
from gsp import logprobs as L

FAKE = ctypes.c_void_p(4096)  # never dereferenced: every call below fails validation first


def test_c_refusals():
    lib = _native.load()

    def forward(**kw):
        a = dict(x=FAKE, xs=64, dtype=0, mask=None, ms=0, batch=2, vocab=64, t=1.0, ts=None, ids=FAKE, tokens=1,
                 top_n=1, lp=FAKE, en=None, ls=None, ti=FAKE, tl=FAKE, st=None)
        a.update(kw)
        return lib.gsp_token_logprobs(*a.values(), None)

    for kw, word in (({"x": None}, b"logits"), ({"batch": 0}, b"batch"), ({"vocab": 0}, b"vocab"), ({"xs": -1}, b"stride"),
                     ({"mask": FAKE, "ms": 1}, b"bitmask"), ({"t": 0.0}, b"temperature"), ({"t": float("nan")}, b"temperature"),
                     ({"ids": None}, b"token_ids"), ({"tokens": 1025}, b"tokens"), ({"tokens": -1}, b"tokens"),
                     ({"top_n": 65}, b"top_n"), ({"lp": None}, b"logprobs"), ({"ti": None}, b"top_ids"),
                     ({"st": ctypes.c_void_p(4100)}, b"stats")):
        assert forward(**kw) == _native.GSP_ERR_INVALID_ARGUMENT, kw
        assert word in lib.gsp_last_error(), (kw, lib.gsp_last_error())
    assert forward(dtype=3) == _native.GSP_ERR_UNSUPPORTED
    assert forward(vocab=(1 << 30) + 1, xs=1 << 31) == _native.GSP_ERR_UNSUPPORTED

    def compact(**kw):
        a = dict(x=FAKE, ids=FAKE, off=FAKE, cap=10, ml=5, dtype=0, batch=2, t=1.0, ts=None, tok=FAKE, tokens=1, top_n=0,
                 lp=FAKE, en=None, ls=None, ti=None, tl=None)
        a.update(kw)
        return lib.gsp_token_logprobs_compact(*a.values(), None)

    for kw, word in (({"off": None}, b"request_offsets"), ({"x": None}, b"compact_logits"), ({"cap": -1}, b"capacity"),
                     ({"ml": -1}, b"max_len"), ({"batch": 0}, b"batch")):
        assert compact(**kw) == _native.GSP_ERR_INVALID_ARGUMENT, kw
        assert word in lib.gsp_last_error(), (kw, lib.gsp_last_error())

    def grad(**kw):
        a = dict(x=FAKE, xs=64, dtype=0, mask=None, ms=0, batch=2, vocab=64, ids=FAKE, tokens=1, st=FAKE, g=FAKE, gh=None,
                 gl=None, out=FAKE, os=64)
        a.update(kw)
        return lib.gsp_token_logprobs_grad(*a.values(), None)

    for kw, word in (({"st": None}, b"stats"), ({"out": None}, b"grad_logits"), ({"os": 32}, b"grad_row_stride"),
                     ({"x": None}, b"logits"), ({"st": ctypes.c_void_p(4100)}, b"stats")):
        assert grad(**kw) == _native.GSP_ERR_INVALID_ARGUMENT, kw
        assert word in lib.gsp_last_error(), (kw, lib.gsp_last_error())


def test_python_refuses_cpu_tensors():
    x, ids = torch.zeros(2, 64), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        L.token_logprobs(x, ids)
    with pytest.raises(ValueError, match="CUDA"):
        L.compact_token_logprobs(ids, x[:, 0].contiguous(), torch.tensor([0, 1, 2]), ids)
