"""Refusals of the fp8 head and the norm, at the C ABI and in Python, before any device work (no kernel is launched)."""
import ctypes

import pytest
import torch

from gsp import _native
from gsp import fp8_head as F
from gsp import norm

FAKE = ctypes.c_void_p(4096)  # never dereferenced: every call below fails validation first


def _logits(**kw):
    a = dict(route=0, h=FAKE, hs=256, hd=0, hsc=None, hss=0, w=FAKE, ws=256, wsc=FAKE, wss=2, mask=None, ms=0, batch=2,
             vocab=300, hdim=256, od=0, off=0, logits=FAKE, ls=300, tv=None, ti=None, tk=None, sc=FAKE, scb=1 << 24)
    a.update(kw)
    return _native.load().gsp_fp8_logits(*a.values(), None)


def test_fp8_logits_refusals():
    lib = _native.load()
    for kw, word in (({"route": 3}, b"route"), ({"h": None}, b"non-null"), ({"w": None}, b"non-null"),
                     ({"wsc": None}, b"weight_scales"), ({"wss": 1}, b"weight_scales_row_stride"), ({"batch": 0}, b"positive"),
                     ({"hd": 4}, b"hidden_scales"), ({"hd": 4, "hsc": FAKE, "hss": 1}, b"hidden_scales_row_stride"),
                     ({"hs": 32}, b"hidden_row_stride"), ({"ws": 32}, b"weight_row_stride"), ({"ls": 32}, b"logits_row_stride"),
                     ({"mask": FAKE, "ms": 1}, b"bitmask_row_stride"), ({"logits": None}, b"output")):
        assert _logits(**kw) == _native.GSP_ERR_INVALID_ARGUMENT, kw
        assert word in lib.gsp_last_error(), (kw, lib.gsp_last_error())
    for kw, word in (({"hd": 3}, b"hidden_dtype"), ({"od": 3}, b"dtype"),
                     ({"hdim": 32896, "hs": 32896, "ws": 32896, "wss": 257}, b"hidden_dim")):
        assert _logits(**kw) == _native.GSP_ERR_UNSUPPORTED, kw
        assert word in lib.gsp_last_error()
    for kw in ({"sc": None}, {"scb": 64}, {"sc": ctypes.c_void_p(4100)}):
        assert _logits(**kw) == _native.GSP_ERR_WORKSPACE, kw
        assert b"scratch" in lib.gsp_last_error()
    assert lib.gsp_fp8_scratch_bytes(0, 8, 8) == 0 and lib.gsp_fp8_scratch_bytes(3, 5000, 100) >= 3 * (112 + 16) + 157 * 4


def test_quantise_and_norm_refusals():
    lib = _native.load()
    for q in (lib.gsp_quantize_rows_fp8, lib.gsp_quantize_weight_fp8):
        assert q(FAKE, 8, -1, 8, 0, FAKE, 8, FAKE, 1, None) == _native.GSP_ERR_INVALID_ARGUMENT
        assert q(FAKE, 8, 4, 0, 0, FAKE, 8, FAKE, 1, None) == _native.GSP_ERR_INVALID_ARGUMENT
        assert q(FAKE, 8, 4, 8, 3, FAKE, 8, FAKE, 1, None) == _native.GSP_ERR_UNSUPPORTED
        assert q(None, 8, 4, 8, 0, FAKE, 8, FAKE, 1, None) == _native.GSP_ERR_INVALID_ARGUMENT
        assert q(FAKE, 8, 4, 8, 0, FAKE, 4, FAKE, 1, None) == _native.GSP_ERR_INVALID_ARGUMENT
        assert q(FAKE, 256, 4, 256, 0, FAKE, 256, FAKE, 1, None) == _native.GSP_ERR_INVALID_ARGUMENT
        assert q(FAKE, 8, 1 << 31, 8, 0, FAKE, 8, FAKE, 1, None) == _native.GSP_ERR_UNSUPPORTED
        assert q(FAKE, 8, 1, (1 << 24) + 1, 0, FAKE, 8, FAKE, 1, None) == _native.GSP_ERR_UNSUPPORTED
        assert q(None, 8, 0, 8, 0, None, 8, None, 1, None) == _native.GSP_OK  # no rows: nothing to do

    def rms(**kw):
        a = dict(x=FAKE, xs=256, r=None, rs=0, w=None, rows=4, cols=256, eps=1e-6, dt=0, ro=None, ros=0, od=0, out=FAKE,
                 os=256, sc=None, ss=0)
        a.update(kw)
        return lib.gsp_rms_norm(*a.values(), None)

    for kw, word in (({"rows": -1}, b"rows"), ({"cols": 0}, b"cols"), ({"x": None}, b"required"), ({"out": None}, b"required"),
                     ({"eps": -1.0}, b"eps"), ({"eps": float("nan")}, b"eps"), ({"r": FAKE}, b"residual_out"),
                     ({"ro": FAKE}, b"residual"), ({"od": 3}, b"scales"), ({"od": 4}, b"scales"),
                     ({"od": 4, "sc": FAKE, "ss": 1}, b"stride"), ({"os": 8}, b"stride"), ({"xs": -1}, b"stride")):
        assert rms(**kw) == _native.GSP_ERR_INVALID_ARGUMENT, kw
        assert word in lib.gsp_last_error(), (kw, lib.gsp_last_error())
    for kw in ({"dt": 3}, {"od": 1}, {"rows": 1 << 31}, {"cols": (1 << 24) + 1}):
        assert rms(**kw) == _native.GSP_ERR_UNSUPPORTED, kw
    assert rms(rows=0, x=None, out=None) == _native.GSP_OK


def test_python_refuses_cpu_tensors():
    h = torch.zeros(2, 64, dtype=torch.float16)
    w = F.Fp8Weight(torch.zeros(96, 64).to(torch.float8_e4m3fn), torch.zeros(1, 1))
    for call in (lambda: F.quantize_rows_fp8(h), lambda: F.quantize_weight_fp8(h), lambda: F.fp8_grammar_logits(h, w, None),
                 lambda: norm.rms_norm(h)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
