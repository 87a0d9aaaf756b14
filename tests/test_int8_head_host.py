"""Refusals of the int8 head, at the C ABI and in Python, before any device work (no kernel is launched)."""
import ctypes

import pytest
import torch

from gsp import _native
from gsp import int8_head as I

FAKE = ctypes.c_void_p(4096)  # never dereferenced: every call below fails validation first


def _logits(**kw):
    a = dict(route=0, h=FAKE, hs=64, hd=0, hsc=None, w=FAKE, ws=64, wsc=FAKE, mask=None, ms=0, batch=2, vocab=64,
             hdim=64, od=0, off=0, logits=None, ls=64, tv=None, ti=None, tk=None, sc=FAKE, scb=1 << 20, wsp=FAKE,
             wsb=1 << 30)
    a.update(kw)
    return _native.load().gsp_int8_logits(*a.values(), None)


def test_int8_logits_refusals():
    lib = _native.load()
    for kw, word in (({"route": 3}, b"route"), ({"h": None}, b"non-null"), ({"w": None}, b"non-null"),
                     ({"wsc": None}, b"weight_scales"), ({"batch": 0}, b"positive"), ({"hd": 3}, b"hidden_scales"),
                     ({"hs": 32}, b"hidden_row_stride"), ({"ws": 32}, b"weight_row_stride"),
                     ({"logits": FAKE, "ls": 32}, b"logits_row_stride"),
                     ({"mask": FAKE, "ms": 1}, b"bitmask_row_stride")):
        assert _logits(**kw) == _native.GSP_ERR_INVALID_ARGUMENT, kw
        assert word in lib.gsp_last_error(), (kw, lib.gsp_last_error())
    for kw, word in (({"hd": 5}, b"hidden_dtype"), ({"od": 3}, b"dtype"),
                     ({"hdim": 131072, "hs": 131072, "ws": 131072}, b"overflow")):
        assert _logits(**kw) == _native.GSP_ERR_UNSUPPORTED, kw
        assert word in lib.gsp_last_error()
    for kw, word in (({"sc": None}, b"scratch"), ({"scb": 64}, b"scratch"), ({"sc": ctypes.c_void_p(4100)}, b"aligned"),
                     ({"route": 1, "wsp": None}, b"workspace"), ({"tv": FAKE, "wsb": 1}, b"workspace")):
        assert _logits(**kw) == _native.GSP_ERR_WORKSPACE, kw
        assert word in lib.gsp_last_error()


def test_int8_compact_and_quantize_refusals():
    lib = _native.load()
    a = [FAKE, 64, 0, None, FAKE, 64, FAKE, FAKE, 2, 2, 64, 64, 0, 0, FAKE, FAKE, 8, FAKE, None, None, None, FAKE,
         1 << 20, None, 0, None]

    def compact(**at):
        b = list(a)
        for i, v in at.items():
            b[int(i[1:])] = v
        return lib.gsp_int8_compact(*b)

    assert compact(_16=-1) == _native.GSP_ERR_INVALID_ARGUMENT and b"capacity" in lib.gsp_last_error()
    assert compact(_14=None) == _native.GSP_ERR_INVALID_ARGUMENT and b"compact_logits" in lib.gsp_last_error()
    assert compact(_17=None) == _native.GSP_ERR_INVALID_ARGUMENT and b"request_offsets" in lib.gsp_last_error()
    assert compact(_18=FAKE) == _native.GSP_ERR_WORKSPACE
    q = lib.gsp_quantize_rows_int8
    assert q(FAKE, 8, -1, 8, 0, FAKE, 8, FAKE, None) == _native.GSP_ERR_INVALID_ARGUMENT
    assert q(FAKE, 8, 4, 0, 0, FAKE, 8, FAKE, None) == _native.GSP_ERR_INVALID_ARGUMENT
    assert q(FAKE, 8, 4, 8, 3, FAKE, 8, FAKE, None) == _native.GSP_ERR_UNSUPPORTED
    assert q(None, 8, 4, 8, 0, FAKE, 8, FAKE, None) == _native.GSP_ERR_INVALID_ARGUMENT
    assert q(FAKE, 8, 4, 8, 0, FAKE, 4, FAKE, None) == _native.GSP_ERR_INVALID_ARGUMENT
    assert q(FAKE, 8, 1 << 31, 8, 0, FAKE, 8, FAKE, None) == _native.GSP_ERR_UNSUPPORTED
    assert q(FAKE, 8, 1, (1 << 30) + 1, 0, FAKE, 8, FAKE, None) == _native.GSP_ERR_UNSUPPORTED
    assert q(None, 8, 0, 8, 0, None, 8, None, None) == _native.GSP_OK  # no rows: nothing to do
    assert lib.gsp_int8_scratch_bytes(0, 8) == 0 and lib.gsp_int8_scratch_bytes(3, 100) >= 3 * (112 + 4)


def test_python_refuses_cpu_tensors_and_bad_operands():
    h = torch.zeros(2, 64, dtype=torch.float16)
    w = I.QuantizedRows(torch.zeros(96, 64, dtype=torch.int8), torch.zeros(96))
    m = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        I.quantize_rows_int8(h)
    with pytest.raises(ValueError, match="CUDA"):
        I.int8_grammar_logits(h, w, m)
    with pytest.raises(ValueError, match="CUDA"):
        I.int8_compact_logits(h, w, m)
    with pytest.raises(ValueError, match="route"):
        I.int8_grammar_logits(h, w, m, route="no-such-route")
    with pytest.raises(ValueError, match="bitmask_gpu"):
        I.int8_compact_logits(h, w, None)
