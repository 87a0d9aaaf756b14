"""The fp8 head refuses vocabularies whose legal rows it could not count, at the C ABI, before any device work."""
import ctypes

from gsp import _native

FAKE = ctypes.c_void_p(4096)  # never dereferenced: every call below fails validation first


def test_vocabularies_above_two_to_the_30():
    lib = _native.load()

    def logits(vocab, scratch_bytes):
        return lib.gsp_fp8_logits(0, FAKE, 16, 0, None, 0, FAKE, 16, FAKE, 1, None, 0, 1, vocab, 16, 0, 0, None, vocab, None, FAKE,
                                  None, FAKE, scratch_bytes, None)

    for vocab in (2 ** 30 + 1, 2 ** 31 - 32, 2 ** 31 - 1):
        assert logits(vocab, 1 << 40) == _native.GSP_ERR_UNSUPPORTED, vocab
    assert b"2^3" in lib.gsp_last_error()
    assert logits(2 ** 30, 64) == _native.GSP_ERR_WORKSPACE  # (its size is taken)
