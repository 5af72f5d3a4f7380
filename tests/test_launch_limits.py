"""CPU tests: more workgroups than a launch takes are refused before anything is
launched."""

import ctypes

import pytest


def _buffer():
    buf = (ctypes.c_float * 64)()
    return buf, (ctypes.addressof(buf) + 15) // 16 * 16


@pytest.mark.parametrize("rows,vocab", [(1 << 22, 10), (1 << 20, 9 * 8192), (1 << 23, 1)])
def test_sampling(rows, vocab):
    from intel_kivi_hybrid_amd import _native
    lib = _native.load()
    buf, p = _buffer()

    def sample(rows, ws):
        rc = lib.kivi_sample(p, 0, 0, rows, vocab, p, 0, None, ctypes.c_double(1.0), None, 0, None,
                             ctypes.c_double(1.0), None, ctypes.c_double(0.0), p, ws, 0, None)
        assert rc == 1
        return _native.last_error()
    assert "too many for one launch" in sample(rows, None)
    assert "workspace must" in sample(rows // 4, None)


@pytest.mark.parametrize("words,text", [({6: 1 << 21}, "items"), ({9: 1 << 21}, "items"),
                                        ({5: 1 << 21}, "tiles to merge")])
def test_attention(words, text):
    from intel_kivi_hybrid_amd import _native
    lib = _native.load()
    buf, p = _buffer()
    info = (ctypes.c_int64 * 16)()
    info[1] = 1
    for i, v in words.items():
        info[i] = v
    if 5 in words:
        info[11] = 1                                  # (rows of a partial)
    rc = lib.kivi_paged_attention(p, 64, 64, 1, p, p, 4, 32, 8, 8, 64, p, ctypes.addressof(info),
                                  ctypes.c_float(0.1), p, None, 0, None)
    assert rc == 1 and text in _native.last_error() and "one launch" in _native.last_error()
