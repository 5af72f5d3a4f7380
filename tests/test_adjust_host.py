"""CPU tests of what kivi_adjust_logits refuses before anything is launched."""

import ctypes

import torch


def _call(rows=2, vocab=8, dtype=0, out_dtype=0, n_tokens=0, biases=0, logits=None, out=None,
          stride=8, out_stride=8, tokens=None):
    from intel_kivi_hybrid_amd import _native
    lib = _native.load()
    f = ctypes.c_float
    buf = (ctypes.c_float * 256)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    rc = lib.kivi_adjust_logits(p if logits is None else p + logits, dtype, stride, rows, vocab,
                                tokens, 0, 0, n_tokens, None, 0, None, 0, None, f(1.0), None, f(0.0),
                                None, f(0.0), None, 0, 0, None, 0, biases, None, 0,
                                p + 512 if out is None else p + out, out_dtype, out_stride, None)
    return rc, _native.last_error() if rc else ""


def test_refusals():
    assert _call(rows=0) == (0, "")
    for kw, text in ((dict(dtype=3), "dtype 3"), (dict(dtype=1, out_dtype=2), "out_dtype 2"),
                     (dict(out_dtype=1), "out_dtype 1"), (dict(vocab=0), "2 rows of 0 tokens"),
                     (dict(rows=-1), "-1 rows"), (dict(n_tokens=-1), "-1 tokens"),
                     (dict(n_tokens=(1 << 30) + 1), "at most 1073741824"),
                     (dict(biases=(1 << 30) + 1), "at most 1073741824"),
                     (dict(n_tokens=1), "null pointer"), (dict(biases=1), "null pointer"),
                     (dict(logits=2), "aligned"), (dict(out=514), "aligned"),
                     (dict(out=4), "apart from them"), (dict(out=0, out_stride=9), "apart from them"),
                     (dict(out=0, dtype=1), "apart from them"),
                     (dict(out_stride=7), "rows of out overlap"),
                     (dict(rows=1 << 20, vocab=1 << 20, stride=0, out_stride=1 << 20, out=1 << 44),
                      "too many for one launch")):
        rc, message = _call(**kw)
        assert rc == 1 and text in message, (kw, message)


def test_words_of_a_mask():
    from intel_kivi_hybrid_amd import _C
    mask = torch.zeros(2, 40, dtype=torch.bool)
    mask[0, [0, 31, 32, 39]] = True
    words = _C.allowed_tokens(mask)
    assert words.dtype is torch.int32 and words.shape == (2, 2)
    bits = [[(int(w) >> b) & 1 for w in row for b in range(32)][:40] for row in words.tolist()]
    assert torch.equal(torch.tensor(bits, dtype=torch.bool), mask)
