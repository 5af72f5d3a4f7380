"""Sampling's checks of arguments, on the host (nothing is launched)."""

import ctypes
import inspect

import pytest
import torch


def test_python_refusals():
    from intel_kivi_hybrid_amd import _C
    x, u = torch.randn(2, 10), torch.rand(2)
    with pytest.raises(RuntimeError, match="logits must be a .rows, vocab. tensor"):
        _C.sample(x, u)
    with pytest.raises(RuntimeError, match="logits must be"):
        _C.sample(x.long(), u)
    with pytest.raises(RuntimeError, match="logits must be"):
        _C.sample([[0.0]], u)


def test_entry_point_rejects_bad_arguments():
    from intel_kivi_hybrid_amd import _native
    lib = _native.load()
    buf = (ctypes.c_float * 64)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    need = lib.kivi_sample_workspace_size(3, 10)
    assert need > 0 and lib.kivi_sample_workspace_size(0, 10) == 0
    assert lib.kivi_sample_workspace_size(3, 0) == 0

    def sample(x=p, dtype=0, stride=10, rows=3, vocab=10, u=p, out=p, ws=p, ws_bytes=need):
        rc = lib.kivi_sample(x, dtype, stride, rows, vocab, u, 0, None, ctypes.c_double(1.0), None,
                             0, None, ctypes.c_double(1.0), None, ctypes.c_double(0.0), out, ws,
                             ws_bytes, None)
        assert rc == 1
        return _native.last_error()
    assert "dtype 3" in sample(dtype=3)
    assert "3 rows and 0 tokens" in sample(vocab=0)
    assert "tokens (1 to 1048576)" in sample(vocab=(1 << 20) + 1)
    assert "-1 rows" in sample(rows=-1)
    assert "row_stride -1" in sample(stride=-1)
    for name in ("x", "u", "out"):
        assert "null pointer" in sample(**{name: None})
    assert "workspace must" in sample(ws=None)
    assert "workspace must" in sample(ws=p + 8)
    assert "workspace must" in sample(ws_bytes=need - 1)
    assert "too many for one launch" in sample(rows=2 ** 31 - 1, vocab=1 << 20)


def test_sample_token_takes_the_cuts_as_options():
    from intel_kivi_hybrid_amd.generation import sample_token
    d = inspect.signature(sample_token).parameters
    assert d["top_p"].default is None and d["min_p"].default is None
    # greedy stays the argmax, whatever the cuts
    logits = torch.tensor([[0.1, 3.0, -1.0, 2.9], [5.0, 0.0, 0.0, 0.0]])
    assert sample_token(logits, 1.0, None, False, top_p=0.1, min_p=0.5).tolist() == [[1], [0]]
    # and what it drew without them, it draws still
    torch.manual_seed(3)
    got = sample_token(logits, 0.7, 2, True)
    torch.manual_seed(3)
    scaled = logits / 0.7
    kth = scaled.topk(2, dim=-1).values[:, -1:]
    scaled = scaled.masked_fill(scaled < kth, float("-inf"))
    assert torch.equal(got, torch.multinomial(torch.softmax(scaled, dim=-1), num_samples=1))
