"""CPU tests of the paged cache's limits: sizes at which the kernels' 32-bit
positions and rows would wrap, and workspaces by what is live."""

import ctypes

import numpy as np
import pytest
import torch

from tests.paged_helpers import make_table
from tests.test_paged_plan import _plan


def _info(table, pool, ctx, new, page_size, Hq, Hkv, D=16, dtype=1):
    from intel_kivi_hybrid_amd import _native
    lib = _native.load()
    info = np.zeros(16, dtype=np.int64)
    c, n = np.asarray(ctx, dtype=np.int32), np.asarray(new, dtype=np.int32)
    rc = lib.kivi_paged_plan(len(ctx), n.ctypes.data, c.ctypes.data, table.ctypes.data,
                             table.shape[1], table.shape[1], page_size, pool, dtype, Hq, Hkv, D,
                             None, 0, info.ctypes.data)
    return rc, (_native.last_error() if rc else info)


@pytest.mark.parametrize("dtype", [0, 1])
def test_contexts_whose_positions_would_wrap(dtype):
    """A sequence of one page many times (a table that repeats): the kernels look a
    few tiles past the end, in 32 bits."""
    table = np.zeros((1, 1 << 23), dtype=np.int32)
    longest = (1 << 31) - 4096
    table[0, (longest - 1) >> 8] = 1
    rc, info = _info(table, 2, [longest], [1], 256, 1, 1, dtype=dtype)
    assert rc == 0 and info[12] == longest
    for c in (longest + 1, (1 << 31) - 1):
        rc, text = _info(table, 2, [c], [1], 256, 1, 1, dtype=dtype)
        assert rc == 1 and "positions" in text


def test_rows_that_would_wrap():
    """Rows of a sequence and kv head (tokens x heads of its group) stay below
    2^31 - 4096: a tile's last rows may lie behind them."""
    table = np.arange(1 << 9, dtype=np.int32)[None]
    n = 1 << 16
    rc, text = _info(table, 1 << 9, [n], [n], 128, 1 << 15, 1)
    assert rc == 1 and "too large" in text
    rc, text = _info(table[:, :1], 1 << 9, [1], [1], 128, (1 << 31) - 1, 1)
    assert rc == 1 and "too large" in text


def test_workspace_follows_the_live_rows():
    """Eight single tokens of 32K positions beside a verification of five tokens:
    partials of 8 rows and of 40, not all of a tile of 128."""
    from intel_kivi_hybrid_amd import _native
    lens = [(32768, 1)] * 8 + [(32768, 5)]
    table, pool, ctx, new = make_table(lens, 256, seed=1)
    words, info = _plan(table, pool, ctx, new, 256, torch.bfloat16, 32, 4, 128)
    merges = words[info[4]:info[4] + 8 * info[5]].reshape(-1, 8)
    need = _native.load().kivi_paged_attention_workspace_size(info.ctypes.data, 4, 128)
    assert need == sum(m[3] * (8 if m[1] == 1 else 40) for m in merges) * 4 * 130 * 4 > 0
    # (partials of few rows come first)
    assert max(m[4] + m[3] for m in merges if m[1] == 1) == min(m[4] for m in merges if m[1] == 5)


def test_scales_whose_log2_units_overflow():
    from intel_kivi_hybrid_amd import _native
    lib = _native.load()
    buf = (ctypes.c_float * 64)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    info = (ctypes.c_int64 * 16)()
    info[1] = 1
    rc = lib.kivi_paged_attention(p, 64, 64, 1, p, p, 4, 32, 4, 2, 64, p, ctypes.addressof(info),
                                  ctypes.c_float(3e38), p, None, 0, None)
    assert rc == 1 and "softmax_scale must be positive" in _native.last_error()
