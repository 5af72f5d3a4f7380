"""CPU tests of the paged cache's plan: what it says against a restatement,
and what it refuses (kivi_paged_plan, include/kivi_hip.h)."""

import ctypes

import numpy as np
import pytest
import torch

from tests.paged_helpers import make_table, slots_of

DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _plan(table, pool, ctx, new, page_size=32, dtype=torch.bfloat16, Hq=8, Hkv=2, D=64,
          expect=0):
    from intel_kivi_hybrid_amd import _native
    lib = _native.load()
    info = np.zeros(16, dtype=np.int64)
    c, n = np.asarray(ctx, dtype=np.int32), np.asarray(new, dtype=np.int32)
    t = table.numpy()
    args = (len(ctx), n.ctypes.data, c.ctypes.data, t.ctypes.data, t.shape[1], t.shape[1],
            page_size, pool, DT.get(dtype, dtype), Hq, Hkv, D)
    rc = lib.kivi_paged_plan(*args, None, 0, info.ctypes.data)
    assert rc == expect, _native.last_error()
    if expect:
        return _native.last_error()
    words = np.full(int(info[0]) + 8, -77, dtype=np.int32)
    assert lib.kivi_paged_plan(*args, words.ctypes.data, int(info[0]), info.ctypes.data) == 0
    assert (words[int(info[0]):] == -77).all()
    if info[0]:
        assert lib.kivi_paged_plan(*args, words.ctypes.data, int(info[0]) - 1,
                                   info.ctypes.data) == 1
    return words[:int(info[0])], info


LENS = [
    [(0, 1)],
    [(1020, 1)],
    [(5, 3), (0, 7), (100, 1), (63, 0), (31, 1)],
    [(0, 300), (0, 33), (9000, 2), (8191, 1)],
    [(8200, 2048)],
    [(4000 + 37 * i, 1) for i in range(64)],
    [(100000, 1), (3, 1), (17, 200)],
]


@pytest.mark.parametrize("lens", LENS, ids=range(len(LENS)))
@pytest.mark.parametrize("dtype,Hq,Hkv,D", [(torch.bfloat16, 32, 8, 128), (torch.float16, 12, 12, 64),
                                            (torch.float32, 6, 2, 128), (torch.bfloat16, 20, 1, 256)])
def test_plan_covers_every_token_and_pair_once(lens, dtype, Hq, Hkv, D):
    page_size = 32
    table, pool, ctx, new = make_table(lens, page_size, seed=3)
    words, info = _plan(table, pool, ctx, new, page_size, dtype, Hq, Hkv, D)
    T, hg = sum(new), Hq // Hkv
    assert info[1] == T and info[12] == max([c for c, n in zip(ctx, new) if n] + [0])
    # tokens: slot and position
    tokens = words[:2 * T].reshape(T, 2)
    want = [(p * page_size + o, pos) for p, o, pos in slots_of(table, ctx, new, page_size)]
    assert tokens.tolist() == [list(x) for x in want]
    # items: every (row, position it sees) exactly once
    pages_at, items_at, merges_at = int(info[2]), int(info[3]), int(info[4])
    assert items_at % 8 == 0
    n_items = int(info[6:10].sum())
    items = words[items_at:items_at + 8 * n_items].reshape(n_items, 8)
    merges = words[merges_at:merges_at + 8 * int(info[5])].reshape(-1, 8)
    kinds = np.repeat(np.arange(4), info[6:10])
    tile_rows = np.array([16, 32, 64, 128])[kinds]
    first = np.cumsum([0] + new)
    seen = {}
    parts = []
    for it, rows, kind in zip(items, tile_rows, kinds):
        tok0, n, c, page0, row0, b, e, part = it.tolist()
        s = [i for i in range(len(ctx)) if first[i] == tok0 and new[i] > 0][0]
        assert n == new[s] and c == ctx[s] and row0 % rows == 0 and row0 < n * hg
        assert dtype != torch.float32 or kind != 3
        np_ = -(-c // page_size)
        assert words[pages_at + page0:pages_at + page0 + np_].tolist() == table[s, :np_].tolist()
        assert 0 <= b < e <= c and b % 64 == 0
        seen.setdefault((s, row0, int(rows)), []).append((b, e, part))
        if part >= 0:
            parts.append(part)
    assert sorted(parts) == list(range(int(info[10])))
    merged = {}
    for tok0, n, row0, splits, part, rows, _, _ in merges.tolist():
        assert splits > 1 and rows <= info[11]
        merged[(tok0, row0)] = list(range(part, part + splits))
    for s in range(len(ctx)):
        rows = new[s] * hg
        covered = 0
        for (q, row0, tile), spans in sorted(seen.items()):
            if q != s:
                continue
            assert row0 == covered
            covered = min(rows, row0 + tile)
            spans.sort()
            assert spans[0][0] == 0 and all(x[1] == y[0] for x, y in zip(spans, spans[1:]))
            # the last position that the tile's last row sees
            assert spans[-1][1] == ctx[s] - new[s] + (covered - 1) // hg + 1
            ids = [p for _, _, p in spans]
            assert ids == ([-1] if len(spans) == 1 else merged.pop((int(first[s]), row0)))
        assert covered == rows
    assert not merged


def test_plan_of_nothing():
    table = torch.full((2, 3), -1, dtype=torch.int32)
    words, info = _plan(table, 4, [0, 40], [0, 0])
    assert len(words) == 0 and info[1] == 0 and info[6:10].sum() == 0
    words, info = _plan(torch.zeros(0, 1, dtype=torch.int32), 4, [], [])
    assert info[1] == 0


def test_plan_refusals():
    table = torch.tensor([[0, 1, 2], [3, 4, 9]], dtype=torch.int32)
    ok = dict(page_size=32, dtype=torch.bfloat16, Hq=8, Hkv=2, D=64)
    assert "page 9 outside the pool of 9" in _plan(table, 9, [70, 96], [70, 1], **ok, expect=1)
    assert "page -1 outside" in _plan(torch.tensor([[-1]], dtype=torch.int32), 9, [3], [3], **ok,
                                      expect=1)
    # (a page that no position reaches is not looked at)
    _plan(table, 9, [70, 64], [70, 1], **ok)
    assert "needs 4 pages, the table has 3" in _plan(table, 10, [97, 5], [1, 1], **ok, expect=1)
    assert "5 new tokens in a context of 4" in _plan(table, 10, [4, 5], [5, 1], **ok, expect=1)
    assert "-1 new tokens" in _plan(table, 10, [4, 5], [-1, 1], **ok, expect=1)
    twice = torch.tensor([[0, 1], [2, 1]], dtype=torch.int32)
    assert "page 1: a slot is given to two" in _plan(twice, 10, [40, 40], [5, 6], **ok, expect=1)
    assert "page 1: a slot" in _plan(torch.tensor([[1, 1]], dtype=torch.int32), 10, [40], [40],
                                     **ok, expect=1)
    # a shared prefix, and disjoint stretches of one page, are fine
    _plan(torch.tensor([[0, 1], [0, 2]], dtype=torch.int32), 10, [40, 40], [5, 6], **ok)
    _plan(twice, 10, [40, 44], [8, 4], **ok)
    one = torch.zeros(1, 1, dtype=torch.int32)
    for kw, text in ((dict(page_size=48), "page_size"), (dict(page_size=8), "page_size"),
                     (dict(dtype=3), "dtype 3"), (dict(Hq=7), "multiple of kv_heads"),
                     (dict(Hkv=0), "kv_heads")):
        assert text in _plan(one, 10, [4], [4], **{**ok, **kw}, expect=1)
    for D in (8, 72, 272):
        assert "head_dim" in _plan(one, 10, [4], [4], **{**ok, "D": D}, expect=4)
    assert "num_pages" in _plan(one, 0, [4], [4], **ok, expect=1)
    assert "num_pages" in _plan(one, 1 << 27, [4], [4], **ok, expect=1)


def test_python_plan_refusals():
    from intel_kivi_hybrid_amd import _C
    t = torch.zeros(1, 2, dtype=torch.int32)
    kw = dict(page_size=32, num_pages=4, q_heads=8, kv_heads=2, head_dim=64)
    with pytest.raises(RuntimeError, match="page_table must be an int32"):
        _C.paged_plan(t.long(), [4], [4], **kw)
    with pytest.raises(RuntimeError, match="one entry for each of the table's 1"):
        _C.paged_plan(t, [4, 5], [4, 4], **kw)
    with pytest.raises(RuntimeError, match=r"context_lens must lie in \[0, 2\^31\)"):
        _C.paged_plan(t, [1 << 32], [4], **kw)
    with pytest.raises(RuntimeError, match="new_lens must hold one int"):
        _C.paged_plan(t, [4], [4.0], **kw)
    with pytest.raises(RuntimeError, match="device must be on cuda but got cpu"):
        _C.paged_plan(t, [4], [4], device="cpu", **kw)
    with pytest.raises(RuntimeError, match="dtype must be float32, bfloat16 or float16, got Long"):
        _C.paged_plan(t, [4], [4], dtype=torch.int64, **kw)
    with pytest.raises(TypeError, match="page_size must be an int"):
        _C.paged_plan(t, [4], [4], **{**kw, "page_size": 32.0})
    with pytest.raises(RuntimeError, match="page 0: a slot is given to two new tokens"):
        _C.paged_plan(t, [64], [64], **kw)


def test_attention_and_append_entry_points_reject_bad_arguments():
    from intel_kivi_hybrid_amd import _native
    lib = _native.load()
    buf = (ctypes.c_float * 64)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    info = (ctypes.c_int64 * 16)()
    info[1] = 1
    ip = ctypes.addressof(info)

    def attend(q=p, st=64, dtype=1, pages=4, page=32, Hq=4, Hkv=2, D=64, scale=0.1, ws=None):
        rc = lib.kivi_paged_attention(q, st, 64, dtype, p, p, pages, page, Hq, Hkv, D, p, ip,
                                      ctypes.c_float(scale), p, ws, 0, None)
        assert rc == 1
        return _native.last_error()
    assert "dtype 5" in attend(dtype=5)
    assert "page_size 40" in attend(page=40)
    assert "head_dim 24" in attend(D=24)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert "softmax_scale must be positive" in attend(scale=scale)
    assert "16-byte aligned" in attend(q=p + 4)
    assert "16-byte aligned" in attend(st=68)
    assert "null pointer" in attend(q=None)
    info[10], info[11] = 2, 16
    assert "workspace must hold" in attend()

    def append(k=p, dtype=1, rot=0, cos=None, tokens=1, q=None, q_out=None, kp=p, nd=1):
        rc = lib.kivi_paged_append(q, 0, 0, k, 0, 0, p, 0, 0, dtype, q_out, kp, p, 4, 32, 4, 2, 64,
                                   p, tokens, cos, cos, rot, 0, None, None, nd,
                                   ctypes.c_float(1e-6), None)
        assert rc == 1
        return _native.last_error()
    assert "rotary_dim must be a multiple of 16 up to head_dim, got 24" in append(rot=24)
    assert "got 80" in append(rot=80)
    assert "rotation needs cos and sin" in append(rot=32)
    assert "null pointer" in append(k=None)
    assert "null pointer" in append(q=p)
    assert "must not be negative" in append(tokens=-1)
    assert "16-byte aligned" in append(kp=p + 2)
    assert "norm_dtype 3" in append(nd=3)
