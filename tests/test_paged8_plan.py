"""CPU tests of the 8-bit paged cache's plan and of what its calls refuse
(kivi_paged8_*, include/kivi_hip.h)."""

import ctypes

import numpy as np
import pytest
import torch

from tests.paged_helpers import make_table, slots_of
from tests.test_paged_plan import DT, LENS
from tests.test_paged_plan import _plan as plain_plan


def _plan(table, pool, ctx, new, page_size=32, dtype=torch.bfloat16, Hq=8, Hkv=2, D=64, expect=0):
    from intel_kivi_hybrid_amd import _native
    lib = _native.load()
    info = np.full(20 + 4, -5, dtype=np.int64)
    c, n = np.asarray(ctx, dtype=np.int32), np.asarray(new, dtype=np.int32)
    t = table.numpy()
    args = (len(ctx), n.ctypes.data, c.ctypes.data, t.ctypes.data, t.shape[1], t.shape[1],
            page_size, pool, DT.get(dtype, dtype), Hq, Hkv, D)
    rc = lib.kivi_paged8_plan(*args, None, 0, info.ctypes.data)
    assert rc == expect, _native.last_error()
    if expect:
        return _native.last_error()
    assert (info[20:] == -5).all()
    words = np.full(int(info[0]) + 8, -77, dtype=np.int32)
    assert lib.kivi_paged8_plan(*args, words.ctypes.data, int(info[0]), info.ctypes.data) == 0
    assert (words[int(info[0]):] == -77).all()
    return words[:int(info[0])], info


@pytest.mark.parametrize("lens", LENS, ids=range(len(LENS)))
@pytest.mark.parametrize("page_size", [16, 64])
def test_blocks_hold_every_new_token_once(lens, page_size):
    table, pool, ctx, new = make_table(lens, page_size, seed=3)
    words, info = _plan(table, pool, ctx, new, page_size)
    blocks = words[info[16]:info[16] + 4 * info[17]].reshape(-1, 4)
    assert info[16] + 4 * info[17] == info[0]
    before = [c - n for c, n in zip(ctx, new) for _ in range(n)]
    slots = slots_of(table, ctx, new, page_size)
    got = []
    for slot, tok, first, packed in blocks.tolist():
        held, n = packed & 0xffff, packed >> 16
        assert first == slots[tok][2]
        assert slot % 16 == 0 and 0 <= held and n >= 1 and held + n <= 16
        for i in range(n):
            page, off, pos = slots[tok + i]
            assert page * page_size + off == slot + held + i
            # what a block held before: all of its positions below the first new one
            assert i or held == pos % 16 and (held == 0 or pos == before[tok])
            got.append(tok + i)
    assert got == list(range(sum(new)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_rest_is_the_plan_of_16_bit_pages_where_costs_agree(dtype):
    table, pool, ctx, new = make_table(LENS[2], 32, seed=3)
    words, info = _plan(table, pool, ctx, new, dtype=dtype)
    plain, plain_info = plain_plan(table, pool, ctx, new, dtype=dtype)
    assert (words[2 * sum(new):len(plain)] == plain[2 * sum(new):]).all()
    assert info[1:16].tolist() == plain_info[1:].tolist()


def test_fp32_rows_go_into_the_tiles_of_the_16_bit_types():
    table, pool, ctx, new = make_table([(40, 50), (7, 1)], 32, seed=3)
    info = _plan(table, pool, ctx, new, dtype=torch.float32)[1]
    assert info[8] == 0 and info[9] > 0


@pytest.mark.parametrize("lens,dtype,dim,wide", [
    ([(8200, 2048)], torch.bfloat16, 128, True), ([(8200, 2048)], torch.float32, 128, False),
    ([(8200, 2048)], torch.float16, 64, False), ([(8200, 2048), (700, 1)], torch.float16, 128, False),
    ([(100, 256)], torch.bfloat16, 128, False), ([(30000, 100)] * 2, torch.float16, 112, True)])
def test_long_chunks_of_128_channels_are_in_tiles_of_256_rows(lens, dtype, dim, wide):
    """Unless sequences of few rows are beside them."""
    table, pool, ctx, new = make_table(lens, 64, seed=3)
    info = _plan(table, pool, ctx, new, 64, dtype, 32, 8, dim)[1]
    assert (info[8] > 0) == wide and (info[9] > 0) == (not wide)


@pytest.mark.parametrize("lens,dtype", [([(8200, 2048)], torch.bfloat16),
                                        ([(40, 50)], torch.float32)])
def test_pages_of_the_models_type_refuse_tiles_that_they_do_not_have(lens, dtype):
    from intel_kivi_hybrid_amd import _native
    lib = _native.load()
    table, pool, ctx, new = make_table(lens, 64, seed=3)
    words, info = _plan(table, pool, ctx, new, 64, dtype, 32, 8, 128)
    size = lib.kivi_paged_attention_workspace_size(info.ctypes.data, 8, 128)
    buf = (ctypes.c_float * 64)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    rc = lib.kivi_paged_attention(p, 4096, 128, DT[dtype], p, p, pool, 64, 32, 8, 128, p,
                                  info.ctypes.data, ctypes.c_float(0.1), p, p, size, None)
    assert rc == 1 and "not one of kivi_paged_plan" in _native.last_error()


def test_a_block_of_two_sequences_is_refused():
    """Disjoint slots of one page are fine in pages of the model's type; here each
    sequence would rescale the other's tokens."""
    twice = torch.tensor([[0, 1], [2, 1]], dtype=torch.int32)
    text = _plan(twice, 10, [40, 44], [8, 4], expect=1)
    assert "page 1: a block of 16 positions is given to two sequences" in text
    _plan(twice, 10, [48, 52], [8, 4])                     # (blocks 0 and 1 of page 1)
    assert "a slot is given to two" in _plan(twice, 10, [40, 40], [5, 6], expect=1)


def test_refusals_are_those_of_the_other_plan():
    one = torch.zeros(1, 1, dtype=torch.int32)
    assert "page_size" in _plan(one, 10, [4], [4], page_size=48, expect=1)
    assert "head_dim" in _plan(one, 10, [4], [4], D=72, expect=4)
    assert "outside the pool" in _plan(one + 12, 10, [4], [4], expect=1)


def test_entry_points_reject_bad_arguments():
    from intel_kivi_hybrid_amd import _native
    lib = _native.load()
    buf = (ctypes.c_float * 64)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    info = (ctypes.c_int64 * 20)()
    info[1] = 1
    ip = ctypes.addressof(info)

    def attend(q=p, ks=p, dtype=1, page=32, scale=0.1):
        rc = lib.kivi_paged8_attention(q, 64, 64, dtype, p, p, ks, p, 4, page, 4, 2, 64, p, ip,
                                       ctypes.c_float(scale), p, None, 0, None)
        assert rc == 1
        return _native.last_error()
    assert "dtype 5" in attend(dtype=5)
    assert "page_size 40" in attend(page=40)
    assert "softmax_scale must be positive" in attend(scale=-1.0)
    assert "null pointer" in attend(q=None)
    assert "null scales" in attend(ks=None)
    info[8] = 1                                  # (tiles of 256 rows: 16 bits, 128 channels)
    assert "not one of kivi_paged8_plan" in attend(dtype=0)
    assert "not one of kivi_paged8_plan" in attend()
    info[8] = 0
    info[6] = 1 << 24
    assert "too many for one launch" in attend()
    info[6] = 0

    def append(k=p, ks=p, rot=0, blocks=1, info_p=ip):
        info[17] = blocks
        rc = lib.kivi_paged8_append(None, 0, 0, k, 0, 0, p, 0, 0, 1, None, p, p, ks, p, 4, 32, 4,
                                    2, 64, p, info_p, None, None, rot, 0, None, None, 1,
                                    ctypes.c_float(1e-6), None)
        assert rc == 1
        return _native.last_error()
    assert "null plan info" in append(info_p=None)
    assert "null pointer" in append(k=None)
    assert "null scales" in append(ks=None)
    assert "rotation needs cos and sin" in append(rot=32)
    assert "too many for one launch" in append(blocks=1 << 24)


@pytest.mark.parametrize("lens,dtype,Hq,Hkv,D,per_cu", [
    ([(20000, 64)], torch.float32, 32, 8, 128, 1), ([(8000, 200)], torch.float32, 16, 4, 96, 1),
    ([(8000, 200)], torch.float32, 8, 2, 64, 2), ([(20000, 64)], torch.float16, 32, 8, 64, 3),
    ([(20000, 64)], torch.bfloat16, 32, 8, 128, 2), ([(3000, 1)] * 16, torch.float32, 28, 4, 256, 2),
    ([(3000, 1)] * 16, torch.bfloat16, 12, 12, 64, 3)])
def test_contexts_are_split_for_the_workgroups_that_a_cu_holds(lens, dtype, Hq, Hkv, D, per_cu):
    """So many pieces that most of them run at once, and none behind them."""
    table, pool, ctx, new = make_table(lens, 64, seed=3)
    info = _plan(table, pool, ctx, new, 64, dtype, Hq, Hkv, D)[1]
    assert 256 * (per_cu - 1) < info[6:10].sum() * Hkv <= 256 * per_cu


@pytest.mark.parametrize("lens", LENS, ids=range(len(LENS)))
def test_entry_points_refuse_plans_of_the_models_type(lens):
    """Whose info ends before the blocks of 8-bit pages: nothing behind it is read."""
    from intel_kivi_hybrid_amd import _native
    lib = _native.load()
    table, pool, ctx, new = make_table(lens, 32, seed=3)
    words, plain = plain_plan(table, pool, ctx, new)
    info = np.full(20, 1 << 40, dtype=np.int64)
    info[:16] = plain[:16]
    buf = (ctypes.c_float * 64)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    ip = info.ctypes.data
    calls = (lambda: lib.kivi_paged8_append(
        None, 0, 0, p, 0, 0, p, 0, 0, 1, None, p, p, p, p, pool, 32, 8, 2, 64, p, ip, None, None,
        0, 0, None, None, 1, ctypes.c_float(1e-6), None),
        lambda: lib.kivi_paged8_attention(p, 512, 64, 1, p, p, p, p, pool, 32, 8, 2, 64, p, ip,
                                          ctypes.c_float(0.1), p, p, 1 << 40, None))
    for call in calls:
        assert call() == 1 and "not one of kivi_paged8_plan" in _native.last_error()


def test_python_plan_refuses_other_cache_types():
    from intel_kivi_hybrid_amd import _C
    t = torch.zeros(1, 2, dtype=torch.int32)
    kw = dict(page_size=32, num_pages=4, q_heads=8, kv_heads=2, head_dim=64)
    for dt in (torch.uint8, torch.float32):
        with pytest.raises(RuntimeError, match="cache_dtype must be BFloat16 or int8"):
            _C.paged_plan(t, [4], [4], cache_dtype=dt, **kw)
