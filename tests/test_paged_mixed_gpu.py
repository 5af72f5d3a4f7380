"""GPU tests of steps that mix single tokens with sequences of many rows: in one
launch, and as two kinds of tiles whose contexts are split."""

import pytest
import torch

from tests.test_paged_gpu import _attend, _check, _setup

pytestmark = pytest.mark.gpu
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("lens,page,Hq,Hkv,D", [
    ([(5000, 1), (300, 30), (2000, 2)], 64, 16, 16, 256),
    ([(3000, 1), (9000, 3), (1500, 70), (20, 1)], 32, 24, 12, 128),
    ([(4000, 1), (4000, 40)], 16, 80, 40, 64),
])
def test_two_kinds_of_tiles_with_split_contexts(hip_device, lens, page, Hq, Hkv, D):
    """fp32 beyond the size up to which single tokens join the larger tiles: partials
    of both kinds lie at the larger one's rows, and one launch merges them."""
    case = _setup(lens, page, FF, Hq, Hkv, D, seed=8)
    info = list(case[6]._info)
    assert info[6] > 0 and info[8] > 0 and info[7] == info[9] == 0
    first = torch.tensor([0] + case[3]).cumsum(0)
    split = {int(m[0]) for m in case[6]._buf[info[4]:info[4] + 8 * info[5]].view(-1, 8).cpu()}
    rows = {int(first[i]): n * (Hq // Hkv) for i, n in enumerate(case[3])}
    assert {rows[t] > 16 for t in split} == {False, True}
    _check(_attend(case), case, page)


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("Hq,Hkv", [(4, 1), (32, 2)])
def test_single_tokens_in_the_launch_of_many_rows(hip_device, dtype, D, Hq, Hkv):
    """Both split: rows of a few tokens and of whole tiles."""
    lens = [(3000, 80), (3000, 1), (700, 1), (0, 1), (1500, 24)]
    case = _setup(lens, 64, dtype, Hq, Hkv, D, seed=8)
    info = list(case[6]._info)
    assert info[6:9] == [0, 0, 0] and info[5] > 1
    _check(_attend(case), case, 64)
