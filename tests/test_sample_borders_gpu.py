"""GPU tests of sampling where a border lies among tokens whose mass is rounded
away, with uniforms next to 1 and at it."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = [1.0 - 2.0 ** -53, 1.0, 1.0 - 2.0 ** -44, 1.0 - 2.0 ** -30]


def _sample(x, u, **kw):
    from intel_kivi_hybrid_amd import _C
    return _C.sample(x.cuda(), torch.tensor(u, dtype=torch.float64, device="cuda:0"), **kw).cpu()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("many", [1, 100, 7000])
def test_cuts_among_tokens_without_mass(hip_device, dtype, many):
    """Token 0 masked, one token at 5, ``many`` at 4.75 and ten from 30.625 nats below
    the first on (each 2^-44.2 of it at most, under half of 2^-43).  Wherever the
    cuts lie among these, the last token with mass is the last one at 4.75."""
    x = torch.full((len(U), many + 12), float("-inf"))
    x[:, 1] = 5.0
    x[:, 2:many + 2] = 4.75
    x[:, many + 2:] = -25.625 - 0.125 * torch.arange(10)
    x = x.to(dtype)
    want = [many + 1] * len(U)
    for k in (many + 1, many + 2, many + 5, many + 11, 0):
        for kw in (dict(), dict(top_p=1.0 - 2.0 ** -53), dict(min_p=2e-14), dict(min_p=4e-14),
                   dict(top_p=1.0 - 2.0 ** -53, min_p=2e-14)):
            assert _sample(x, U, top_k=k, **kw).tolist() == want, (k, kw)
        assert _sample(x, [0.0] * len(U), top_k=k).tolist() == [1] * len(U)


def test_top_k_at_every_depth(hip_device):
    """One token for each quarter of a nat down to 40 below the largest, and u = 1: the
    last of the kept ones that has mass (half of 2^-43 and more: 30.498 nats)."""
    x = torch.full((1, 200), float("-inf"))
    x[0, 20:180] = -0.25 * torch.arange(160)
    last = 20 + 121
    for k in range(1, 161):
        assert int(_sample(x, [1.0], top_k=k)[0]) == min(19 + k, last), k
        assert int(_sample(x, [1.0], top_k=k, top_p=1.0 - 2.0 ** -53)[0]) == min(19 + k, last), k
    w = np.exp(-0.25 * np.arange(160))
    for u in (0.2, 0.9, 0.999):
        want = 20 + int(np.searchsorted(np.cumsum(w), u * w.sum(), "right"))
        assert int(_sample(x, [u])[0]) == want
