"""GPU tests of the paged cache's calls: tensors that derivatives are asked of,
and captures."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from tests.test_paged_gpu import _c, _setup

pytestmark = pytest.mark.gpu
BF, FF = torch.bfloat16, torch.float32


def _inputs(dtype=FF):
    table, pool, ctx, new, kp, vp, plan, q = _setup([(20, 2)], 32, dtype, 4, 2, 64, seed=3)
    k = torch.randn(2, 2, 64, device="cuda:0").to(dtype)
    cos, sin = _c().rotary_tables(22, 64, device="cuda:0")
    return plan, dict(q=q.cuda(), k_pages=kp.cuda(), v_pages=vp.cuda(), k=k, v=k.clone(), cos=cos,
                      sin=sin, q_norm=torch.ones(64, device="cuda:0"),
                      k_norm=torch.ones(64, device="cuda:0"))


def _calls(plan, x):
    attend = {n: x[n] for n in ("q", "k_pages", "v_pages")}
    yield attend, lambda: _c().paged_attention(plan=plan, **attend)
    yield x, lambda: _c().paged_append(plan=plan, **x)


def test_every_tensor_that_needs_a_gradient_is_refused(hip_device):
    plan, x = _inputs()
    for i in range(2):
        names = list(list(_calls(plan, x))[i][0])
        for name in names:
            y = {**x, name: x[name].clone().requires_grad_()}
            with pytest.raises(RuntimeError, match="inference only"):
                list(_calls(plan, y))[i][1]()
            with torch.no_grad():
                list(_calls(plan, y))[i][1]()
    # outputs of the caller's too
    for name, call in (("out", lambda o: _c().paged_attention(x["q"], x["k_pages"], x["v_pages"],
                                                              plan, out=o)),
                       ("q_out", lambda o: _c().paged_append(x["k"], x["v"], x["k_pages"],
                                                             x["v_pages"], plan, q=x["q"],
                                                             q_out=o))):
        with pytest.raises(RuntimeError, match="inference only"):
            call(torch.empty_like(x["q"]).requires_grad_())


def test_forward_mode_tangents_are_refused(hip_device):
    plan, x = _inputs()
    with fwd.dual_level():
        for i in range(2):
            for name in list(_calls(plan, x))[i][0]:
                y = {**x, name: fwd.make_dual(x[name], torch.ones_like(x[name]))}
                for mode in (torch.enable_grad, torch.no_grad):
                    with mode(), pytest.raises(RuntimeError, match="inference only"):
                        list(_calls(plan, y))[i][1]()
            list(_calls(plan, x))[i][1]()                     # (a level without tangents)


def test_capture_on_the_plans_own_stream_needs_a_settled_plan(hip_device):
    s = torch.cuda.Stream()
    table, pool, ctx, new, kp, vp, other, q = _setup([(20, 1)], 32, BF, 4, 2, 64, seed=3)
    kd, vd, qd = kp.cuda(), vp.cuda(), q.cuda()
    want = _c().paged_attention(qd, kd, vd, other)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        plan = _c().paged_plan(table, ctx, new, page_size=32, num_pages=pool, q_heads=4,
                               kv_heads=2, head_dim=64, device="cuda:0")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        with pytest.raises(RuntimeError, match="wait"):
            _c().paged_attention(qd, kd, vd, plan)
        torch.zeros(1, device="cuda:0")
    plan.wait()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = _c().paged_attention(qd, kd, vd, plan)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
