"""A batch of sequences that come and go over a cache of 8 bits, with penalties,
biases and grammars before sampling: each step a plan, for each layer an append and
an attention, then logits, their adjustment and the next tokens, which are the next
step's inputs.  Every stage is checked against its formula in float64, on the stage's
own inputs."""

import threading

import numpy as np
import pytest
import torch

from tests.paged8_helpers import attention8_tolerance, empty_pool, fill, largest_weight, values
from tests.paged_helpers import attention64, rows64, slots_of
from tests.test_adjust_gpu import _check as check_adjusted
from tests.test_sample_gpu import _reference
from tests.test_serving_steps_gpu import STEPS, Pages

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _c():
    from intel_kivi_hybrid_amd import _C
    return _C


@pytest.mark.parametrize("dtype,Hq,Hkv,D,page", [(torch.bfloat16, 8, 2, 128, 16),
                                                 (torch.float16, 4, 4, 64, 32),
                                                 (torch.float32, 6, 2, 80, 64)])
def test_sequences_come_and_go(hip_device, dtype, Hq, Hkv, D, page):
    C = _c()
    layers, vocab, pool = 2, 517, 24 if page == 16 else 14
    g = torch.Generator().manual_seed(D)
    rand = lambda *s: torch.randn(*s, generator=g)                        # noqa: E731
    width = Hq * D
    embed = rand(vocab, width).to(DEV)
    w_qkv = [(rand(width, (Hq + 2 * Hkv) * D) * width ** -0.5).to(DEV) for _ in range(layers)]
    w_out = [(rand(width, width) * width ** -0.5).to(DEV) for _ in range(layers)]
    norms = [(1 + 0.1 * rand(D)).to(dtype).to(DEV) for _ in range(2)]
    cos, sin = C.rotary_tables(256, D // 16 * 16 if D != 80 else 32, device=DEV)
    # codes and scales of a layer's keys and values, here and on the device
    host = [[*empty_pool(pool, Hkv, page, D, 3), *empty_pool(pool, Hkv, page, D, 4)]
            for _ in range(layers)]
    pools = [[t.to(DEV) for t in h] for h in host]
    pages, text, prompt = Pages(pool, page), {}, {}
    rs = np.random.RandomState(5)
    for step in STEPS:
        for name in step.get("leave", ()):
            pages.remove(name)
        for name, n in step.get("back", {}).items():
            pages.cut(name, n)
            # (its last token is an input that has not been appended)
            text[name] = text[name][:pages.length[name]] + text[name][-1:]
        names = list(step["bring"])
        new = [step["bring"][n] for n in names]
        ids = []
        for name, n in zip(names, new):
            had = pages.length.get(name, 0)
            pages.add(name, n)
            own = text.setdefault(name, [])
            own += rs.randint(0, vocab, max(0, had + n - len(own))).tolist()
            prompt.setdefault(name, len(own))
            ids += own[had:had + n]
        ctx, table = [pages.length[n] for n in names], pages.table(names)
        plan = C.paged_plan(table, ctx, new, page_size=page, num_pages=pool, q_heads=Hq,
                            kv_heads=Hkv, head_dim=D, dtype=dtype, device=DEV,
                            cache_dtype=torch.int8)
        plan.wait()
        slots = slots_of(table, ctx, new, page)
        held = [c - n for c, n in zip(ctx, new) for _ in range(n)]
        at = torch.tensor([p for _, _, p in slots])
        h = embed[torch.tensor(ids, device=DEV)]
        for layer in range(layers):
            kc, ks, vc, vs = pools[layer]
            qkv = (h @ w_qkv[layer]).to(dtype).view(len(ids), Hq + 2 * Hkv, D)
            q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]

            def run():
                r = C.paged_append(k, v, kc, vc, plan, q=q, k_scales=ks, v_scales=vs, cos=cos,
                                   sin=sin, q_norm=norms[0], k_norm=norms[1])
                return r, C.paged_attention(r, kc, vc, plan, k_scales=ks, v_scales=vs)
            r, o = run()
            # the append: the definition's codes and scales, and nothing else in the pages
            cs = cos.cpu()[at], sin.cpu()[at]
            fill(*host[layer][:2], rows64(k.cpu(), norms[1].cpu(), *cs, False), slots, held)
            fill(*host[layer][2:], v.cpu().double(), slots, held)
            for now, want in zip(pools[layer], host[layer]):
                assert torch.equal(now.cpu().view(torch.uint8), want.view(torch.uint8))
            # the attention
            K, KS, V, VS = host[layer]
            where = table, ctx, new, page, D ** -0.5
            ref, mag, size = attention64(r.cpu(), values(K, KS), values(V, VS), *where)
            largest = largest_weight(r.cpu(), values(K, KS), VS, *where)
            tol = attention8_tolerance(ref, mag, size, largest, D, max(ctx), dtype)
            assert bool(((o.cpu().double() - ref).abs() <= tol).all())
            # captured: appending the same tokens once more changes nothing
            if layer == 0:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    r2, o2 = run()
                for _ in range(2):
                    o2.zero_()
                    graph.replay()
                    assert torch.equal(r2, r) and torch.equal(o2, o)
                for now, want in zip(pools[layer], host[layer]):
                    assert torch.equal(now.cpu().view(torch.uint8), want.view(torch.uint8))
            h = h + o.float().reshape(len(ids), width) @ w_out[layer]
        # the last token of each sequence that brought some: its next
        ends, end = [], -1
        for n in new:
            end += n
            ends.append(end)
        live = [i for i, n in enumerate(new) if n]
        logits = (h[torch.tensor([ends[i] for i in live], device=DEV)] @ embed.t() * 0.1).to(dtype)
        rows = len(live)
        history = [text[names[i]][:ctx[i]] for i in live]
        tokens = torch.zeros(rows, max(map(len, history)), dtype=torch.int64)
        for j, own in enumerate(history):
            tokens[j, :len(own)] = torch.tensor(own)
        mask = torch.from_numpy(rs.rand(rows, vocab) < 0.5)
        kw = dict(tokens=tokens,
                  lengths=torch.tensor([len(own) for own in history], dtype=torch.int32),
                  prompt_lengths=torch.tensor([prompt[names[i]] for i in live], dtype=torch.int32),
                  repetition_penalty=torch.tensor([1.2, 1.0, 1.5, 0.9][:rows]),
                  presence_penalty=0.5, frequency_penalty=torch.tensor([0.1, 0.0, 0.3, 0.2][:rows]),
                  bias_ids=torch.tensor([1, 5, 100]), bias=torch.tensor([-2.0, 3.0, 0.5]),
                  allowed=C.allowed_tokens(mask))
        # (in place, as a step would, after into a tensor of fp32)
        wide = check_adjusted(logits, out=torch.empty(rows, vocab, device=DEV), **kw)
        ready = check_adjusted(logits.clone(), **kw)
        C.adjust_logits(logits, out=logits,
                        **{n: x.to(DEV) if torch.is_tensor(x) else x for n, x in kw.items()})
        assert torch.equal(logits, ready) and torch.equal(wide.to(dtype), ready)
        u = torch.from_numpy(rs.rand(rows))
        top_k = torch.tensor([0, 40, 5, 100][:rows], dtype=torch.int32)
        got = C.sample(ready, u.to(DEV), temperature=0.9, top_k=top_k.to(DEV), top_p=0.95)
        for j, i in enumerate(live):
            want, margin = _reference(ready[j].cpu().double().numpy(), float(u[j]), 0.9,
                                      int(top_k[j]), 0.95, 0.0)
            assert margin > 2.0 ** -25 and int(got[j]) == want and bool(mask[j, want])
            text[names[i]] = text[names[i]][:ctx[i]] + [want]


def test_two_threads_on_one_stream(hip_device):
    """Launches of two host threads alternate on the stream they share; neither's
    partial results reach the other's."""
    C = _c()
    runs = []
    for seed, (ctx, V) in enumerate(((5000, 9001), (7000, 20000))):
        g = torch.Generator().manual_seed(seed)
        pages = -(-ctx // 64)
        table = torch.randperm(pages, generator=g).to(torch.int32)[None]
        plan = C.paged_plan(table, [ctx], [1], page_size=64, num_pages=pages, q_heads=8,
                            kv_heads=2, head_dim=128, device=DEV, cache_dtype=torch.int8)
        codes = [torch.randint(-127, 128, (pages, 2, 64, 128), generator=g).to(torch.int8).to(DEV)
                 for _ in range(2)]
        scales = [(2.0 ** torch.randint(-8, -5, (pages, 2, 4), generator=g)).to(DEV)
                  for _ in range(2)]
        q = torch.randn(1, 8, 128, generator=g).to(torch.bfloat16).to(DEV)
        x = torch.randn(3, V, generator=g).to(torch.bfloat16).to(DEV)
        t = torch.randint(0, V, (3, 4000), generator=g).to(DEV)
        runs.append(lambda q=q, codes=codes, scales=scales, plan=plan, x=x, t=t: (
            C.paged_attention(q, *codes, plan, k_scales=scales[0], v_scales=scales[1]),
            C.adjust_logits(x, tokens=t, frequency_penalty=0.1)))
    want = [run() for run in runs]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        for _ in range(50):
            got[i].append(runs[i]())
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 50
        for o, y in got[i]:
            assert torch.equal(o, want[i][0]) and torch.equal(y, want[i][1])
