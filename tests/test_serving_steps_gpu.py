"""A batch of sequences that come and go, served with the paged cache and sampling
as they are used together: each step a plan, for each layer an append and an
attention, then logits and the next tokens, which are the next step's inputs.
Every stage is checked against its formula in float64, on the stage's own inputs."""

import threading

import numpy as np
import pytest
import torch

from tests.paged_helpers import EPS, attention64, attention_tolerance, rows64, slots_of
from tests.test_sample_gpu import _reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _c():
    from intel_kivi_hybrid_amd import _C
    return _C


class Pages:
    """A pool's free pages, and each sequence's."""

    def __init__(self, pages, page_size):
        self.free, self.page = list(range(pages))[::-1], page_size
        self.of, self.length = {}, {}

    def add(self, name, tokens):
        self.length[name] = self.length.get(name, 0) + tokens
        own = self.of.setdefault(name, [])
        while len(own) * self.page < self.length[name]:
            own.append(self.free.pop())

    def cut(self, name, tokens):
        self.length[name] -= tokens
        keep = -(-self.length[name] // self.page)
        self.free += self.of[name][keep:]
        del self.of[name][keep:]

    def remove(self, name):
        self.free += self.of.pop(name)
        del self.length[name]

    def table(self, names):
        t = np.full((len(names), max(len(self.of[n]) for n in names)), -1, dtype=np.int32)
        for i, n in enumerate(names):
            t[i, :len(self.of[n])] = self.of[n]
        return torch.from_numpy(t)


# what each step does: tokens that a sequence brings (a chunk of its prompt, one
# token, or some to verify), those it takes back before, sequences that leave
STEPS = [
    dict(bring={"a": 37}),
    dict(bring={"a": 1, "b": 70}),
    dict(bring={"a": 1, "b": 64, "c": 5}),              # b's prompt in two chunks
    dict(bring={"a": 4, "b": 1, "c": 1}),               # a verifies four
    dict(back={"a": 3}, bring={"a": 1, "b": 1, "c": 1}),
    dict(leave=["b"], bring={"c": 1, "d": 90, "a": 0}),
    dict(bring={"d": 1, "c": 1, "a": 1}),
    dict(leave=["a", "c"], bring={"d": 1}),
]


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
    kp = [torch.full((pool, Hkv, page, D), float("nan"), dtype=dtype, device=DEV)
          for _ in range(layers)]
    vp = [x.clone() for x in kp]
    pages, text = Pages(pool, page), {}
    rs = np.random.RandomState(5)
    for step in STEPS:
        for name in step.get("leave", ()):
            pages.remove(name)
        for name, n in step.get("back", {}).items():
            pages.cut(name, n)
        names = list(step["bring"])
        new = [step["bring"][n] for n in names]
        ids = []
        for name, n in zip(names, new):
            pages.add(name, n)
            last = text.get(name)
            ids += ([last] if last is not None and n else []) + list(
                rs.randint(0, vocab, max(0, n - (last is not None))))
        ctx, table = [pages.length[n] for n in names], pages.table(names)
        plan = C.paged_plan(table, ctx, new, page_size=page, num_pages=pool, q_heads=Hq,
                            kv_heads=Hkv, head_dim=D, dtype=dtype, device=DEV)
        slots = slots_of(table, ctx, new, page)
        at = torch.tensor([p for _, _, p in slots])
        h = embed[torch.tensor(ids, device=DEV)]
        for layer in range(layers):
            before = kp[layer].clone(), vp[layer].clone()
            qkv = (h @ w_qkv[layer]).to(dtype).view(len(ids), Hq + 2 * Hkv, D)
            q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
            r = C.paged_append(k, v, kp[layer], vp[layer], plan, q=q, cos=cos, sin=sin,
                               q_norm=norms[0], k_norm=norms[1])
            o = C.paged_attention(r, kp[layer], vp[layer], plan)
            # the append: its rows (half a step, and fp32's sums over D channels), and
            # nothing else in the pages
            cs = cos.cpu()[at], sin.cpu()[at]
            for src, w, got in ((q, norms[0], r), (k, norms[1], None)):
                want = rows64(src.cpu(), w.cpu(), *cs, False)
                if got is None:
                    got = torch.stack([kp[layer][p, :, i] for p, i, _ in slots])
                size = want.abs().amax(-1, keepdim=True)
                tol = EPS[dtype] / 2 * want.abs() + 2.0 ** -24 * (3 + D + 8) * 2 * size
                assert bool(((got.cpu().double() - want).abs() <= tol).all())
            assert torch.equal(torch.stack([vp[layer][p, :, i] for p, i, _ in slots]), v)
            for now, then in zip((kp[layer], vp[layer]), before):
                for p, i, _ in slots:
                    then[p, :, i] = now[p, :, i]
                assert torch.equal(now.view(torch.uint8), then.view(torch.uint8))
            # the attention
            ref, mag, size = attention64(r.cpu(), kp[layer].cpu(), vp[layer].cpu(), table, ctx,
                                         new, page, D ** -0.5)
            tol = attention_tolerance(ref, mag, size, D, max(ctx), dtype)
            assert bool(((o.cpu().double() - ref).abs() <= tol).all())
            h = h + o.float().reshape(len(ids), width) @ w_out[layer]
        # the last token of each sequence that brought some: its next
        ends, end = [], -1
        for n in new:
            end += n
            ends.append(end)
        live = [i for i, n in enumerate(new) if n]
        logits = (h[torch.tensor([ends[i] for i in live], device=DEV)] @ embed.t() * 0.1).to(dtype)
        u = torch.from_numpy(rs.rand(len(live)))
        top_k = torch.tensor([0, 40, 5, 100][:len(live)], dtype=torch.int32)
        got = C.sample(logits, u.to(DEV), temperature=0.9, top_k=top_k.to(DEV), top_p=0.95)
        for j, i in enumerate(live):
            want, margin = _reference(logits[j].cpu().double().numpy(), float(u[j]), 0.9,
                                      int(top_k[j]), 0.95, 0.0)
            assert margin > 2.0 ** -25 and int(got[j]) == want
            text[names[i]] = want


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
                            kv_heads=2, head_dim=128, device=DEV)
        put = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(DEV)   # noqa: E731
        q, kp, vp = put(1, 8, 128), put(pages, 2, 64, 128), put(pages, 2, 64, 128)
        x, u = put(3, V), torch.rand(3, generator=g).to(DEV)
        kw = dict(temperature=0.8, top_k=50, top_p=0.9)
        runs.append((lambda q=q, kp=kp, vp=vp, plan=plan, x=x, u=u, kw=kw:
                     (C.paged_attention(q, kp, vp, plan), C.sample(x, u, **kw))))
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
        for o, ids in got[i]:
            assert torch.equal(o, want[i][0]) and torch.equal(ids, want[i][1])
