"""The serving operators on the paged cache and on logits, as timed cases.

Three operators that a serving loop runs one after the other at every step:

* ``append``: the step's queries, keys and values of one layer: per-head RMS
  norms of queries and keys (where the model has them), rotation by each
  token's position, keys and values written to their pages.
* ``attend``: attention of the step's new tokens over the paged cache: a
  prompt's chunk, a verification pass or one token for each sequence, all in
  one call; a token sees its sequence up to itself.
* ``sample``: next tokens from logits, temperature, top-k, top-p, min-p and
  given random numbers.

With ``own`` false the operators are computed from elementary torch
operations; with ``own`` true by the package.
"""

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}


def _paged(name, kind, seqs, ctx, new, Hq, Hkv, D, page=64, dtype="bf16", chunks=None,
           rotary=None, style="halves", norm=False):
    """``seqs`` sequences, ``new`` tokens each, with up to ``ctx`` tokens of
    context before them (ragged: from half of it up).  ``chunks``: so many of
    the sequences bring a prompt's chunk of ``new`` tokens, the others one
    token.  ``rotary``: rotated channels."""
    case = {"kind": kind, "seqs": seqs, "ctx": ctx, "new": new, "Hq": Hq, "Hkv": Hkv, "D": D,
            "page": page, "dtype": dtype, "chunks": seqs if chunks is None else chunks}
    if kind == "append":
        case.update(rotary=D if rotary is None else rotary, style=style, norm=norm)
    return {"name": name, **case} if name else case


def _sample(name, B, V, dtype, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False):
    """``mixed``: each row is a request with settings of its own."""
    case = {"kind": "sample", "B": B, "V": V, "dtype": dtype, "temperature": temperature,
            "top_k": top_k, "top_p": top_p, "min_p": min_p, "mixed": mixed}
    return {"name": name, **case} if name else case


def listed():
    return [
        # One user's next token on an 8B-shaped model with per-head norms:
        # the smallest call, all latency.
        _paged("append_single", "append", 1, 1020, 1, 32, 8, 128, norm=True),
        # One step of 64 running requests of a 70B-shaped model.
        _paged("append_serving", "append", 64, 600, 1, 64, 8, 128, page=32, dtype="f16"),
        # Three prompts of unequal lengths entering the cache.
        _paged("append_prompts", "append", 3, 100, 4111, 32, 8, 128, norm=True),
        # Neighbouring channels rotated, half of each head, fp32: a small
        # multi-head model's prompts.
        _paged("append_partial", "append", 8, 40, 301, 12, 12, 64, page=16, dtype="f32",
               rotary=32, style="neighbours"),
        # One user's next token after a thousand: all latency.
        _paged("attend_single", "attend", 1, 1020, 1, 32, 8, 128),
        # The benchmark's serving batch, unequal lengths up to 8K.
        _paged("attend_serving", "attend", 64, 8191, 1, 32, 8, 128),
        # A chunk of a long prompt after 8K tokens of it.
        _paged("attend_chunk", "attend", 1, 8200, 2048, 32, 8, 128),
        # Continuous batching: two prompts' chunks among running requests, 8
        # query heads for each kv head.
        _paged("attend_mixed", "attend", 32, 5001, 777, 64, 8, 128, page=16, dtype="f16",
               chunks=2),
        # Assisted decoding: five drafted tokens for each of 16 requests.
        _paged("attend_verify", "attend", 16, 3001, 5, 28, 4, 128, page=128),
        # A small multi-head model in fp32.
        _paged("attend_f32", "attend", 4, 500, 301, 12, 12, 64, page=32, dtype="f32"),
        # One request, a 50257-word vocabulary.
        _sample("sample_single", 1, 50257, "f32", temperature=0.8, top_k=50, top_p=0.95),
        # A serving batch of requests with settings of their own.
        _sample("sample_serving", 64, 128256, "bf16", mixed=True),
    ]


_HEADS = [(32, 8), (32, 32), (12, 12), (64, 8), (24, 8), (16, 2), (28, 4), (16, 4)]
_DIMS = [128, 128, 128, 64, 64, 256, 96, 80]
_MOST_PAIRS = 2048 * 7000 * 32 * 128          # attend_chunk's scores x channels
_MOST_CACHE = 64 * 6100 * 8 * 128             # attend_serving's elements for each of K and V


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "sample"])
    if kind == "sample":
        V = _log_int(rng, 200, 131072)
        B = _log_int(rng, 1, max(1, min(256, 64 * 128256 // V)))
        return _sample(None, B, V, rng.choice(["f32", "bf16", "f16"]),
                       rng.choice([0.0, 0.3, 0.7, 1.0, 1.0, 1.7]),
                       rng.choice([0, 0, 1, 20, 50, 400]), rng.choice([1.0, 0.5, 0.9, 0.95]),
                       rng.choice([0.0, 0.0, 0.05, 0.3]), rng.random() < 0.4)
    Hq, Hkv = rng.choice(_HEADS)
    D = rng.choice(_DIMS)
    page = rng.choice([16, 32, 64, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "append":
        seqs = _log_int(rng, 1, 64)
        new = rng.choice([1, _log_int(rng, 1, max(1, 12000 * 40 // (seqs * (Hq + Hkv))))])
        ctx = _log_int(rng, 1, max(1, min(1000, 40000 // seqs)))
        rotary = rng.choice([D, D, D // 32 * 16])
        return _paged(None, kind, seqs, ctx, new, Hq, Hkv, D, page, dtype, rng.randint(0, seqs),
                      rotary, rng.choice(["halves", "halves", "neighbours"]),
                      rng.random() < 0.5)
    seqs = _log_int(rng, 1, 64)
    ctx = _log_int(rng, 1, max(1, min(16384, _MOST_CACHE // (2 * seqs * Hkv * D))))
    new, chunks = 1, seqs
    if rng.random() < 0.7:
        chunks = rng.choice([1, seqs, rng.randint(1, seqs)])
        # (fp32 products run at a sixteenth of the 16-bit rate)
        most = _MOST_PAIRS // (chunks * Hq * D * (16 if dtype == "f32" else 1))
        new = max(1, min(2048, _log_int(rng, 1, 2048),
                         int((-ctx + math.sqrt(ctx * ctx + 2.0 * most)))))
    return _paged(None, kind, seqs, ctx, new, Hq, Hkv, D, page, dtype, chunks)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(case):
    """New tokens and context lengths (these tokens included) of each
    sequence; they go by the case alone, so that its work does."""
    rs = np.random.RandomState(97 * case["seqs"] + case["ctx"])
    n = np.ones(case["seqs"], dtype=np.int64)
    chunked = rs.permutation(case["seqs"])[:case["chunks"]]
    n[chunked] = rs.randint((case["new"] + 1) // 2, case["new"] + 1, case["chunks"])
    before = rs.randint(case["ctx"] // 2, case["ctx"] + 1, case["seqs"])
    if case["chunks"]:
        n[chunked[0]] = case["new"]
    before[0] = case["ctx"]
    return n, before + n


def _generator(seed, part):
    return torch.Generator(device=DEVICE).manual_seed(1_000_003 * seed + part)


def _tables(case, rows):
    """cos and sin of position x frequency for the rotated pairs, fp32 (the
    angles of far positions in fp64)."""
    half = case["rotary"] // 2
    inv = 10000.0 ** (-np.arange(half, dtype=np.float64) / half)
    ang = np.arange(rows, dtype=np.float64)[:, None] * inv[None, :]
    return (torch.from_numpy(np.cos(ang).astype(np.float32)).to(DEVICE),
            torch.from_numpy(np.sin(ang).astype(np.float32)).to(DEVICE))


def _page_table(case, ctx, seed):
    """Each sequence's pages, scattered over the pool; the pool's size."""
    pages = -(-ctx // case["page"])
    pool = int(pages.sum()) + 7
    order = np.random.RandomState(seed % 2 ** 31).permutation(pool)
    table = np.zeros((len(ctx), int(pages.max())), dtype=np.int32)
    at = 0
    for b, c in enumerate(pages):
        table[b, :c] = order[at:at + c]
        at += c
    return table, pool


def _rand(shape, seed, part, dt, scale=None):
    """N(0,1) in pieces (fp32 on the way), with a few loud channels where
    ``scale`` is given."""
    out = torch.empty(shape, dtype=dt, device=DEVICE)
    g = _generator(seed, part)
    step = max(1, (1 << 26) // max(1, out[0].numel()))
    for i in range(0, shape[0], step):
        x = torch.randn(min(step, shape[0] - i), *shape[1:], generator=g, device=DEVICE)
        out[i:i + step] = x if scale is None else x * scale
    return out


def _logits(case, seed):
    """Logits of a language model's kind: a broad bell, and a few likely words."""
    B, V = case["B"], case["V"]
    g = _generator(seed, 0)
    x = 2.5 * torch.randn(B, V, generator=g, device=DEVICE)
    top = torch.randint(0, V, (B, min(V, 12)), generator=g, device=DEVICE)
    x.scatter_add_(1, top, 9.0 * torch.rand(top.shape, generator=g, device=DEVICE))
    return x.to(DTYPES[case["dtype"]])


def _settings(case, seed):
    """The settings of each row, as fp32 / int32 tensors (``mixed``) or numbers."""
    B = case["B"]
    if not case["mixed"]:
        return {k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")}
    rs = np.random.RandomState((seed + 5) % 2 ** 31)

    def pick(values, dt):
        return torch.from_numpy(rs.choice(values, B).astype(dt)).to(DEVICE)
    return {"temperature": pick([0.0, 0.3, 0.6, 0.8, 1.0, 1.0, 1.3], np.float32),
            "top_k": pick([0, 0, 0, 1, 20, 50, 200], np.int32),
            "top_p": pick([1.0, 1.0, 0.9, 0.95, 0.7], np.float32),
            "min_p": pick([0.0, 0.0, 0.0, 0.02, 0.1], np.float32)}


def _inputs(case, seed):
    if case["kind"] == "sample":
        return {"logits": _logits(case, seed), "settings": _settings(case, seed),
                "u": torch.rand(case["B"], dtype=torch.float64, generator=_generator(seed, 1),
                                device=DEVICE)}
    n, ctx = _lengths(case)
    table, pool = _page_table(case, ctx, seed)
    Hq, Hkv, D, dt = case["Hq"], case["Hkv"], case["D"], DTYPES[case["dtype"]]
    loud = 1.0 + 3.0 * (torch.rand(Hkv, 1, D, generator=_generator(seed, 9),
                                   device=DEVICE) < 0.03)
    T = int(n.sum())
    s = {"n": n, "ctx": ctx, "table": table,
         "k_pages": _rand((pool, Hkv, case["page"], D), seed, 2, dt, loud),
         "v_pages": _rand((pool, Hkv, case["page"], D), seed, 3, dt)}
    if case["kind"] == "attend":
        s["q"] = _rand((T, Hq, D), seed, 4, dt)
        return s
    # (one projection's rows hold a token's queries, keys and values)
    qkv = _rand((T, Hq + 2 * Hkv, D), seed, 4, dt)
    s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    s["cos"], s["sin"] = _tables(case, int(ctx.max()))
    s["q_norm"] = s["k_norm"] = None
    if case["norm"]:
        s["q_norm"] = (1.0 + 0.2 * _rand((1, D), seed, 5, torch.float32)[0]).to(dt)
        s["k_norm"] = (1.0 + 0.2 * _rand((1, D), seed, 6, torch.float32)[0]).to(dt)
    return s


def _host(case, s):
    """Where each new token goes and which pages each sequence has, on the
    GPU (a serving program makes this once a step, for every layer)."""
    pos = np.concatenate([np.arange(c - m, c) for c, m in zip(s["ctx"], s["n"])])
    seq = np.repeat(np.arange(len(s["n"])), s["n"])
    page = s["table"][seq, pos // case["page"]]
    return {k: torch.from_numpy(v.astype(np.int64)).to(DEVICE)
            for k, v in (("pos", pos), ("page", page), ("off", pos % case["page"]),
                         ("pages", s["table"]))}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["kind"] == "sample":
        return s
    if own:
        from intel_kivi_hybrid_amd import _C
        s["plan"] = _C.paged_plan(
            torch.from_numpy(s["table"]), s["ctx"].tolist(), s["n"].tolist(),
            page_size=case["page"], num_pages=s["k_pages"].shape[0], q_heads=case["Hq"],
            kv_heads=case["Hkv"], head_dim=case["D"], dtype=DTYPES[case["dtype"]],
            device=DEVICE)
    else:
        s.update(_host(case, s))
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if own:
        from intel_kivi_hybrid_amd import _C
        if kind == "append":
            q = _C.paged_append(state["k"], state["v"], state["k_pages"], state["v_pages"],
                                state["plan"], q=state["q"], cos=state["cos"], sin=state["sin"],
                                interleaved=state["case"]["style"] == "neighbours",
                                q_norm=state["q_norm"], k_norm=state["k_norm"], eps=1e-6)
            return [q, state["k_pages"], state["v_pages"]]
        if kind == "attend":
            return _C.paged_attention(state["q"], state["k_pages"], state["v_pages"],
                                      state["plan"])
        return _C.sample(state["logits"], state["u"], **state["settings"])
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[kind](state)


def _plain_rows(x, w, cos, sin, neighbours):
    """Norm and rotation of head rows ``[T, H, D]``, in fp32."""
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.float()
    r = 2 * cos.shape[-1]
    c, s = cos[:, None, :], sin[:, None, :]
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if neighbours else (y[..., :r // 2], y[..., r // 2:r])
    out = y.clone()
    if neighbours:
        out[..., 0:r:2], out[..., 1:r:2] = a * c - b * s, b * c + a * s
    else:
        out[..., :r // 2], out[..., r // 2:r] = a * c - b * s, b * c + a * s
    return out.to(x.dtype)


def _plain_append(s):
    neighbours = s["case"]["style"] == "neighbours"
    cos, sin = s["cos"][s["pos"]], s["sin"][s["pos"]]
    q = _plain_rows(s["q"], s["q_norm"], cos, sin, neighbours)
    s["k_pages"][s["page"], :, s["off"]] = _plain_rows(s["k"], s["k_norm"], cos, sin, neighbours)
    s["v_pages"][s["page"], :, s["off"]] = s["v"]
    return [q, s["k_pages"], s["v_pages"]]


def _plain_attend(s):
    case, q = s["case"], s["q"]
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    g = Hq // Hkv
    out = torch.empty_like(q)
    at = 0
    for b, (n, c) in enumerate(zip(s["n"].tolist(), s["ctx"].tolist())):
        pages = s["pages"][b, :-(-c // case["page"])]
        k, v = (s[x][pages].transpose(0, 1).reshape(Hkv, -1, D)[:, :c].float()
                for x in ("k_pages", "v_pages"))
        # query rows of a kv head: [token, head of its group]
        rows = q[at:at + n].float().view(n, Hkv, g, D).transpose(0, 1).reshape(Hkv, n * g, D)
        sc = torch.matmul(rows, k.transpose(1, 2).contiguous()) * D ** -0.5
        if n > 1:
            last = torch.arange(c - n, c, device=DEVICE).repeat_interleave(g)
            sc.masked_fill_(torch.arange(c, device=DEVICE)[None, :] > last[:, None],
                            float("-inf"))
        sc = torch.exp(sc - sc.amax(-1, keepdim=True))
        o = torch.matmul(sc, v) / sc.sum(-1, keepdim=True)
        out[at:at + n] = o.view(Hkv, n, g, D).transpose(0, 1).reshape(n, Hq, D).to(q.dtype)
        at += n
    return out


def _plain_sample(s):
    # in fp64: a token next to the border of a cumulative sum goes by bits
    # that fp32 sums lose
    x = s["logits"].double()
    B, V = x.shape
    t, k, p, m = (torch.as_tensor(s["settings"][n], device=DEVICE).double().expand(B)[:, None]
                  for n in ("temperature", "top_k", "top_p", "min_p"))
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    w = torch.exp((x - x[:, :1]) / torch.where(t > 0, t, torch.ones_like(t)))
    rank = torch.arange(V, device=DEVICE)[None, :]
    keep = (rank < torch.where(k > 0, k, torch.full_like(k, V))) & ((rank < 1) | (t > 0))
    w = torch.where(keep, w, torch.zeros_like(w))
    c = w.cumsum(-1)
    # the shortest prefix that holds the mass: up to the first sum that reaches it
    w = torch.where((c - w < p * c[:, -1:]) | (p >= 1) | (rank < 1), w, torch.zeros_like(w))
    w = torch.where(w >= m, w, torch.zeros_like(w))
    c = w.cumsum(-1)
    at = (c <= s["u"][:, None] * c[:, -1:]).sum(-1, keepdim=True)
    at = torch.minimum(at, (w > 0).sum(-1, keepdim=True) - 1)
    return order.gather(1, at)[:, 0]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["kind"] == "sample":
        n = case["B"] * case["V"]
        # a difference, a quotient, an exponential and a sum for each logit
        return {"bytes": n * SIZES[case["dtype"]] + 8 * case["B"], "flops": 4 * n}
    n, ctx = _lengths(case)
    T, size = int(n.sum()), SIZES[case["dtype"]]
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if case["kind"] == "append":
        rows = T * (Hq + 2 * Hkv) * D
        turned = T * (Hq + Hkv)
        flops = 3 * turned * case["rotary"] + (4 * turned * D if case["norm"] else 0)
        table = 4 * case["rotary"] * len(np.unique(np.concatenate(
            [np.arange(c - m, c) for c, m in zip(ctx, n)])))
        return {"bytes": 2 * rows * size + table, "flops": flops}
    pairs = int((n * ctx - n * (n - 1) // 2).sum())
    return {"bytes": (2 * int(ctx.sum()) * Hkv + 2 * T * Hq) * D * size,
            "flops": 4 * pairs * Hq * D}


# ---------------------------------------------------------------------------
# the definition in fp64
# ---------------------------------------------------------------------------
def _exact_sample(s, B, V):
    logits = s["logits"].double().cpu().numpy()
    u = s["u"].cpu().numpy()
    get = {n: np.broadcast_to(np.asarray(v.cpu() if torch.is_tensor(v) else v, dtype=np.float64),
                              (B,)) for n, v in s["settings"].items()}
    out = np.empty(B, dtype=np.int64)
    for b in range(B):
        x, t = logits[b], get["temperature"][b]
        order = np.argsort(-x, kind="stable")
        if t <= 0:
            out[b] = order[0]
            continue
        k = int(get["top_k"][b])
        order = order[:k] if k > 0 else order
        w = np.exp((x[order] - x[order[0]]) / t)
        mass = np.cumsum(w)
        kept = len(w)
        if get["top_p"][b] < 1:
            kept = min(kept, int(np.searchsorted(mass, get["top_p"][b] * mass[-1], "left")) + 1)
        kept = min(kept, max(1, int((w >= get["min_p"][b]).sum())))
        at = int(np.searchsorted(mass[:kept], u[b] * mass[kept - 1], "right"))
        out[b] = order[min(at, kept - 1)]
    return torch.from_numpy(out).to(DEVICE)


def _exact_append(case, s):
    pos = torch.cat([torch.arange(c - m, c) for c, m in zip(s["ctx"], s["n"])]).to(DEVICE)
    seq = torch.arange(len(s["n"])).repeat_interleave(torch.from_numpy(s["n"]))
    page = torch.from_numpy(s["table"]).long()[seq, pos.cpu() // case["page"]].to(DEVICE)
    off = pos % case["page"]
    half = case["rotary"] // 2
    i = torch.arange(half, device=DEVICE)
    first, second = (2 * i, 2 * i + 1) if case["style"] == "neighbours" else (i, i + half)
    # (the tables are inputs: their fp32 values)
    turn = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, None, :]

    def rows(x, w):
        y = x.double()
        if w is not None:
            y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w.double()
        z = torch.complex(y[..., first], y[..., second]) * turn
        y = y.index_copy(2, first, z.real)
        return y.index_copy(2, second, z.imag)
    k, v = s["k_pages"].double(), s["v_pages"].double()
    k[page, :, off] = rows(s["k"], s["k_norm"])
    v[page, :, off] = s["v"].double()
    return [rows(s["q"], s["q_norm"]), k, v]


def _exact_attend(case, s):
    Hq, Hkv, D, ps = case["Hq"], case["Hkv"], case["D"], case["page"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    at = 0
    for b in range(len(s["n"])):
        n, c = int(s["n"][b]), int(s["ctx"][b])
        p = torch.arange(c, device=DEVICE)
        page = torch.from_numpy(s["table"][b]).to(DEVICE).long()[p // ps]
        for h in range(Hkv):
            k, v = s["k_pages"][page, h, p % ps].double(), s["v_pages"][page, h, p % ps].double()
            kt = k.t().contiguous()
            for j in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                z = s["q"][at:at + n, j].double().mm(kt) / math.sqrt(D)
                z = torch.where(p[None, :] <= p[c - n:, None], z, float("-inf"))
                out[at:at + n, j] = torch.softmax(z, -1).mm(v)
        at += n
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(s, case["B"], case["V"])
    if case["kind"] == "append":
        return _exact_append(case, s)
    return _exact_attend(case, s)
