"""A serving step on a paged cache of 8 bits, as timed cases.

Three operators that a serving loop runs one after the other at every step:

* ``append``: the step's queries, keys and values of one layer: per-head RMS
  norms of queries and keys (where the model has them), rotation by each
  token's position, keys and values rounded to 8 bits with a scale for each
  block of 16 positions of a page and kv head, and written to their pages.
* ``attend``: attention of the step's new tokens over those pages: a prompt's
  chunk, a verification pass or one token for each sequence, all in one call;
  a token sees its sequence up to itself.
* ``adjust``: logits changed before sampling: penalties for repeated tokens,
  biases, and a grammar's mask.

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
BLOCK = 16                           # positions that share a scale
LEAST = 2.0 ** -126                  # the smallest scale


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


def _adjust(name, B, V, dtype, history, penalties, biased=0, mask=False, mixed=False):
    """``history``: tokens of the longest row so far, a part of them its
    prompt.  ``penalties``: some of "r" (repetition), "p" (presence) and "f"
    (frequency).  ``biased``: tokens of a row with a bias.  ``mixed``: each row
    is a request with settings of its own."""
    case = {"kind": "adjust", "B": B, "V": V, "dtype": dtype, "history": history,
            "penalties": penalties, "biased": biased, "mask": mask, "mixed": mixed}
    return {"name": name, **case} if name else case


def listed():
    return [
        # One user's next token on an 8B-shaped model with per-head norms, into
        # a block that holds some already: the smallest call, all latency.
        _paged("append_single", "append", 1, 300, 1, 32, 8, 128, norm=True),
        # One step of 64 running requests of a 70B-shaped model.
        _paged("append_serving", "append", 64, 90, 1, 64, 8, 128, page=32, dtype="f16"),
        # Three prompts of unequal lengths entering the cache.
        _paged("append_prompts", "append", 3, 100, 4111, 32, 8, 128, norm=True),
        # A small multi-head model in fp32 with learned positions: its keys
        # are only rounded.
        _paged("append_f32", "append", 8, 40, 301, 12, 12, 64, page=16, dtype="f32", rotary=0),
        # One user's next token after a thousand: all latency.
        _paged("attend_single", "attend", 1, 1020, 1, 32, 8, 128),
        # The benchmark's serving batch, unequal lengths up to 8K.
        _paged("attend_serving", "attend", 64, 8191, 1, 32, 8, 128),
        # A chunk of a long prompt after 8K tokens of it.
        _paged("attend_chunk", "attend", 1, 8200, 2048, 32, 8, 128),
        # Assisted decoding: five drafted tokens for each of 16 requests.
        _paged("attend_verify", "attend", 16, 3001, 5, 28, 4, 128, page=128, dtype="f16"),
        # A small multi-head model in fp32: prompts' chunks among running
        # requests.
        _paged("attend_f32", "attend", 12, 500, 301, 12, 12, 64, page=32, dtype="f32", chunks=4),
        # One request with a repetition penalty, a 50257-word vocabulary.
        _adjust("adjust_single", 1, 50257, "f32", 300, "r"),
        # A serving batch of requests with settings of their own, some of them
        # held to a grammar.
        _adjust("adjust_serving", 64, 128256, "bf16", 4000, "rpf", 40, True, True),
        # Long conversations.
        _adjust("adjust_long", 16, 32000, "f16", 30011, "pf", 3),
    ]


_HEADS = [(32, 8), (32, 32), (12, 12), (64, 8), (20, 4), (16, 2), (28, 4), (16, 4)]
_DIMS = [128, 128, 128, 64, 64, 256, 96, 80]
_MOST_PAIRS = 2048 * 7000 * 32 * 128          # attend_chunk's scores x channels
_MOST_CACHE = 64 * 6100 * 8 * 128             # attend_serving's elements for each of K and V


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "adjust"])
    if kind == "adjust":
        V = _log_int(rng, 200, 131072)
        B = _log_int(rng, 1, max(1, min(256, 64 * 128256 // V)))
        most = max(2, min(32768, 64 * 4000 // B))
        penalties = rng.choice(["", "r", "r", "p", "f", "pf", "rpf", "rpf"])
        return _adjust(None, B, V, rng.choice(["f32", "bf16", "f16"]), _log_int(rng, 1, most),
                       penalties, rng.choice([0, 0, 1, rng.randint(1, min(V // 2, 300))]),
                       rng.random() < 0.5 or not penalties, rng.random() < 0.5)
    Hq, Hkv = rng.choice(_HEADS)
    D = rng.choice(_DIMS)
    page = rng.choice([16, 32, 64, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "append":
        seqs = _log_int(rng, 1, 64)
        new = rng.choice([1, _log_int(rng, 1, max(1, 12000 * 40 // (seqs * (Hq + Hkv))))])
        ctx = _log_int(rng, 1, max(1, min(1000, 6000 // seqs)))
        if dtype == "f32":           # (learned positions)
            return _paged(None, kind, seqs, ctx, new, Hq, Hkv, D, page, dtype,
                          rng.randint(0, seqs), 0)
        rotary = rng.choice([D, D, D // 32 * 16])
        return _paged(None, kind, seqs, ctx, new, Hq, Hkv, D, page, dtype, rng.randint(0, seqs),
                      rotary, rng.choice(["halves", "halves", "neighbours"]),
                      rng.random() < 0.5)
    seqs = _log_int(rng, 1, 64)
    ctx = _log_int(rng, 1, max(1, min(16384, _MOST_CACHE // (2 * seqs * Hkv * D))))
    new, chunks = 1, seqs
    if rng.random() < 0.7:
        chunks = rng.choice([1, seqs, rng.randint(1, seqs)])
        # (fp32 queries and weights take several products each)
        most = _MOST_PAIRS // (chunks * Hq * D * (4 if dtype == "f32" else 1))
        new = max(1, min(2048, _log_int(rng, 1, 2048),
                         int((-ctx + math.sqrt(ctx * ctx + 2.0 * most)))))
    return _paged(None, kind, seqs, ctx, new, Hq, Hkv, D, page, dtype, chunks)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(case):
    """New tokens and context lengths (these tokens included) of each
    sequence; they go by the case alone, so that its work does."""
    rs = np.random.RandomState(89 * case["seqs"] + case["ctx"])
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
    inv = 10000.0 ** (-np.arange(half, dtype=np.float64) / max(half, 1))
    ang = np.arange(rows, dtype=np.float64)[:, None] * inv[None, :]
    return (torch.from_numpy(np.cos(ang).astype(np.float32)).to(DEVICE),
            torch.from_numpy(np.sin(ang).astype(np.float32)).to(DEVICE))


def _page_table(case, ctx, seed):
    """Each sequence's pages, scattered over the pool; the pool's size."""
    pages = -(-ctx // case["page"])
    pool = int(pages.sum()) + 7
    order = np.random.RandomState((seed + 3) % 2 ** 31).permutation(pool)
    table = np.zeros((len(ctx), int(pages.max())), dtype=np.int32)
    at = 0
    for b, c in enumerate(pages):
        table[b, :c] = order[at:at + c]
        at += c
    return table, pool


def _scale_for(top):
    """The smallest power of two from 2^-126 on whose 127-fold reaches ``top``."""
    m, e = torch.frexp(top)
    k = e - 7 + (m > 127.0 / 128).to(e.dtype)
    s = torch.where(top > 0, torch.ldexp(torch.ones_like(top), k.clamp_min(-126)), LEAST)
    return s.float()


def _pool(case, pool, seed, part, loud):
    """A pool of 8 bits and its scales: N(0,1), a few loud channels where
    ``loud`` is given, in blocks of a loudness of their own."""
    Hkv, D, page = case["Hkv"], case["D"], case["page"]
    g = _generator(seed, part)
    codes = torch.empty(pool, Hkv, page, D, dtype=torch.int8, device=DEVICE)
    scales = torch.empty(pool, Hkv, page // BLOCK, dtype=torch.float32, device=DEVICE)
    step = max(1, (1 << 26) // (Hkv * page * D))
    for i in range(0, pool, step):
        x = torch.randn(min(step, pool - i), Hkv, page // BLOCK, BLOCK, D, generator=g,
                        device=DEVICE)
        x *= 0.6 + 0.8 * torch.rand(x.shape[:3], generator=g, device=DEVICE)[..., None, None]
        if loud is not None:
            x *= loud[:, None]
        s = _scale_for(x.abs().amax((-1, -2)))
        scales[i:i + step] = s
        codes[i:i + step] = torch.round(x / s[..., None, None]).view(-1, Hkv, page, D).to(torch.int8)
    return codes, scales


def _rows(shape, seed, part, dt):
    return torch.randn(shape, generator=_generator(seed, part), device=DEVICE).to(dt)


def _adjust_inputs(case, seed):
    """Logits of a language model's kind (a broad bell, and a few likely
    words), and what each request has said and asks for."""
    B, V, L = case["B"], case["V"], case["history"]
    g = _generator(seed, 0)
    x = 2.5 * torch.randn(B, V, generator=g, device=DEVICE)
    top = torch.randint(0, V, (B, min(V, 12)), generator=g, device=DEVICE)
    x.scatter_add_(1, top, 9.0 * torch.rand(top.shape, generator=g, device=DEVICE))
    # a text's words: few of them often, most of them seldom
    tokens = (V * torch.rand(B, L, generator=g, device=DEVICE) ** 4).long().clamp_max(V - 1)
    rs = np.random.RandomState((seed + 11) % 2 ** 31)
    lengths = rs.randint((L + 1) // 2, L + 1, B)
    lengths[0] = L
    s = {"logits": x.to(DTYPES[case["dtype"]]), "tokens": tokens,
         "lengths": torch.from_numpy(lengths.astype(np.int32)).to(DEVICE),
         "prompts": torch.from_numpy((lengths * rs.rand(B)).astype(np.int32)).to(DEVICE)}

    def setting(key, neutral, usual, values):
        if key not in case["penalties"]:
            return neutral
        if not case["mixed"]:
            return usual
        return torch.from_numpy(rs.choice(values, B).astype(np.float32)).to(DEVICE)
    s["repetition"] = setting("r", 1.0, 1.125, [1.0, 1.0, 1.05, 1.2, 0.9])
    s["presence"] = setting("p", 0.0, 0.5, [0.0, 0.0, 0.25, 0.7, -0.3])
    s["frequency"] = setting("f", 0.0, 0.25, [0.0, 0.0, 0.1, 0.6, -0.2])
    s["bias_ids"] = s["bias"] = s["allowed"] = None
    if case["biased"]:
        K = case["biased"]
        # (distinct in a row: spread over the vocabulary from a start of its own)
        s["bias_ids"] = (torch.randint(0, V, (B, 1), generator=g, device=DEVICE)
                         + (V // K) * torch.arange(K, device=DEVICE)) % V
        s["bias"] = 3.0 * torch.randn(B, K, generator=g, device=DEVICE)
    if case["mask"]:
        # some rows free, some banned from half the words, some held to a few
        kind = torch.from_numpy(rs.randint(0, 3, B)).to(DEVICE)[:, None]
        words = torch.randint(-2 ** 31, 2 ** 31, (B, -(-V // 32)), generator=g, device=DEVICE)
        few = torch.rand(words.shape, generator=g, device=DEVICE) < 0.01
        s["allowed"] = torch.where(kind == 0, torch.full_like(words, -1), torch.where(
            (kind == 1) | few, words, torch.zeros_like(words))).to(torch.int32)
    return s


def _inputs(case, seed):
    if case["kind"] == "adjust":
        return _adjust_inputs(case, seed)
    n, ctx = _lengths(case)
    table, pool = _page_table(case, ctx, seed)
    Hq, Hkv, D, dt = case["Hq"], case["Hkv"], case["D"], DTYPES[case["dtype"]]
    loud = 1.0 + 3.0 * (torch.rand(Hkv, 1, D, generator=_generator(seed, 9),
                                   device=DEVICE) < 0.03)
    T = int(n.sum())
    s = {"n": n, "ctx": ctx, "table": table}
    s["k_pages"], s["k_scales"] = _pool(case, pool, seed, 2, loud)
    s["v_pages"], s["v_scales"] = _pool(case, pool, seed, 3, None)
    if case["kind"] == "attend":
        s["q"] = _rows((T, Hq, D), seed, 4, dt)
        return s
    # (one projection's rows hold a token's queries, keys and values; some
    # tokens are louder than what their block held)
    qkv = _rows((T, Hq + 2 * Hkv, D), seed, 4, torch.float32)
    qkv *= 0.5 + 2.0 * torch.rand(T, 1, 1, generator=_generator(seed, 7), device=DEVICE)
    qkv = qkv.to(dt)
    s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    s["cos"], s["sin"] = _tables(case, int(ctx.max())) if case["rotary"] else (None, None)
    s["q_norm"] = s["k_norm"] = None
    if case["norm"]:
        s["q_norm"] = (1.0 + 0.2 * _rows((D,), seed, 5, torch.float32)).to(dt)
        s["k_norm"] = (1.0 + 0.2 * _rows((D,), seed, 6, torch.float32)).to(dt)
    return s


def _host(case, s):
    """Where each new token goes, which pages each sequence has, and which
    sequences bring several tokens, on the GPU (a serving program makes this
    once a step, for every layer)."""
    n, ctx, table = s["n"], s["ctx"], s["table"]
    pos = np.concatenate([np.arange(c - m, c) for c, m in zip(ctx, n)])
    seq = np.repeat(np.arange(len(n)), n)
    page = table[seq, pos // case["page"]]
    index = {"pos": pos, "page": page, "off": pos % case["page"]}
    # blocks that get tokens, and how many of their positions were there before
    size = case["page"] // BLOCK
    keys, which = np.unique(page.astype(np.int64) * size + index["off"] // BLOCK,
                            return_inverse=True)
    first = np.full(len(keys), BLOCK, dtype=np.int64)
    np.minimum.at(first, which, pos % BLOCK)
    index.update(block=which.reshape(-1), block_page=keys // size, block_in_page=keys % size,
                 held=first)
    for key, several in (("one", False), ("more", True)):
        at = np.nonzero((n > 1) == several)[0]
        if not len(at):
            continue
        t = np.arange(n[at].max())[None, :]
        pages = -(-ctx[at].max() // case["page"])
        index.update({key + "_row": np.minimum(np.cumsum(n)[at][:, None] - n[at][:, None] + t,
                                               n.sum() - 1),
                      key + "_live": t < n[at][:, None], key + "_pages": table[at, :pages],
                      key + "_sees": (ctx[at] - n[at])[:, None] + 1 + t})
    return {k: torch.from_numpy(np.ascontiguousarray(v)).to(DEVICE).to(
        torch.bool if v.dtype == bool else torch.int64) for k, v in index.items()}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["kind"] == "adjust":
        return s
    if own:
        from intel_kivi_hybrid_amd import _C
        s["plan"] = _C.paged_plan(
            torch.from_numpy(s["table"]), s["ctx"].tolist(), s["n"].tolist(),
            page_size=case["page"], num_pages=s["k_pages"].shape[0], q_heads=case["Hq"],
            kv_heads=case["Hkv"], head_dim=case["D"], dtype=DTYPES[case["dtype"]],
            device=DEVICE, cache_dtype=torch.int8)
    else:
        s["at"] = _host(case, s)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _values(s):
    """What the pools' codes stand for."""
    return [s[x + "_pages"].view(*s[x + "_scales"].shape, BLOCK, -1)
            * s[x + "_scales"][..., None, None] for x in ("k", "v")]


def run(state):
    case, s = state["case"], state
    kind = case["kind"]
    if own:
        from intel_kivi_hybrid_amd import _C
        if kind == "append":
            q = _C.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["plan"], q=s["q"],
                                cos=s["cos"], sin=s["sin"],
                                interleaved=case["style"] == "neighbours", q_norm=s["q_norm"],
                                k_norm=s["k_norm"], eps=1e-6, k_scales=s["k_scales"],
                                v_scales=s["v_scales"])
            return [q, *_values(s)]
        if kind == "attend":
            return _C.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["plan"],
                                      k_scales=s["k_scales"], v_scales=s["v_scales"])
        return _C.adjust_logits(s["logits"], tokens=s["tokens"], lengths=s["lengths"],
                                prompt_lengths=s["prompts"], repetition_penalty=s["repetition"],
                                presence_penalty=s["presence"],
                                frequency_penalty=s["frequency"], bias_ids=s["bias_ids"],
                                bias=s["bias"], allowed=s["allowed"])
    return {"append": _plain_append, "attend": _plain_attend, "adjust": _plain_adjust}[kind](s)


def _plain_rows(x, w, cos, sin, neighbours, dt):
    """Norm and rotation of head rows ``[T, H, D]``."""
    y = x.to(dt)
    if w is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.to(dt)
    if cos is None:
        return y
    r = 2 * cos.shape[-1]
    c, s = cos[:, None, :], sin[:, None, :]
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if neighbours else (y[..., :r // 2], y[..., r // 2:r])
    out = y.clone()
    if neighbours:
        out[..., 0:r:2], out[..., 1:r:2] = a * c - b * s, b * c + a * s
    else:
        out[..., :r // 2], out[..., r // 2:r] = a * c - b * s, b * c + a * s
    return out


def _plain_store(s, rows, codes, scales):
    at = s["at"]
    Hkv, D, size = s["case"]["Hkv"], s["case"]["D"], s["case"]["page"] // BLOCK
    top = torch.zeros(len(at["held"]), Hkv, dtype=rows.dtype, device=DEVICE)
    top = top.scatter_reduce(0, at["block"][:, None].expand(-1, Hkv), rows.abs().amax(-1), "amax")
    need = _scale_for(top)
    old = scales[at["block_page"], :, at["block_in_page"]]
    held = at["held"][:, None] > 0
    new = torch.where(held, torch.maximum(old, need), need)
    scales[at["block_page"], :, at["block_in_page"]] = new
    blocks = codes.view(len(codes), Hkv, size, BLOCK, D)
    x = blocks[at["block_page"], :, at["block_in_page"]]
    again = torch.round(x.float() * (old / new)[..., None, None]).to(torch.int8)
    keep = torch.arange(BLOCK, device=DEVICE) < at["held"][:, None]
    blocks[at["block_page"], :, at["block_in_page"]] = torch.where(keep[:, None, :, None], again, x)
    codes[at["page"], :, at["off"]] = torch.round(rows / new[at["block"]][..., None]).to(torch.int8)


def _plain_append(s):
    at, neighbours = s["at"], s["case"]["style"] == "neighbours"
    cos = sin = None
    if s["cos"] is not None:
        cos, sin = s["cos"][at["pos"]], s["sin"][at["pos"]]
    q = _plain_rows(s["q"], s["q_norm"], cos, sin, neighbours, torch.float32).to(s["q"].dtype)
    # (keys in fp64: a code goes by which side of a border its value lies on)
    k = _plain_rows(s["k"], s["k_norm"], cos, sin, neighbours, torch.float64)
    _plain_store(s, k, s["k_pages"], s["k_scales"])
    _plain_store(s, s["v"].float(), s["v_pages"], s["v_scales"])
    return [q, *_values(s)]


def _plain_some(s, key, out):
    """Attention of the sequences with one new token, or with more, each side
    padded to its longest."""
    at, case = s["at"], s["case"]
    if key + "_row" not in at:
        return
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    row, pages = at[key + "_row"], at[key + "_pages"]
    S, n = row.shape
    k, v = ((s[x + "_pages"][pages].float().view(*pages.shape, Hkv, -1, BLOCK, D)
             * s[x + "_scales"][pages][..., None, None]).transpose(1, 2).reshape(S, Hkv, -1, D)
            for x in ("k", "v"))
    # query rows of a kv head: [token, head of its group]
    rows = s["q"][row].float().view(S, n, Hkv, -1, D).transpose(1, 2).reshape(S, Hkv, -1, D)
    sc = torch.matmul(rows, k.transpose(2, 3).contiguous())
    sees = at[key + "_sees"].repeat_interleave(Hq // Hkv, 1)[:, None, :, None]
    sc = (sc * D ** -0.5).masked_fill_(torch.arange(k.shape[2], device=DEVICE) >= sees,
                                       float("-inf"))
    sc = torch.exp(sc - sc.amax(-1, keepdim=True))
    o = torch.matmul(sc, v) / sc.sum(-1, keepdim=True)
    o = o.view(S, Hkv, n, -1, D).transpose(1, 2).reshape(S, n, Hq, D).to(out.dtype)
    live = at[key + "_live"]
    out[row[live]] = o[live]


def _plain_attend(s):
    out = torch.empty_like(s["q"])
    _plain_some(s, "one", out)
    _plain_some(s, "more", out)
    return out


def _plain_adjust(s):
    x = s["logits"].float()
    B, V = x.shape
    L = s["tokens"].shape[1]
    t = torch.arange(L, device=DEVICE)[None, :]
    live = t < s["lengths"][:, None]
    said = live & (t >= s["prompts"][:, None])
    seen = torch.zeros(B, V, device=DEVICE).scatter_add_(1, s["tokens"], live.float()) > 0
    count = torch.zeros(B, V, device=DEVICE).scatter_add_(1, s["tokens"], said.float())
    r, p, f = (torch.as_tensor(s[k], dtype=torch.float32, device=DEVICE).expand(B)[:, None]
               for k in ("repetition", "presence", "frequency"))
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - (f * count + p * (count > 0))
    if s["bias_ids"] is not None:
        x = x.scatter_add(1, s["bias_ids"], s["bias"])
    if s["allowed"] is not None:
        v = torch.arange(V, device=DEVICE)
        x = x.masked_fill((s["allowed"][:, v // 32] >> (v % 32)) & 1 == 0, float("-inf"))
    return x.to(s["logits"].dtype)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    size = SIZES[case["dtype"]]
    if case["kind"] == "adjust":
        n = case["B"] * case["V"]
        rows = case["B"] * (8 * case["history"] * 3 / 4 + 12 * case["biased"])
        # a quotient, a product and two sums for each logit
        return {"bytes": 2 * n * size + (n / 8 if case["mask"] else 0) + rows, "flops": 4 * n}
    n, ctx = _lengths(case)
    T = int(n.sum())
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if case["kind"] == "append":
        blocks = int(((ctx - 1) // BLOCK - (ctx - n) // BLOCK + 1).sum())
        turned = T * (Hq + Hkv)
        flops = (3 * turned * case["rotary"] + (4 * turned * D if case["norm"] else 0)
                 + 4 * T * Hkv * D)
        table = 4 * case["rotary"] * len(np.unique(np.concatenate(
            [np.arange(c - m, c) for c, m in zip(ctx, n)])))
        return {"bytes": T * D * (Hq * 2 * size + 2 * Hkv * (size + 1)) + 8 * blocks * Hkv + table,
                "flops": flops}
    pairs = int((n * ctx - n * (n - 1) // 2).sum())
    held = int((ctx * D + -(-ctx // BLOCK) * 4).sum())
    return {"bytes": 2 * held * Hkv + 2 * T * Hq * D * size, "flops": 4 * pairs * Hq * D}


# ---------------------------------------------------------------------------
# the definition in fp64
# ---------------------------------------------------------------------------
def _exact_adjust(s):
    x = s["logits"].double().cpu().numpy()
    B, V = x.shape
    host = {k: v.cpu().numpy() if torch.is_tensor(v) else v for k, v in s.items()
            if k != "logits"}
    get = {k: np.broadcast_to(np.asarray(host[k], dtype=np.float64), (B,))
           for k in ("repetition", "presence", "frequency")}
    for b in range(B):
        row = x[b]
        words = host["tokens"][b, :host["lengths"][b]]
        ids = np.unique(words)
        y = row[ids]
        row[ids] = np.where(y > 0, y / get["repetition"][b], y * get["repetition"][b])
        ids, count = np.unique(words[host["prompts"][b]:], return_counts=True)
        row[ids] -= get["frequency"][b] * count + get["presence"][b]
        if host["bias_ids"] is not None:
            np.add.at(row, host["bias_ids"][b], host["bias"][b].astype(np.float64))
        if host["allowed"] is not None:
            bits = np.unpackbits(host["allowed"][b].view(np.uint8), bitorder="little")[:V]
            row[bits == 0] = -np.inf
    return torch.from_numpy(x).to(DEVICE)


def _exact_pool(case, s, x, which, where):
    """The pool of ``which`` after the rows ``x [T, Hkv, D]`` in fp64."""
    codes, scales = s[which + "_pages"].double(), s[which + "_scales"].double()
    held = codes.view(*scales.shape, BLOCK, -1)
    page, block, slot, first = where
    # each block's tokens, by slot, beside what it held
    got, at = np.unique(np.stack([page, block]), axis=1, return_inverse=True)
    at = torch.from_numpy(at.reshape(-1)).to(DEVICE)
    rows = torch.full((got.shape[1], BLOCK, case["Hkv"], case["D"]), float("nan"),
                      dtype=torch.float64, device=DEVICE)
    rows[at, torch.from_numpy(slot).to(DEVICE)] = x
    keep = torch.zeros(got.shape[1], dtype=torch.int64, device=DEVICE)
    keep[at] = torch.from_numpy(first).to(DEVICE)
    rows = rows.transpose(1, 2)
    p, j = (torch.from_numpy(g).to(DEVICE) for g in got)
    before, old = held[p, :, j], scales[p, :, j]
    top = torch.nan_to_num(rows, nan=0.0).abs().amax((2, 3))
    need = torch.exp2(torch.ceil(torch.log2(top / 127.0)).clamp_min(-126.0))
    # (log2's own rounding, at a power of two)
    need = torch.where(top > 127.0 * need, 2 * need, need)
    need = torch.where((top <= 63.5 * need) & (need > LEAST), need / 2, need)
    new = torch.where((keep > 0)[:, None], torch.maximum(old, need), need)
    kept = torch.round(before * (old / new)[..., None, None]) * new[..., None, None]
    put = torch.round(rows / new[..., None, None]) * new[..., None, None]
    value = held * scales[..., None, None]
    old_slot = torch.arange(BLOCK, device=DEVICE)[None, :] < keep[:, None]
    # (slots behind the last token keep their codes, which now stand for others)
    free = before * new[..., None, None]
    value[p, :, j] = torch.where(torch.isnan(put), torch.where(
        old_slot[:, None, :, None], kept, free), put)
    return value.view(codes.shape)


def _exact_append(case, s):
    pos = np.concatenate([np.arange(c - m, c) for c, m in zip(s["ctx"], s["n"])])
    seq = np.repeat(np.arange(len(s["n"])), s["n"])
    start = np.repeat(s["ctx"] - s["n"], s["n"])
    where = (s["table"][seq, pos // case["page"]].astype(np.int64),
             pos % case["page"] // BLOCK, pos % BLOCK,
             np.maximum(0, np.minimum(BLOCK, start - pos // BLOCK * BLOCK)))
    half = case["rotary"] // 2
    i = torch.arange(half, device=DEVICE)
    first, second = (2 * i, 2 * i + 1) if case["style"] == "neighbours" else (i, i + half)

    def rows(x, w):
        y = x.double()
        if w is not None:
            y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w.double()
        if half:
            # (the tables are inputs: their fp32 values)
            at = torch.from_numpy(pos).to(DEVICE)
            turn = torch.complex(s["cos"].double(), s["sin"].double())[at][:, None, :]
            z = torch.complex(y[..., first], y[..., second]) * turn
            y = y.index_copy(2, first, z.real).index_copy(2, second, z.imag)
        return y
    return [rows(s["q"], s["q_norm"]),
            _exact_pool(case, s, rows(s["k"], s["k_norm"]), "k", where),
            _exact_pool(case, s, s["v"].double(), "v", where)]


def _exact_attend(case, s):
    Hq, Hkv, D, ps = case["Hq"], case["Hkv"], case["D"], case["page"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    at = 0
    for b in range(len(s["n"])):
        n, c = int(s["n"][b]), int(s["ctx"][b])
        p = torch.arange(c, device=DEVICE)
        page = torch.from_numpy(s["table"][b]).to(DEVICE).long()[p // ps]
        for h in range(Hkv):
            k, v = (s[x + "_pages"][page, h, p % ps].double()
                    * s[x + "_scales"][page, h, p % ps // BLOCK].double()[:, None]
                    for x in ("k", "v"))
            kt = k.t().contiguous()
            for j in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                z = s["q"][at:at + n, j].double().mm(kt) / math.sqrt(D)
                z = torch.where(p[None, :] <= p[c - n:, None], z, float("-inf"))
                out[at:at + n, j] = torch.softmax(z, -1).mm(v)
        at += n
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "adjust":
        return _exact_adjust(s)
    if case["kind"] == "append":
        return _exact_append(case, s)
    return _exact_attend(case, s)
