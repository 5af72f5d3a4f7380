"""GPU tests of attention over 8-bit pages whose blocks' scales are far apart, against
float64: blocks of zeros have the smallest scale, and what a row sees, or sees first, may
be nothing else; and bounds by each weight's own scale."""

import pytest
import torch

from tests.paged8_helpers import BLOCK, EPS, filled_pool8, values
from tests.paged_helpers import make_table, sequence_kv

pytestmark = pytest.mark.gpu
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda:0"
TYPES = pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "f16", "f32"])


def _c():
    from intel_kivi_hybrid_amd import _C
    return _C


class Case:
    """A step's inputs, and what they should make."""

    def __init__(self, lens, page, dtype, Hq, Hkv, D, seed=0, spread=0):
        self.page, self.lens = page, lens
        self.table, self.pool, self.ctx, self.new = make_table(lens, page, seed)
        self.kc, self.ks = filled_pool8(self.table, self.pool, self.ctx, Hkv, D, page, seed + 1)
        self.vc, self.vs = filled_pool8(self.table, self.pool, self.ctx, Hkv, D, page, seed + 5,
                                        spread)
        g = torch.Generator().manual_seed(seed + 2)
        self.q = (1.5 * torch.randn(sum(self.new), Hq, D, generator=g)).to(dtype)
        self.plan = _c().paged_plan(self.table, self.ctx, self.new, page_size=page,
                                    num_pages=self.pool, q_heads=Hq, kv_heads=Hkv, head_dim=D,
                                    dtype=dtype, device=DEV, cache_dtype=torch.int8)

    def blocks(self, s, first, last):
        """Pages and blocks of them that positions first .. last - 1 of sequence s lie in."""
        for b in range(first // BLOCK, -(-min(last, self.ctx[s]) // BLOCK)):
            yield int(self.table[s, b * BLOCK // self.page]), b * BLOCK % self.page // BLOCK

    def set_values(self, first, last, scale, zero):
        """Scale of the values of positions first .. last - 1 (whole blocks) of every
        sequence, and codes of 0."""
        for s in range(len(self.ctx)):
            for page, j in self.blocks(s, first, last):
                self.vs[page, :, j] = scale
                if zero:
                    self.vc[page, :, j * BLOCK:(j + 1) * BLOCK] = 0

    def run(self, **kw):
        return _c().paged_attention(self.q.cuda(), self.kc.cuda(), self.vc.cuda(), self.plan,
                                    k_scales=self.ks.cuda(), v_scales=self.vs.cuda(), **kw)

    def expected(self, heads=None):
        """Outputs of the kv heads in float64, and each element's bound: that of
        attention8_tolerance (tests/paged8_helpers.py) with the largest product of a weight
        and its own value's scale, which the kernels keep between 2^12 and 2^15; a row of
        values below 2^-52 has its weights' exponents rounded to 2^-18 (they reach 2^77
        there): 2^-18 of each weight and of their sum; a weight below 2^-112 of its row's
        largest, of a value whose scale is above 2^36, may count for less, down to nothing;
        and what lies below 2^-126 may come out as 0."""
        T, Hq, D = self.q.shape
        Hkv = self.kc.shape[1]
        hg, dtype = Hq // Hkv, self.q.dtype
        kp, vp = values(self.kc, self.ks), values(self.vc, self.vs)
        sp = self.vs.double().repeat_interleave(BLOCK, -1)[..., None]
        ref = torch.zeros(T, Hq, D, dtype=torch.float64)
        tol = torch.zeros_like(ref)
        eps, u, at = EPS[dtype], 2.0 ** -24, 0
        half = 2.0 ** -22 if dtype == FF else 2.0 ** -11
        least = 2.0 ** -25 if dtype == HF else 2.0 ** -126
        for s, (c, n) in enumerate(zip(self.ctx, self.new)):
            if n == 0:
                continue
            k, v, sc = (sequence_kv(x, self.table, s, c, self.page) for x in (kp, vp, sp))
            sees = torch.arange(c) <= torch.arange(c - n, c)[:, None]
            for h in heads if heads is not None else range(Hkv):
                for i in range(h * hg, (h + 1) * hg):
                    q = self.q[at:at + n, i].double()
                    z = (q @ k[h].T) * D ** -0.5
                    p = torch.softmax(z.masked_fill(~sees, -float("inf")), -1)
                    o, mag = p @ v[h], p @ v[h].abs()
                    size = ((q.abs() @ k[h].abs().T) * D ** -0.5 * sees).amax(-1, keepdim=True)
                    largest = (p * sc[h, :, 0]).amax(-1, keepdim=True)
                    moved = 2 * ((2 * D + 10) * u * size + (3 * c + 16) * u)
                    most = p.amax(-1, keepdim=True)
                    quiet = 2 * 2.0 ** -18 * (largest < 2.0 ** -50 * most)
                    far = p * ((p < 2.0 ** -112 * most) & (sc[h, :, 0] > 2.0 ** 36))
                    ref[at:at + n, i] = o
                    tol[at:at + n, i] = (eps / 2 * o.abs()
                                         + ((half + moved + quiet) * mag
                                            + far @ v[h].abs() + 127 * c * 2.0 ** -37 * largest)
                                         * (1 + eps) + least)
            at += n
        return ref, tol

    def check(self, name, heads=None, **kw):
        o = self.run(**kw).double().cpu()
        ref, tol = self.expected(heads)
        if heads is not None:
            hg = self.q.shape[1] // self.kc.shape[1]
            rows = [h * hg + i for h in heads for i in range(hg)]
            o, ref, tol = o[:, rows], ref[:, rows], tol[:, rows]
        err = (o - ref).abs()
        print(f"[quiet] {name} {self.q.dtype} D={self.q.shape[2]} worst "
              f"{float((err / tol).max()):.3f} of the bound", flush=True)
        assert bool((err <= tol).all()), (name, float((err / tol).max()))
        return o


# rows of a kv head: single tokens; more than 16; single tokens beside these
FEW = [(0, 1), (15, 1), (63, 1), (64, 1), (299, 1), (2999, 1)]
MANY = [(0, 20), (0, 70), (280, 20), (2961, 40)]
BOTH = [(0, 1), (63, 1), (2999, 1), (300, 33)]
ROWS = pytest.mark.parametrize("lens", [FEW, MANY, BOTH], ids=["few", "many", "both"])


@TYPES
@ROWS
@pytest.mark.parametrize("D", [64, 128, 256])
def test_contexts_of_zeros(hip_device, D, lens, dtype):
    """Zeros as an append leaves them, and in a pool that was cleared."""
    case = Case(lens, 32, dtype, 8, 2, D, seed=D)
    for scale in (2.0 ** -126, 0.0):
        case.set_values(0, 1 << 20, scale, zero=True)
        assert bool((case.check(f"zeros {scale}") == 0).all())


@TYPES
@ROWS
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("last", [16, 64, 300, 1 << 20])
def test_values_next_to_zero(hip_device, last, D, lens, dtype):
    """The first positions, or all of them, with scales from the smallest on, codes as
    they are."""
    for e in (-126, -120, -116, -115, -100, -60):
        case = Case(lens, 64, dtype, 4, 1, D, seed=-e)
        case.set_values(0, last, 2.0 ** e, zero=False)
        case.check(f"2^{e} up to {last}")


@TYPES
@ROWS
@pytest.mark.parametrize("first", [64, 128, 1024])
def test_zeros_behind_values(hip_device, first, lens, dtype):
    """And values behind zeros, in one piece of the context or in several."""
    for back in (False, True):
        case = Case(lens, 16, dtype, 8, 2, 128, seed=first)
        case.set_values(*((0, first) if back else (first, 1 << 20)), 2.0 ** -126, zero=True)
        case.check(f"zeros {'before' if back else 'from'} {first}")


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "f16"])
@pytest.mark.parametrize("lens,page,Hq,Hkv,D", [
    ([(3900, 512)], 64, 64, 32, 128),
    ([(1100, 340), (2100, 341), (2003, 511), (1500, 171)], 16, 96, 32, 112)], ids=[0, 1])
def test_tiles_of_256_rows(hip_device, lens, page, Hq, Hkv, D, dtype):
    case = Case(lens, page, dtype, Hq, Hkv, D, seed=3)
    assert case.plan._info[8] > 0 and case.plan._info[9] == 0
    for last in (64, 1 << 20):
        for scale, zero in ((2.0 ** -116, False), (2.0 ** -126, True), (0.0, True)):
            case.set_values(0, last, scale, zero)
            o = case.check(f"{scale} up to {last}", heads=[0, 17, Hkv - 1])
            assert last == 64 or not zero or bool((o == 0).all())


@TYPES
@ROWS
@pytest.mark.parametrize("lead", [30, 60, 90, 105, 120, 150])
def test_a_leading_score_of_zero_values(hip_device, lead, lens, dtype):
    """One position's score leads all others of its row by `lead` log2 units, and its
    block's values are zeros."""
    D = 64
    for at in (3, 200):
        case = Case(lens, 32, dtype, 4, 1, D, seed=lead)
        case.q[..., 0] = 8
        for s, c in enumerate(case.ctx):
            for j, (page, b) in enumerate(case.blocks(s, 0, c)):
                case.kc[page, 0, b * BLOCK:(b + 1) * BLOCK, 0] = 0
                if j != at // BLOCK or at >= c:
                    continue
                # (a lead of this many units over a key without the channel)
                scale = lead / 1.4426950408889634 / (8 * D ** -0.5 * 127)
                case.ks[page, 0, b] = scale
                case.kc[page, 0, b * BLOCK:(b + 1) * BLOCK] = 0
                case.kc[page, 0, b * BLOCK + at % BLOCK, 0] = 127
                case.vs[page, 0, b] = 2.0 ** -126
                case.vc[page, 0, b * BLOCK:(b + 1) * BLOCK] = 0
        case.check(f"lead {lead} at {at}")


@TYPES
@ROWS
def test_loud_values_far_below_a_quiet_leader(hip_device, lens, dtype):
    """Scales from one end of the range to the other: of 2^e beside a leader of zeros
    that takes nearly all of the weight, and beside values of a scale of 1, with their
    scores or 300 log2 units below."""
    top = 4 if dtype == HF else 115
    for e in (top, top // 2 + 5):
        for lead, below in ((40, 0), (100, 0), (200, 0), (40, 300), (115, 300)):
            case = Case(lens, 16, dtype, 4, 1, 64, seed=e)
            case.q[..., 0] = 8
            for s, c in enumerate(case.ctx):
                for j, (page, b) in enumerate(case.blocks(s, 0, c)):
                    case.kc[page, 0, b * BLOCK:(b + 1) * BLOCK, 0] = 0
                    case.vs[page, 0, b] = 2.0 ** e if j % 3 == 1 else 1.0
                    if j % 3 == 1 and below:
                        case.kc[page, 0, b * BLOCK:(b + 1) * BLOCK] = 0
                        case.kc[page, 0, b * BLOCK:(b + 1) * BLOCK, 0] = -127
                        case.ks[page, 0, b] = below / 1.4426950408889634 / 127
                    if j % 3 == 0:
                        case.kc[page, 0, b * BLOCK:(b + 1) * BLOCK] = 0
                        case.kc[page, 0, b * BLOCK + 2, 0] = 127
                        case.ks[page, 0, b] = lead / 1.4426950408889634 / 127
                        case.vs[page, 0, b] = 2.0 ** -126
                        case.vc[page, 0, b * BLOCK:(b + 1) * BLOCK] = 0
            case.check(f"2^{e} {lead} and {below} below")


@pytest.mark.parametrize("dtype,spread", [(BF, 3), (BF, 10), (BF, 20), (HF, 3), (HF, 10), (FF, 3),
                                          (FF, 10), (FF, 20)])
@pytest.mark.parametrize("n", [1, 70])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_whose_weights_lie_on_quiet_blocks(hip_device, D, n, dtype, spread):
    """Beside blocks up to 2^41 times louder, whose keys have tiny scores: the bound is by
    the largest product of a weight and its own scale."""
    case = Case([(200, n), (90, n)], 32, dtype, 4, 2, D, seed=8, spread=spread)
    for s, c in enumerate(case.ctx):
        for page, j in case.blocks(s, 0, c):
            for h in range(2):
                if case.vs[page, h, j] > case.vs[int(case.table[s, 0]), h, 0]:
                    case.kc[page, h, j * BLOCK:(j + 1) * BLOCK] = 0
    case.q *= 4
    case.check(f"spread {spread}")


@TYPES
@ROWS
@pytest.mark.parametrize("e", [4, 12, 14, 15, 16, 17, 20, 40])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_beyond_the_whole_numbers_of_fp32(hip_device, sign, e, lens, dtype):
    """Scores of 2^(e + 14) (in log2), where one position's leads the others', which lie 0
    or below: what sees it has its values, loud, ordinary or quiet, by weights that are 1
    or 0, off by the weight's and the output's rounding alone; a position before it has
    the mean of the others.  From 2^29 on fp32's numbers are 32 apart and more: a maximum
    that weights are formed against cannot lie up to 75 below the largest score there, as
    values below 2^-51 ask for, so those may count for less, down to nothing."""
    D = 64
    for scale in (2.0 ** -126, 2.0 ** -60, 1.0, 4.0 if dtype == HF else 2.0 ** 21):
        case = Case(lens, 32, dtype, 4, 1, D, seed=e)
        case.q[:] = 0
        case.q[..., 0] = 1024
        case.kc[:] = 0
        leads = []
        for s, c in enumerate(case.ctx):
            lead = (c - case.new[s]) * 2 // 3 + (3 if case.new[s] > 5 else 0)
            leads += [c - case.new[s] + i >= lead for i in range(case.new[s])]
            for page, b in case.blocks(s, 0, c):
                case.kc[page, 0, b * BLOCK:(b + 1) * BLOCK, 0] = -100 if sign < 0 else 0
                case.ks[page, 0, b] = 2.0 ** e
                case.vs[page, 0, b] = 1.0 if scale < 1 else scale
            page, b = next(case.blocks(s, lead // BLOCK * BLOCK, lead + 1))
            case.kc[page, 0, b * BLOCK + lead % BLOCK, 0] = -64 if sign < 0 else 127
            case.vs[page, 0, b] = scale
        o = case.run().double().cpu()
        ref, tol = case.expected()
        half = 2.0 ** -22 if dtype == FF else 2.0 ** -11
        least = 2.0 ** -25 if dtype == HF else 2.0 ** -126
        one = (EPS[dtype] / 2 + half + 32 * 2.0 ** -24) * ref.abs() + least
        if e >= 15 and scale < 2.0 ** -51:
            one += ref.abs()
        tol = torch.where(torch.tensor(leads)[:, None, None], one, tol)
        err = (o - ref).abs()
        assert bool((err <= tol).all()), (e, scale, float((err / tol).max()))


@TYPES
def test_an_appended_context_of_zeros(hip_device, dtype):
    """Through the append: a prompt of zeros, then tokens of zeros, then one of numbers."""
    C, page, Hq, Hkv, D = _c(), 32, 8, 2, 64
    table = torch.arange(8, dtype=torch.int32)[None]
    pools = [torch.randint(-128, 128, (8, Hkv, page, D), dtype=torch.int8, device=DEV)
             for _ in range(2)]
    scales = dict(k_scales=torch.full((8, Hkv, page // 16), float("nan"), device=DEV),
                  v_scales=torch.full((8, Hkv, page // 16), float("nan"), device=DEV))
    g = torch.Generator().manual_seed(1)
    at = 0
    for n in (50, 1, 1, 80, 1, 1):
        at += n
        k = torch.randn(n, Hkv, D, generator=g).to(dtype).cuda()
        v = torch.zeros_like(k) if at < 134 else torch.ones_like(k)
        q = torch.randn(n, Hq, D, generator=g).to(dtype).cuda()
        plan = C.paged_plan(table, [at], [n], page_size=page, num_pages=8, q_heads=Hq,
                            kv_heads=Hkv, head_dim=D, dtype=dtype, device=DEV,
                            cache_dtype=torch.int8)
        C.paged_append(k, v, *pools, plan, **scales)
        o = C.paged_attention(q, *pools, plan, **scales)
        assert bool((o == 0).all() if at < 134 else ((o > 0) & (o < 1)).all()), (n, at)
