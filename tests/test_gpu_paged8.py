"""Pages of 8-bit codes and norms of heads on the GPU (lmrs_b200.paged) against 64-bit restatements (tests/paged8_oracle.py).  Scales that a call must not read are NaN, codes of e4m3 that it must not
read are NaN as well, and what it must not write is looked at afterwards."""
import math
import random

import pytest

torch = pytest.importorskip("torch")
import paged8_oracle as oracle  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INT8, E4M3 = torch.int8, torch.float8_e4m3fn
P_EPS = {BF16: 2.0 ** -11, F16: 2.0 ** -11, F32: 0.0}   # what rounding a weight to float16 costs at most


@pytest.fixture(scope="module")
def paged(gpu_lib):
    from lmrs_b200 import paged
    return paged


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def laid_out(t, how):
    """the same values on the GPU: packed, with gaps between rows and heads, or one element off every 16-byte boundary"""
    if how == "packed":
        return t.cuda()
    n, h, d = t.shape
    pad, off = (8, 0) if how == "gaps" else (3, 1)
    big = torch.full((n * (h + 1) * (d + pad) + 16,), math.nan, dtype=t.dtype, device="cuda")
    view = big[off:].as_strided((n, h, d), ((h + 1) * (d + pad), d + pad, 1), off)
    view.copy_(t)
    return view


# ---- norms -----------------------------------------------------------------------------------------------------------------------------------
NORM = [  # rows, heads, size, rot, sections, layout, far, weight of every head?
    (1, 1, 2, 2, [1], "halves", 10, False), (1, 40, 64, 64, [32], "halves", 8192, True), (5, 3, 128, 128, [16, 24, 24], "halves", 2 ** 31 - 300, True), (7, 2, 96, 48, [8, 16], "pairs", 100000, False),
    (3, 5, 80, 20, [1, 2, 3, 4], "halves", 1000, False), (300, 9, 64, 64, [16, 16], "pairs", 64, True), (2, 4, 256, 256, [128], "pairs", 1000000, False), (17, 1, 33, 10, [5], "pairs", 77, True),
    (6, 3, 40, 8, [1, 3], "halves", 5, False), (1000, 40, 128, 128, [22, 21, 21], "halves", 130000, True), (9, 4, 256, 16, [8], "halves", 99, False), (4, 7, 1, 0, [], "halves", 1, True), (4, 7, 130, 0, [], "halves", 1, None),
    (50, 3, 256, 64, [32], "halves", 4000, True),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("how", ["packed", "gaps", "odd"])
@pytest.mark.parametrize("case", NORM, ids=str)
def test_norm_rope(paged, case, how, dtype):
    n, heads, size, rot, sections, layout, far, each = case
    g = gen(n + heads)
    x = (torch.randn(n, heads, size, generator=g) * 3).to(dtype)
    x[0, 0] = 0.0   # (a head of zeros stays one)
    weight = None if each is None else torch.randn((heads, size) if each else (size,), generator=g)
    rope = pos = None
    freq, axis = [], []
    if rot:
        pos = (far + torch.randint(0, 200, (len(sections), n), generator=g)).to(torch.int32)
        rope = paged.RopeAxes.sections(rot, 10000.0, sections, "cycle", layout)
        freq, axis = [10000.0 ** (-2.0 * j / rot) for j in range(rot // 2)], list(rope._c.axis[:rot // 2])
    for eps in (1e-6, 0.5):
        normed = oracle.norm(x, weight, eps)
        want = oracle.turn(normed, pos, freq, axis, layout) if rot else normed
        tol = oracle.norm_tolerance(normed, want, freq, layout, dtype)
        if rot:
            tol += normed.abs().amax(-1, keepdim=True) * float(pos.double().abs().max()) * 2.0 ** -51   # the oracle's 64-bit angles
        xg, pg = laid_out(x, how), None if not rot else pos.cuda() if how == "packed" else pos.T.contiguous().cuda().T
        wg = None if weight is None else weight.cuda()
        if how == "gaps" and each:   # rows of weights with a gap, off every 16-byte boundary
            wg = torch.zeros(heads, size + 3, device="cuda")[:, 1:size + 1]
            wg.copy_(weight)
        got = paged.norm_rope(xg, wg, pg, rope, eps)
        assert ((got.cpu().double() - want).abs() <= tol).all(), float(((got.cpu().double() - want).abs() - tol).max())
        assert torch.equal(xg.cpu(), x)
        out = laid_out(torch.zeros_like(x), how)
        assert paged.norm_rope(xg, wg, pg, rope, eps, out=out) is out and torch.equal(out.contiguous(), got)
    paged.norm_rope(xg, wg, pg, rope, 0.5, out=xg)   # in place
    assert torch.equal(xg.contiguous(), got)


def test_norm_rope_of_nothing_and_of_what_is_not_finite(paged):
    rope = paged.RopeAxes([1.0])
    assert paged.norm_rope(torch.zeros(0, 3, 8, device="cuda"), None, torch.zeros(1, 0, dtype=torch.int32, device="cuda"), rope).shape == (0, 3, 8)
    assert paged.norm_rope(torch.zeros(2, 0, 8, device="cuda")).shape == (2, 0, 8)
    x = torch.randn(4, 2, 64, generator=gen(1))
    x[1, 0, 3], x[2, 1, 40] = math.nan, math.inf
    got = paged.norm_rope(x.cuda(), None, torch.arange(4, dtype=torch.int32, device="cuda"), rope).cpu()
    bad = torch.zeros(4, 2, dtype=torch.bool)
    bad[1, 0] = bad[2, 1] = True   # a head, and no other
    assert torch.isfinite(got[~bad]).all() and torch.isnan(got[bad]).any(-1).all()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("size", [16, 64, 96, 200, 256, 33])
def test_norms_of_heads_far_from_one(paged, size, dtype):
    """squares up to the ends of float32 (elements of 2^59, or 2^-60 with no eps beside them), heads of all sizes in a row; without an eps and with one"""
    n, heads = 7, 9
    g = gen(size)
    x = torch.randn(n, heads, size, generator=g)
    for r, f in enumerate((57, 40, 20, -20, -40, -57)):
        x[r, ::2 + r % 2] *= 2.0 ** f
    x[2, 1, 1:], x[3, 1, :-1] = 0.0, 0.0   # (one element only)
    x = x.to(dtype)
    weight = torch.randn(heads, size, generator=g)
    pos = torch.randint(0, 200, (1, n), generator=g).to(torch.int32)
    rot = size // 8 * 4
    rope = paged.RopeAxes.sections(rot, 10000.0)
    freq = [10000.0 ** (-2.0 * j / rot) for j in range(rot // 2)]
    codes, scales = torch.zeros(n, 8, 1, size, dtype=INT8, device="cuda"), torch.ones(n, 1, 1, device="cuda")
    pages = paged.QuantPages(codes, codes.clone(), scales, scales.clone())
    batch = paged.Batch(torch.ones(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")[:, None])
    k = torch.ones(n, 1, size, dtype=dtype, device="cuda")
    for eps in (0.0, 1e-30, 1e-6, 1e30):
        normed = oracle.norm(x, weight, eps)
        want = oracle.turn(normed, pos, freq, [0] * len(freq), "halves")
        tol = oracle.norm_tolerance(normed, want, freq, "halves", dtype) + normed.abs().amax(-1, keepdim=True) * 200 * 2.0 ** -51
        for how in ("packed", "gaps", "odd"):
            for got in (paged.norm_rope(laid_out(x, how), weight.cuda(), pos.cuda(), rope, eps), paged.append(pages, batch, k, k, rope=rope, pos=pos.cuda(), q=laid_out(x, how), q_norm=weight.cuda(), eps=eps)):
                assert ((got.cpu().double() - want).abs() <= tol).all(), (eps, how, float(((got.cpu().double() - want).abs() - tol).max()))


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("layout", ["halves", "pairs"])
def test_elements_that_do_not_turn_pass_unchanged(paged, layout, dtype):
    """an infinity, a NaN or a zero's sign behind the pairs that turn: the elements beside it know nothing of it, wherever the rows lie"""
    n, heads, size, rot = 12, 3, 64, 16
    x = torch.randn(n, heads, size, generator=gen(1)).to(dtype)
    for r, e in enumerate((16, 19, 23, 40, 63)):
        x[r, 0, e], x[r + 5, 1, e] = math.inf, math.nan
    x[10:] = -0.0
    pos = torch.arange(5, 5 + n, dtype=torch.int32, device="cuda")
    rope = paged.RopeAxes.sections(rot, 10000.0, layout=layout)
    codes, scales = torch.zeros(n, 8, 1, size, dtype=INT8, device="cuda"), torch.ones(n, 1, 1, device="cuda")
    pages = paged.QuantPages(codes, codes.clone(), scales, scales.clone())
    batch = paged.Batch(torch.ones(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")[:, None])
    k = torch.ones(n, 1, size, dtype=dtype, device="cuda")
    normed = []
    for how in ("packed", "gaps", "odd"):
        q = paged.append(pages, batch, k, k, rope=rope, pos=pos, q=laid_out(x, how)).cpu()
        assert torch.equal(torch.isnan(q), torch.isnan(x)) and torch.equal(torch.isinf(q), torch.isinf(x))
        bits = torch.int32 if dtype == F32 else torch.int16
        assert torch.equal(torch.where(torch.isnan(x), 0, q.view(bits))[..., rot:], torch.where(torch.isnan(x), 0, x.view(bits))[..., rot:])
        normed.append(paged.norm_rope(laid_out(x, how), None, pos, rope).cpu())
        spoilt = torch.zeros(n, heads, size, dtype=torch.bool)
        spoilt[torch.isinf(x)] = True                    # (an infinite element over an infinite root; the others of its head over it are 0)
        spoilt[torch.isnan(x).any(-1)] = True            # (a NaN is in the root of the whole head)
        assert torch.equal(torch.isnan(normed[-1]), spoilt)


# ---- a batch: sequences of given lengths in a pool whose unused places hold NaN ------------------------------------------------------------------
class Made:
    def __init__(self, paged, seed, dtype, form, lens, counts, page, block, kv_heads, group, size, prefix=0, one_each=False, order="pshd", tail=0, bad=(), empty=False):
        r = random.Random(seed)
        g = gen(seed)
        self.lens, self.dtype, self.form, self.prefix_len, self.one_each, self.block = lens, dtype, form, prefix, one_each, block
        held, shared = [-(-max(0, n) // page) for n in lens], -(-prefix // page)
        pages = sum(held) + shared + 3
        ids = list(range(pages))
        r.shuffle(ids)
        width = max([1] + held) + r.randrange(3)
        self.tables = torch.full((len(lens), width), -1, dtype=torch.int32)
        at = shared
        for b, h in enumerate(held):
            self.tables[b, :h] = torch.tensor(ids[at:at + h], dtype=torch.int32)
            at += h
        self.prefix = torch.tensor(ids[:shared], dtype=torch.int32)
        for b, i, value in bad:   # entries that are no pages
            if b < 0:
                self.prefix[i] = value
            else:
                self.tables[b, i] = value
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        self.rows, self.n = (None if one_each else torch.tensor(starts, dtype=torch.int32)), starts[-1] + tail
        empty_code = 99.0 if form == INT8 else math.nan
        self.k = torch.full((pages, page, kv_heads, size), empty_code, dtype=torch.float64)
        self.v = self.k.clone()
        self.ks = torch.full((pages, page // block, kv_heads), math.nan, dtype=torch.float64)
        self.vs = self.ks.clone()
        self.page, self.heads, self.kv_heads, self.size, self.counts = page, kv_heads * group, kv_heads, size, counts
        spread = 40.0 if form == INT8 else 100.0
        for b, (table, n) in enumerate([(self.tables[b], n) for b, n in enumerate(lens)] + [(self.prefix, prefix)]):
            for x in range(max(0, n - (counts[b] if empty and b < len(counts) else 0))):   # (empty: what the call appends is not there yet)
                p = oracle.place(table, pages, page, x)
                if p:
                    for codes, scales in ((self.k, self.ks), (self.v, self.vs)):
                        codes[p] = oracle.nearest(spread * torch.randn(kv_heads, size, generator=g).double(), form)
                        if x % block == 0:
                            scales[p[0], p[1] // block] = (torch.exp(1.5 * torch.randn(kv_heads, generator=g)) / spread).float().double()
        self.q = (1.5 * torch.randn(self.n, self.heads, size, generator=g)).to(dtype)
        self.order = order
        self.paged = paged

    def on_gpu(self):
        perm, back = ["pshd".index(c) for c in self.order], [self.order.index(c) for c in "pshd"]
        k, v = (t.float().to(self.form).permute(perm).contiguous().cuda().permute(back) for t in (self.k, self.v))
        ks, vs = self.ks.float().cuda(), self.vs.float().permute(2, 0, 1).contiguous().cuda().permute(1, 2, 0)
        pages = self.paged.QuantPages(k, v, ks, vs)
        batch = self.paged.Batch(torch.tensor(self.lens, dtype=torch.int32).cuda(), self.tables.cuda(), rows=None if self.rows is None else self.rows.cuda(),
                                 max_rows=max([1] + self.counts) if self.rows is not None else 1, prefix=self.prefix.cuda() if self.prefix_len else None, prefix_len=self.prefix_len)
        return pages, batch

    def wanted(self, scale=None, cap=0.0):
        scale = self.size ** -0.5 if scale is None else scale
        return oracle.attention(self.k, self.v, self.ks, self.vs, self.block, self.lens, self.tables, self.rows, self.prefix, self.prefix_len, self.q, scale, cap, P_EPS[self.dtype])

    def check(self, out, lse, scale=None, cap=0.0):
        want, want_lse, tol, tol_lse = self.wanted(scale, cap)
        seen = ~torch.isnan(want_lse)   # rows of some sequence
        got, got_lse = out.cpu().double(), lse.cpu().double()
        assert torch.equal(torch.isinf(got_lse)[seen], torch.isinf(want_lse)[seen])
        assert ((got - want).abs() <= tol)[seen].all(), float(((got - want).abs() - tol)[seen].max())
        finite = seen & torch.isfinite(want_lse)
        assert ((got_lse - want_lse).abs() <= tol_lse)[finite].all(), float(((got_lse - want_lse).abs() - tol_lse)[finite].max())


# ---- appending and reading back ------------------------------------------------------------------------------------------------------------------
APPEND = [  # tokens held, rows, page, block, kv heads, group, size, rot, sections, layout, prefix, positions given, norms
    ([1], None, 16, 16, 1, 1, 64, 64, [32], "halves", 0, False, True), ([9, 0, 33, 16], None, 16, 8, 2, 4, 64, 32, [8, 8], "pairs", 20, False, True),
    ([700], None, 64, 16, 8, 4, 128, 128, [16, 24, 24], "halves", 0, True, False), ([20, 5, 0, 60], [20, 2, 1, 33], 7, 7, 2, 3, 96, 96, [20, 28], "halves", 33, True, True),
    ([300, 300], [257, 300], 64, 64, 1, 2, 48, 20, [10], "pairs", 0, False, True), ([4, 9], [6, 9], 1, 1, 3, 1, 256, 256, [128], "halves", 5, False, False),
    ([50] * 70, None, 48, 12, 2, 2, 64, 64, [10, 11, 11], "pairs", 100, True, True), ([12, 30], [5, 5], 4, 2, 1, 1, 33, 10, [5], "halves", 0, False, True),
    ([8] * 9, [3] * 9, 8, 4, 5, 1, 16, 2, [1], "pairs", 0, True, False), ([150, 40], [140, 7], 128, 128, 17, 1, 32, 0, [], "halves", 0, False, True), ([40], [21], 16, 1, 2, 2, 80, 80, [40], "halves", 3, False, True),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("form", [INT8, E4M3], ids=str)
@pytest.mark.parametrize("how", ["packed", "gaps", "odd"])
@pytest.mark.parametrize("case", APPEND, ids=lambda c: f"{len(c[0])}x{max(c[0])}-page{c[2]}-block{c[3]}-{c[4]}x{c[6]}-rot{c[7]}{c[9]}")
def test_append_and_read(paged, case, how, form, dtype):
    lens, counts, page, block, kv, group, size, rot, sections, layout, prefix, given, norms = case
    m = Made(paged, len(lens) + size, dtype, form, lens, counts or [1] * len(lens), page, block, kv, group, size, prefix, one_each=counts is None, order="phsd" if how == "gaps" else "pshd",
             tail=0 if counts is None else 3, empty=True)
    g = gen(3)
    k, v = (torch.exp(torch.randn(m.n, kv, 1, generator=g)) * torch.randn(m.n, kv, size, generator=g) for _ in range(2))
    k, v = k.to(dtype), v.to(dtype)
    v[0] = 0.0   # (the smallest scale)
    k_norm, q_norm = (torch.randn(size, generator=g), torch.randn(m.heads, size, generator=g)) if norms else (None, None)
    eps = 1e-5
    pos = torch.randint(0, 100000, (max(1, len(sections)), m.n), generator=g).to(torch.int32)
    rope = paged.RopeAxes.sections(rot, 10000.0, sections, "cycle", layout) if rot else None
    freq, axis = [10000.0 ** (-2.0 * j / rot) for j in range(rot // 2)], list(rope._c.axis[:rot // 2]) if rot else []
    pages, batch = m.on_gpu()
    where, index, mine = [], torch.zeros(m.n, dtype=torch.int64), []
    for b, (first, c, have) in enumerate(oracle.spans(lens, m.rows, m.n)):
        where.append([])
        for i in range(c):
            index[first + i] = have - c + i
            p = oracle.place(m.tables[b], len(m.k), page, have - c + i)
            where[-1].append(None if p is None else (*p, have - c + i))
        mine.append((first, c))
    real = sum(c for _, c in mine)
    use = (pos if given else (prefix + index).to(torch.int32).expand(max(1, len(sections)), -1))
    k_in, q_in = (oracle.norm(k, k_norm, eps), oracle.norm(m.q, q_norm, eps)) if norms else (k.double(), m.q.double())
    k_in, q_want = (oracle.turn(k_in, use, freq, axis, layout), oracle.turn(q_in, use, freq, axis, layout)) if rot else (k_in, q_in)
    args = [laid_out(t, how) for t in (k, v, m.q)]
    # the same call twice, from the same pool
    q_out = None
    if rot or norms:
        q_out = torch.full(m.q.shape, 7.0, dtype=dtype, device="cuda") if how == "packed" else laid_out(torch.full_like(m.q, 7.0), how)
    more = dict(k_norm=k_norm.cuda(), q_norm=q_norm.cuda(), eps=eps) if norms else {}
    before = m.k.clone(), m.v.clone(), m.ks.clone(), m.vs.clone()
    call = dict(rope=rope, pos=pos.cuda() if given and rot else None, q=None if q_out is None else args[2], q_out=q_out, **more)
    assert paged.append(pages, batch, args[0], args[1], **call) is q_out
    got = [t.cpu() for t in (pages.k, pages.v, pages.k_scale, pages.v_scale)]
    slack = 2.0 ** -38 if rot else 2.0 ** -46 if norms else 0.0   # (of the largest value: the oracle's 64-bit angles, the order of 64-bit sums)
    for codes, scales, x, off, left in ((m.k, m.ks, k_in, slack, got[2]), (m.v, m.vs, v.double(), 0.0, got[3])):
        for (first, c), w in zip(mine, where):
            oracle.put(codes, scales, block, form, x[first:first + c], w, off, left)
    for codes, left in ((m.k, got[0]), (m.v, got[1])):
        left = left.float().double()
        sure = ~torch.isnan(codes)
        assert torch.equal(left[sure], codes[sure]), int((left != codes)[sure].sum())
    unsure = sum(int((torch.isnan(codes) & ~torch.isnan(old)).sum()) for codes, old in ((m.k, before[0]), (m.v, before[1])))
    assert unsure <= 1
    for scales, left in ((m.ks, got[2]), (m.vs, got[3])):
        assert torch.equal(left.double().nan_to_num(-1.0), scales.nan_to_num(-1.0))
    if q_out is not None:
        tol = oracle.norm_tolerance(q_in, q_want, freq, layout, dtype) + q_in.abs().amax(-1, keepdim=True) * 100200 * 2.0 ** -51
        assert ((q_out.cpu().double() - q_want).abs() <= tol)[:real].all()
        assert (q_out[real:] == 7.0).all()
    # again: nothing moves, queries in place
    paged.append(pages, batch, args[0], args[1], **{**call, "q_out": None if q_out is None else args[2]})
    for t, old in zip((pages.k, pages.v, pages.k_scale, pages.v_scale), got):
        assert torch.equal(t.cpu().contiguous().view(torch.uint8), old.contiguous().view(torch.uint8))
    if q_out is not None:
        assert torch.equal(args[2][:real], q_out[:real])
    # what the sequences hold, read back; in rows laid out as the call's
    lens0 = [max(0, n) for n in lens]
    starts = [sum(lens0[:b]) for b in range(len(lens) + 1)]
    every = paged.Batch(batch.lens, batch.tables, rows=torch.tensor(starts, dtype=torch.int32).cuda(), max_rows=max(1, *lens0))
    kk, vv = (laid_out(torch.full((starts[-1] + 2, kv, size), 5.0, dtype=dtype), how) for _ in range(2))
    assert paged.read(pages, every, rows=starts[-1] + 2, k=kk, v=vv)[0] is kk
    for values, codes, scales in ((kk, pages.k.cpu().float(), pages.k_scale.cpu()), (vv, pages.v.cpu().float(), pages.v_scale.cpu())):
        for b, n in enumerate(lens0):
            for x in range(n):
                p = oracle.place(m.tables[b], len(m.k), page, x)
                assert torch.equal(values[starts[b] + x].cpu(), (codes[p] * scales[p[0], p[1] // block][:, None]).to(dtype))
        assert (values[-2:] == 5.0).all()
    new = paged.read(pages, batch, rows=m.n, dtype=F32)   # the call's own rows
    for (first, c), w in zip(mine, where):
        for i, p in enumerate(w):
            assert torch.equal(new[1][first + i].cpu(), torch.zeros(kv, size) if p is None else got[1][p[0], p[1]].float() * got[3][p[0], p[1] // block][:, None])


LONG = [  # (windows of several rows, queries in a kernel of their own) tokens held, rows, page, block, kv heads, group, size, rot, layout, prefix, weights of norms, entries that are no pages
    ([900, 40, 0, 700, 333, 5, 500], [800, 60, 3, 700, 333, 5, 499], 32, 16, 2, 8, 64, 64, "halves", 20, "each", [(0, 20, -1)]), ([1200, 130], [1150, 77], 16, 4, 3, 2, 64, 24, "halves", 0, None, []),
    ([2600, 77], [2433, 20], 64, 64, 1, 8, 128, 32, "pairs", 0, "all", []), ([1000] * 3, [990, 1000, 991], 48, 12, 2, 3, 96, 96, "halves", 7, "each", [(1, 0, 10 ** 6)]), ([1500, 9], [1400, 30], 8, 1, 2, 2, 33, 10, "halves", 0, "all", []),
    ([3] * 500, [3, 2, 1, 5, 4] * 100, 16, 8, 4, 4, 128, 64, "halves", 0, "each", []), ([4000, 17], [3900, 17], 128, 128, 2, 2, 64, 16, "pairs", 0, None, []),
]


@pytest.mark.parametrize("form, dtype, how", [(INT8, BF16, "packed"), (E4M3, F16, "packed"), (E4M3, F32, "packed"), (INT8, F32, "odd")], ids=str)
@pytest.mark.parametrize("case", LONG, ids=lambda c: f"{len(c[0])}x{sum(c[1])}-page{c[2]}-block{c[3]}-{c[4]}x{c[5]}x{c[6]}-rot{c[7]}{c[8]}")
def test_append_of_many_rows(paged, case, how, form, dtype):
    """blocks that begin before a window of rows and end behind it, starts inside a block, padding in front and rows behind; the attention that follows reads the same queries and codes as a later one"""
    lens, counts, page, block, kv, group, size, rot, layout, prefix, norms, bad = case
    m = Made(paged, len(lens) + size, dtype, form, lens, counts, page, block, kv, group, size, prefix, tail=5, empty=True, bad=bad)
    g = gen(4)
    k, v = ((torch.exp(torch.randn(m.n, kv, 1, generator=g)) * torch.randn(m.n, kv, size, generator=g)).to(dtype) for _ in range(2))
    k_norm, q_norm = (None, None) if norms is None else (torch.randn(kv, size, generator=g), torch.randn(m.heads, size, generator=g)) if norms == "each" else (torch.randn(size, generator=g), torch.randn(size, generator=g))
    rope = paged.RopeAxes.sections(rot, 10000.0, layout=layout)
    freq, axis = [10000.0 ** (-2.0 * j / rot) for j in range(rot // 2)], [0] * (rot // 2)
    (pages, batch), twin = m.on_gpu(), m.on_gpu()[0]
    spans = oracle.spans(lens, m.rows, m.n)
    where, index = [], torch.zeros(m.n, dtype=torch.int64)
    for b, (first, c, have) in enumerate(spans):
        index[first:first + c] = have - c + torch.arange(c)
        where.append([None if p is None else (*p, have - c + i) for i in range(c) for p in [oracle.place(m.tables[b], len(m.k), page, have - c + i)]])
    real, use = sum(c for _, c, _ in spans), (prefix + index).to(torch.int32)[None]
    k_in, q_in = (oracle.norm(k, k_norm, 1e-5), oracle.norm(m.q, q_norm, 1e-5)) if norms else (k.double(), m.q.double())
    k_want, q_want = oracle.turn(k_in, use, freq, axis, layout), oracle.turn(q_in, use, freq, axis, layout)
    args = [laid_out(t, how) for t in (k, v, m.q)]
    more = dict(k_norm=k_norm.cuda(), q_norm=q_norm.cuda(), eps=1e-5) if norms else {}
    q_out = torch.full(m.q.shape, 7.0, dtype=dtype, device="cuda")
    paged.append(pages, batch, args[0], args[1], rope=rope, q=args[2], q_out=q_out, **more)
    attend = size % 16 == 0
    at_once = paged.attention(pages, batch, q_out) if attend else None
    torch.cuda.synchronize()
    if attend:
        assert torch.equal(paged.attention(pages, batch, q_out)[:real], at_once[:real])
    got = [t.cpu() for t in (pages.k, pages.v, pages.k_scale, pages.v_scale)]
    before = m.k.clone(), m.v.clone()
    for codes, scales, x, off, left in ((m.k, m.ks, k_want, 2.0 ** -38, got[2]), (m.v, m.vs, v.double(), 0.0, got[3])):
        for (first, c, _), w in zip(spans, where):
            oracle.put(codes, scales, block, form, x[first:first + c], w, off, left)
    if not norms:   # (keys' elements that pass are the inputs themselves: 24 bits over 24 bits, which 64 tell from the middle of two codes)
        for (first, _, _), w in zip(spans, where):
            for i, p in enumerate(w):
                if p is not None:
                    m.k[p[0], p[1], :, rot:] = oracle.nearest(k[first + i, :, rot:].double() / m.ks[p[0], p[1] // block][:, None], form)
    for codes, left in ((m.k, got[0]), (m.v, got[1])):
        left, sure = left.float().double(), ~torch.isnan(codes)
        assert torch.equal(left[sure], codes[sure]), int((left != codes)[sure].sum())
    assert sum(int((torch.isnan(codes) & ~torch.isnan(old)).sum()) for codes, old in zip((m.k, m.v), before)) <= 1
    for scales, left in ((m.ks, got[2]), (m.vs, got[3])):
        assert torch.equal(left.double().nan_to_num(-1.0), scales.nan_to_num(-1.0))
    tol = oracle.norm_tolerance(q_in, q_want, freq, layout, dtype) + q_in.abs().amax(-1, keepdim=True) * 4100 * 2.0 ** -51
    assert ((q_out.cpu().double() - q_want).abs() <= tol)[:real].all() and (q_out[real:] == 7.0).all()
    # captured, over a pool as the first one was, with the queries in place: the same bits
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.append(twin, batch, args[0], args[1], rope=rope, q=args[2], q_out=args[2], **more)
        again = paged.attention(twin, batch, args[2]) if attend else None
    graph.replay()
    assert torch.equal(args[2][:real], q_out[:real])
    for t, left in zip((twin.k, twin.v, twin.k_scale, twin.v_scale), got):
        assert torch.equal(t.cpu().contiguous().view(torch.uint8), left.contiguous().view(torch.uint8))
    if attend:
        assert torch.equal(again[:real], at_once[:real])


@pytest.mark.parametrize("form", [INT8, E4M3], ids=str)
def test_token_by_token(paged, form):
    """a sequence that grows by single tokens: a block's scale is the largest so far, and codes follow it"""
    g = gen(4)
    n, kv, size, page, block = 41, 2, 64, 16, 8
    x = torch.exp(1.5 * torch.randn(n, kv, 1, generator=g)) * torch.randn(n, kv, size, generator=g)
    tables = torch.tensor([[2, 0, 1]], dtype=torch.int32)
    codes = [torch.zeros(4, page, kv, size, dtype=torch.float64) for _ in range(2)]
    scales = [torch.full((4, page // block, kv), 123.0, dtype=torch.float64) for _ in range(2)]   # (of a block that is begun: not looked at)
    pages = paged.QuantPages(*(c.float().to(form).cuda() for c in codes), *(s.float().cuda() for s in scales))
    lens = torch.zeros(1, dtype=torch.int32, device="cuda")
    batch = paged.Batch(lens, tables.cuda())
    for i in range(n):
        lens.fill_(i + 1)
        paged.append(pages, batch, x[i:i + 1].cuda(), -x[i:i + 1].cuda())
        for c, s, sign, left in zip(codes, scales, (1.0, -1.0), (pages.k_scale.cpu(), pages.v_scale.cpu())):
            oracle.put(c, s, block, form, sign * x[i:i + 1].double(), [(int(tables[0, i // page]), i % page, i)], 0.0, left)
    for t, c in zip((pages.k, pages.v), codes):
        assert torch.equal(t.cpu().float().double(), c)
    for t, s in zip((pages.k_scale, pages.v_scale), scales):
        assert torch.equal(t.cpu().double(), s)


@pytest.mark.parametrize("form", [INT8, E4M3], ids=str)
def test_ties_go_to_even(paged, form):
    """a largest size of the format's own makes the scale 1: values in the middle of two numbers"""
    numbers = oracle.numbers(form)[0].float()
    middle = (numbers[1:] + numbers[:-1]) / 2
    x = torch.zeros(4, 1, 256)
    x.view(-1)[:2 * len(middle):2] = middle
    x.view(-1)[1:2 * len(middle):2] = torch.nextafter(middle, torch.full_like(middle, 1e9))
    x[:, :, 255] = numbers[-1]
    k = torch.zeros(1, 4, 1, 256).to(form).cuda()
    pages = paged.QuantPages(k, k.clone(), torch.zeros(1, 4, 1, device="cuda"), torch.zeros(1, 1, 1, device="cuda").expand(1, 1, 1).repeat(1, 4, 1))
    batch = paged.Batch(torch.tensor([4], dtype=torch.int32).cuda(), torch.zeros(1, 1, dtype=torch.int32).cuda(), rows=torch.tensor([0, 4], dtype=torch.int32).cuda(), max_rows=4)
    paged.append(pages, batch, x.cuda(), x.cuda())
    assert (pages.k_scale == 1.0).all()
    for t in (pages.k, pages.v):
        assert torch.equal(t.cpu()[0].float().double(), oracle.nearest(x.double(), form))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("how", ["packed", "odd"])
@pytest.mark.parametrize("form", [INT8, E4M3], ids=str)
def test_inputs_next_to_the_middle_of_two_codes(paged, form, how, dtype):
    """all 8 bits of mantissa of elements against all of the largest: quotients that only the scale's rounding keeps from the middle"""
    x = torch.zeros(128, 1, 256)
    x[:, 0, :128] = torch.arange(128, 256)
    x[:, 0, 128:255] = torch.arange(129, 256) / 64.0
    x[:, 0, 255] = 256 + 2 * torch.arange(128)   # the largest of each token
    x[1::2] *= -0.37109375   # (another 8 bits' worth of scales: rounded to the type)
    x = x.to(dtype)
    k = torch.zeros(8, 16, 1, 256).to(form).cuda()
    pages = paged.QuantPages(k, k.clone(), torch.zeros(8, 16, 1, device="cuda"), torch.zeros(8, 16, 1, device="cuda"))
    batch = paged.Batch(torch.tensor([128], dtype=torch.int32).cuda(), torch.arange(8, dtype=torch.int32).cuda()[None], rows=torch.tensor([0, 128], dtype=torch.int32).cuda(), max_rows=128)
    paged.append(pages, batch, laid_out(x, how), laid_out(-x, how))
    for t, s, sign in ((pages.k, pages.k_scale, 1.0), (pages.v, pages.v_scale, -1.0)):
        scale = s.cpu().double().view(128, 1, 1)
        assert ((scale[:, 0, 0] - x.double().abs().amax((1, 2)) / oracle.MOST[form]).abs() <= scale[:, 0, 0] * 2.0 ** -24).all()
        assert torch.equal(t.cpu().float().double().view(128, 1, 256), oracle.nearest(sign * x.double() / scale, form))


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("form", [INT8, E4M3], ids=str)
def test_what_is_not_finite_and_what_is_far_from_one(paged, form, dtype):
    x = torch.randn(6, 2, 64, generator=gen(5))
    x[0, 0, 3], x[1, 1, 60], x[2, 0] = math.nan, -math.inf, 0.0
    x[3], x[4], x[5, 0] = x[3] * 1e-25, x[4] * 1e30, 1e38
    x = x.to(dtype)
    k = torch.zeros(3, 2, 2, 64).to(form).cuda()
    pages = paged.QuantPages(k, k.clone(), torch.ones(3, 2, 2, device="cuda"), torch.ones(3, 2, 2, device="cuda"))
    batch = paged.Batch(torch.tensor([6], dtype=torch.int32).cuda(), torch.tensor([[0, 2, 1]], dtype=torch.int32).cuda(), rows=torch.tensor([0, 6], dtype=torch.int32).cuda(), max_rows=6)
    paged.append(pages, batch, x.cuda(), x.cuda())
    kk, vv = (t.cpu().double() for t in paged.read(pages, batch, rows=6, dtype=F32))
    most = oracle.MOST[form]
    for got, scale in ((kk, pages.k_scale.cpu()), (vv, pages.v_scale.cpu())):
        assert torch.isnan(got[0, 0]).all() and torch.isnan(got[1, 1]).all() and torch.isfinite(got[0, 1]).all() and torch.isfinite(got[1, 0]).all()
        assert (got[2, 0] == 0).all() and scale[2, 0, 0] == 2.0 ** -60   # (token 2: page 2, its first block)
        assert (got[3] == 0).all()                                       # less than half a step of the smallest scale
        assert scale[1, 0].max() == 2.0 ** 60 and (got[4].abs() <= most * 2.0 ** 60).all() and torch.equal(got[5, 0], torch.full((64,), most * 2.0 ** 60, dtype=torch.float64))


def test_reading_rows_that_are_not_counted(paged):
    """the rows of k and v, or one a sequence; a batch with rows of its own is refused, since fewer of them would be other tokens"""
    m = Made(paged, 7, BF16, INT8, [10, 40, 33], [4, 1, 9], 16, 4, 2, 1, 64)
    pages, batch = m.on_gpu()
    with pytest.raises(paged.LmrsError, match="rows"):
        paged.read(pages, batch)
    want = paged.read(pages, batch, rows=m.n)
    k, v = (torch.full((m.n + 2, 2, 64), 5.0, dtype=BF16, device="cuda") for _ in range(2))
    paged.read(pages, batch, k=k, v=v)
    for got, w in ((k, want[0]), (v, want[1])):
        assert torch.equal(got[:m.n], w) and (got[m.n:] == 5.0).all()
    last = paged.read(pages, paged.Batch(batch.lens, batch.tables))
    for got, w in zip(last, want):
        assert torch.equal(got, w[[3, 4, 13]])


def test_entries_that_are_no_pages_and_lengths_beyond_the_table(paged):
    m = Made(paged, 3, BF16, INT8, [40, 20, 64], [9, 20, 64], 16, 4, 2, 1, 64, bad=[(0, 2, -1), (1, 0, 2 ** 31 - 1), (2, 1, 1000), (2, 3, -2 ** 31)], empty=True)
    pages, batch = m.on_gpu()
    x = torch.randn(m.n, 2, 64, generator=gen(1)).to(BF16).cuda()
    old = pages.k.clone()
    paged.append(pages, batch, x, x)
    k, v = paged.read(pages, batch, rows=m.n)
    at = [None if m.tables[b, i // 16] < 0 or m.tables[b, i // 16] >= len(m.k) else (int(m.tables[b, i // 16]), i % 16) for b, c in enumerate(m.counts) for i in range(m.lens[b] - c, m.lens[b])]
    for r, p in enumerate(at):
        assert (k[r] == 0).all() if p is None else not torch.equal(k[r], torch.zeros_like(k[r]))
        if p:
            old[p] = pages.k[p]
    page = int(m.tables[0, 1])
    old[page, 12:15] = pages.k[page, 12:15]   # (tokens 28 .. 30 of the first sequence share a scale with token 31, which the call appends)
    assert torch.equal(old, pages.k)
    batch.lens.copy_(torch.tensor([2 ** 31 - 1, -2 ** 31, 10 ** 9], dtype=torch.int32))   # nowhere to write to or to read from
    paged.append(pages, batch, x + 1, x)
    assert torch.equal(old, pages.k)
    k, v = paged.read(pages, batch, rows=m.n)
    assert (k == 0).all() and (v == 0).all()


# ---- attention -----------------------------------------------------------------------------------------------------------------------------------
SINGLE = [  # tokens held, page, block, kv heads, group, size, prefix, order of the pool
    ([1], 16, 16, 1, 1, 64, 0, "pshd"), ([1], 1, 1, 2, 4, 64, 1, "pshd"), ([63, 64, 65], 16, 8, 2, 4, 64, 0, "pshd"), ([130, 1, 17, 0, 255], 7, 7, 3, 2, 128, 33, "pshd"), ([700], 64, 16, 8, 4, 64, 0, "phsd"),
    ([5, 0, 0, 9], 5, 1, 2, 5, 96, 129, "pshd"), ([200, 300], 128, 32, 1, 16, 256, 64, "phsd"), ([33, 40], 3, 3, 4, 1, 16, 70, "pshd"), ([90] * 20, 32, 4, 2, 8, 128, 200, "sphd"), ([257, 3], 48, 12, 1, 20, 64, 100, "hpsd"),
    ([40, 41, 42], 16, 2, 5, 3, 48, 513, "pshd"), ([64] * 3, 64, 64, 2, 12, 208, 64, "pshd"), ([2000, 1], 16, 16, 1, 6, 128, 0, "pshd"), ([10] * 70, 16, 16, 1, 4, 64, 400, "pshd"), ([0, 0], 16, 16, 1, 2, 64, 50, "pshd"),
    ([12] * 40, 8, 8, 2, 8, 128, 1100, "phsd"), ([100] * 3, 16, 4, 1, 64, 64, 300, "pshd"), ([150] * 9, 16, 16, 2, 16, 256, 260, "pshd"), ([127, 128, 129, 385], 16, 16, 2, 4, 128, 0, "pshd"),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("form", [INT8, E4M3], ids=str)
@pytest.mark.parametrize("case", SINGLE, ids=lambda c: f"{len(c[0])}x{max(c[0])}-page{c[1]}-block{c[2]}-{c[3]}x{c[4]}x{c[5]}-prefix{c[6]}-{c[7]}")
def test_attention_of_single_tokens(paged, case, form, dtype):
    lens, page, block, kv, group, size, prefix, order = case
    m = Made(paged, len(lens) + size, dtype, form, lens, [1] * len(lens), page, block, kv, group, size, prefix, one_each=True, order=order)
    pages, batch = m.on_gpu()
    out, lse = paged.attention(pages, batch, m.q.cuda(), return_lse=True)
    m.check(out, lse)
    assert torch.equal(paged.attention(pages, batch, laid_out(m.q, "odd"), out=laid_out(m.q, "odd")).contiguous(), out)   # the same bits, wherever the rows lie
    assert torch.equal(paged.attention(pages, batch, laid_out(m.q, "gaps")), out)


MANY = [  # tokens held, rows of the call, page, block, kv heads, group, size, prefix
    ([3], [3], 16, 16, 1, 1, 64, 0), ([100, 40, 9], [100, 3, 9], 16, 8, 2, 4, 64, 0), ([70, 300, 65], [1, 130, 65], 7, 1, 2, 3, 128, 35), ([20, 0, 90], [20, 1, 33], 32, 16, 1, 8, 96, 200),
    ([150, 150], [64, 65], 64, 64, 3, 2, 256, 64), ([5, 2, 40], [7, 0, 40], 4, 2, 2, 2, 64, 65), ([260], [257], 48, 24, 1, 2, 128, 0), ([9] * 30, [3] * 30, 16, 4, 2, 2, 64, 130), ([33], [33], 1, 1, 1, 5, 32, 10),
    ([130, 200], [128, 129], 16, 16, 1, 4, 128, 700),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("form", [INT8, E4M3], ids=str)
@pytest.mark.parametrize("case", MANY, ids=lambda c: f"{len(c[0])}x{max(c[0])}-rows{max(c[1])}-page{c[2]}-block{c[3]}-{c[4]}x{c[5]}x{c[6]}-prefix{c[7]}")
def test_attention_of_several_rows(paged, case, form, dtype):
    """(a sequence with more rows than tokens: the first ones are padding; rows behind the last sequence stay as they are)"""
    lens, counts, page, block, kv, group, size, prefix = case
    m = Made(paged, len(lens) + size, dtype, form, lens, counts, page, block, kv, group, size, prefix, tail=2)
    pages, batch = m.on_gpu()
    out = torch.full((m.n, m.heads, size), 7.0, dtype=dtype, device="cuda")
    got, lse = paged.attention(pages, batch, m.q.cuda(), out=out, return_lse=True)
    assert got is out
    m.check(out, lse)
    assert (out[-2:] == 7.0).all()


LARGE = [  # (many rows against the same keys: tensor-core products) tokens held, rows of the call or None, page, block, kv heads, group, size, prefix
    ([40] * 29 + [0, 7], None, 16, 16, 2, 8, 128, 4500), ([200, 130], [200, 65], 32, 8, 2, 2, 64, 700), ([300], [257], 48, 12, 1, 2, 112, 0), ([90, 70, 5], [80, 64, 5], 7, 7, 1, 1, 128, 133),
    ([10] * 9, None, 8, 8, 4, 4, 256, 3700), ([10] * 9, None, 8, 8, 4, 8, 256, 4000), ([3] * 40, None, 16, 4, 4, 4, 64, 6700), ([64, 129], [64, 128], 1, 1, 1, 4, 64, 65), ([150, 260], [33, 140], 64, 64, 2, 3, 208, 515), ([130] * 3, [70] * 3, 128, 128, 1, 5, 128, 1000),
]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("form", [INT8, E4M3], ids=str)
@pytest.mark.parametrize("case", LARGE, ids=lambda c: f"{len(c[0])}x{max(c[0])}-rows{max(c[1] or [1])}-page{c[2]}-block{c[3]}-{c[4]}x{c[5]}x{c[6]}-prefix{c[7]}")
def test_attention_of_many_rows(paged, case, form, dtype):
    lens, counts, page, block, kv, group, size, prefix = case
    m = Made(paged, len(lens) + size, dtype, form, lens, counts or [1] * len(lens), page, block, kv, group, size, prefix, one_each=counts is None, tail=0 if counts is None else 2,
             order="phsd" if page == 64 else "pshd", bad=[(-1, 3, -1)] if page == 32 else [(0, 0, 10 ** 6)] if page == 48 else [])
    pages, batch = m.on_gpu()
    for cap in (0.0, 30.0):
        out = torch.full((m.n, m.heads, size), 7.0, dtype=dtype, device="cuda")
        got, lse = paged.attention(pages, batch, m.q.cuda(), out=out, softcap=cap, return_lse=True)
        m.check(out, lse, cap=cap)
        assert counts is None or (out[-2:] == 7.0).all()
        assert torch.equal(paged.attention(pages, batch, laid_out(m.q, "odd"), softcap=cap)[:m.n - 2], out[:m.n - 2])
    out, lse = paged.attention(pages, batch, m.q.cuda(), scale=-0.3, return_lse=True)
    m.check(out, lse, scale=-0.3)


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("form", [INT8, E4M3], ids=str)
def test_attention_scale_and_cap(paged, form, dtype):
    m = Made(paged, 5, dtype, form, [100, 37, 200], [1, 37, 70], 16, 8, 2, 4, 64, 90)
    pages, batch = m.on_gpu()
    for scale, cap in ((1.0, 0.0), (0.125, 20.0), (0.5, 1.5), (0.0, 0.0), (-0.125, 0.0), (4.0, 50.0)):
        out, lse = paged.attention(pages, batch, m.q.cuda(), scale=scale, softcap=cap, return_lse=True)
        m.check(out, lse, scale, cap)


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_attention_with_missing_pages(paged, dtype):
    """what lies there is not seen, wherever the entry is; a row all of whose pages are missing sees nothing"""
    lens = [100, 64, 16, 40]
    bad = [(0, 2, -1), (0, 4, 2 ** 31 - 1), (1, 0, -2 ** 31), (1, 3, 1000), (2, 0, -5), (-1, 1, 99999), (-1, 3, -1)]
    for one, prefix, form in ((True, 80, INT8), (False, 80, E4M3), (True, 0, E4M3), (False, 0, INT8)):
        m = Made(paged, 3, dtype, form, lens, [1] * 4 if one else [1, 30, 16, 40], 16, 8, 2, 4, 64, prefix, one_each=one, bad=[x for x in bad if prefix or x[0] >= 0])
        out, lse = paged.attention(*m.on_gpu(), m.q.cuda(), return_lse=True)
        m.check(out, lse)
        if not prefix:
            row = 2 if one else 31
            assert (out[row] == 0).all() and (lse[row] == -math.inf).all()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_attention_beyond_the_table_and_a_wrong_max_rows(paged, dtype):
    """a length that the table does not reach: what it does reach counts.  max_rows chooses kernels, and nothing else"""
    m = Made(paged, 4, dtype, INT8, [40, 70, 200], [1, 1, 1], 16, 8, 1, 2, 64, 20, one_each=True)
    pages, batch = m.on_gpu()
    m.tables = m.tables[:, :3]
    short = paged.Batch(batch.lens, m.tables.cuda(), prefix=batch.prefix, prefix_len=20)   # 48 tokens at most
    m.check(*paged.attention(pages, short, m.q.cuda(), return_lse=True))
    batch.lens.copy_(torch.tensor([2 ** 31 - 1, -2 ** 31, 0], dtype=torch.int32))
    out, lse = paged.attention(pages, short, m.q.cuda(), return_lse=True)
    assert (out[1:] == 0).all() and (lse[1:] == -math.inf).all()   # (the first row sees all that the table has, scales of blocks that hold nothing among it)
    empty = paged.Batch(batch.lens, m.tables[:, :0].cuda(), prefix=batch.prefix, prefix_len=20)
    batch.lens.fill_(5)
    m.lens, m.tables = [5, 5, 5], m.tables[:, :0]
    m.check(*paged.attention(pages, empty, m.q.cuda(), return_lse=True))
    m = Made(paged, 5, dtype, E4M3, [300, 90], [150, 70], 16, 8, 1, 2, 64, 90)
    pages, batch = m.on_gpu()
    for most in (1, 7, 10 ** 6):
        batch = paged.Batch(batch.lens, batch.tables, rows=batch.rows, max_rows=most, prefix=batch.prefix, prefix_len=90)
        m.check(*paged.attention(pages, batch, m.q.cuda(), return_lse=True))
        x = torch.randn(m.n, 1, 64, generator=gen(most)).to(dtype).cuda()
        paged.append(pages, batch, x, x)
        k, v = paged.read(pages, batch, rows=m.n, dtype=dtype)
        step = x.float().abs().amax() / 16   # (half a step of e4m3, and what the block's older scale makes of it)
        assert ((k.float() - x.float()).abs() <= step + 448 * 2.0 ** -4 * pages.k_scale[~torch.isnan(pages.k_scale)].max()).all() and torch.isfinite(v).all()
        m = Made(paged, 5, dtype, E4M3, [300, 90], [150, 70], 16, 8, 1, 2, 64, 90)
        pages = m.on_gpu()[0]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("form", [INT8, E4M3], ids=str)
def test_scales_that_are_not_finite(paged, form, dtype):
    """a block that reads as NaN reaches the rows that see it, and no other: not those of other sequences, nor those before it in its own"""
    m = Made(paged, 6, dtype, form, [130, 80, 50], [100, 80, 1], 16, 4, 2, 2, 64, 70)
    for codes, b, x, g in ((m.vs, 0, 60, 1), (m.ks, 0, 96, 0), (m.vs, 1, 76, 0)):
        p = oracle.place(m.tables[b], len(m.k), 16, x)
        codes[p[0], p[1] // 4, g] = math.nan
    out, lse = paged.attention(*m.on_gpu(), m.q.cuda(), return_lse=True)
    out, lse = out.cpu(), lse.cpu()
    want, want_lse, tol, tol_lse = m.wanted()
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    fine = torch.isfinite(want)
    assert fine.sum() > 0.5 * fine.numel() and ((out.double() - want).abs() <= tol)[fine].all()
    seen = torch.isnan(want_lse)   # (a NaN among the values leaves the sum of the exponentials to the kernel: it may be NaN too)
    assert torch.isnan(lse)[seen].all() and not torch.isnan(lse)[~torch.isnan(want).any(-1)].any()


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_scores_far_apart_and_scales_far_apart(paged, dtype):
    for big in (200.0, 1.0 / 4000):
        m = Made(paged, 8, dtype, INT8, [70, 90, 1], [1, 40, 1], 16, 8, 2, 2, 64, 50)
        m.q = (m.q.float() * big).to(dtype)
        m.check(*paged.attention(*m.on_gpu(), m.q.cuda(), return_lse=True))
    # values of heads and blocks that differ by many powers of ten, a block of zeros with a scale of 0 among them
    m = Made(paged, 9, dtype, E4M3, [70, 90, 3], [1, 40, 1], 16, 8, 2, 2, 64, 50)
    m.vs *= 10.0 ** torch.randint(-4, 3, m.vs.shape, generator=gen(2))
    m.vs = m.vs.float().double()
    p = oracle.place(m.tables[1], len(m.k), 16, 8)
    m.vs[p[0], p[1] // 8], m.v[p[0], p[1]:p[1] + 8] = 0.0, 0.0
    m.check(*paged.attention(*m.on_gpu(), m.q.cuda(), return_lse=True))


# ---- together ------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("form", [INT8, E4M3], ids=str)
def test_steps_as_a_server_makes_them(paged, form):
    """a prompt, then single tokens, captured into a graph and replayed with other lengths; the same on two streams at once with pools of their own"""
    g = gen(11)
    kv, group, size, page, block, seqs = 2, 4, 128, 16, 8, 3
    heads, steps = kv * group, 20
    counts = [30, 17, 1]
    rope = paged.RopeAxes.sections(size, 10000.0)
    wk, wq = torch.rand(size, generator=g).add(0.5).cuda(), torch.rand(size, generator=g).add(0.5).cuda()
    tables = torch.arange(seqs * 4, dtype=torch.int32).view(seqs, 4).cuda()

    def tokens(n):
        return [torch.randn(n, h, size, generator=g).to(BF16).cuda() for h in (heads, kv, kv)]

    prompt, singles = tokens(sum(counts)), [tokens(seqs) for _ in range(steps)]

    def pool():
        c = torch.zeros(seqs * 4, page, kv, size).to(form).cuda()
        s = torch.ones(seqs * 4, page // block, kv, device="cuda")
        return paged.QuantPages(c, c.clone(), s, s.clone())

    def step(pages, batch, q, k, v):
        q = paged.append(pages, batch, k, v, rope=rope, q=q, k_norm=wk, q_norm=wq)
        return paged.attention(pages, batch, q)

    def begin(pages, lens):
        starts = torch.tensor([0, 30, 47, 48], dtype=torch.int32).cuda()
        return step(pages, paged.Batch(lens, tables, rows=starts, max_rows=30), *prompt)

    lens = torch.tensor(counts, dtype=torch.int32).cuda()
    plain = pool()
    results = [begin(plain, lens)]
    for t in singles:
        lens += 1
        results.append(step(plain, paged.Batch(lens, tables), *t))
    # the formula on what the pool holds, in 64 bits, for the last step
    every = paged.Batch(lens, tables, rows=torch.tensor([0, 50, 87, 108], dtype=torch.int32).cuda(), max_rows=50)
    k, v = (t.cpu().double() for t in paged.read(plain, every, rows=108, dtype=F32))
    q = oracle.turn(oracle.norm(singles[-1][0].cpu(), wq.cpu(), 1e-6), (lens.cpu() - 1)[None], [10000.0 ** (-2.0 * j / size) for j in range(size // 2)], [0] * (size // 2), "halves").to(BF16).double()
    for b, (a, e) in enumerate(((0, 50), (50, 87), (87, 108))):
        for h in range(heads):
            want = torch.softmax(k[a:e, h // group] @ q[b, h] * size ** -0.5, 0) @ v[a:e, h // group]
            # queries here may be rounded to the neighbour (2^-8 of a score's terms), weights by 2^-11, the result by 2^-9
            off = 2.0 ** -8 * float((k[a:e, h // group].abs() @ q[b, h].abs()).max()) * size ** -0.5
            assert ((results[-1][b, h].cpu().double() - want).abs() <= (2 * off + 2.0 ** -8) * v[a:e, h // group].abs().max()).all()
    # captured
    lens.copy_(torch.tensor(counts, dtype=torch.int32))
    pages = pool()
    assert torch.equal(begin(pages, lens), results[0])
    batch, static = paged.Batch(lens, tables), [t.clone() for t in singles[0]]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):   # (a warm-up writes what the first replay writes again)
        lens += 1
        step(pages, batch, *static)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(pages, batch, *static)
    for i, t in enumerate(singles):
        if i:
            lens += 1
        for a, b in zip(static, t):
            a.copy_(b)
        graph.replay()
        assert torch.equal(out, results[i + 1]), i
    # two streams
    streams, pools, outs = [torch.cuda.Stream() for _ in range(2)], [pool() for _ in range(2)], [[], []]
    own = [torch.tensor(counts, dtype=torch.int32).cuda() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(-1, steps):
        for s, pages, n, o in zip(streams, pools, own, outs):
            with torch.cuda.stream(s):
                if i < 0:
                    o.append(begin(pages, n))
                else:
                    n += 1
                    o.append(step(pages, paged.Batch(n, tables), *singles[i]))
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, results))
