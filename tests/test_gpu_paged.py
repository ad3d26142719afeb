"""Many sequences at once on the GPU (lmrs_b200.paged) against 64-bit restatements (tests/paged_oracle.py).  Whatever a call must not read holds NaN, and whatever
it must not write is looked at afterwards."""
import math
import random

import pytest

torch = pytest.importorskip("torch")
import paged_oracle as oracle  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
P_EPS = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 0.0}   # what rounding a weight to the type costs at most


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


# ---- rotary positions ------------------------------------------------------------------------------------------------------------------------
ROPE = [  # rows, heads, size, rot, sections, order, layout, far
    (1, 1, 2, 2, [1], "blocks", "halves", 10), (1, 40, 64, 64, [32], "blocks", "halves", 8192), (5, 3, 128, 128, [16, 24, 24], "blocks", "halves", 2 ** 31 - 300),
    (7, 2, 96, 48, [8, 16], "cycle", "pairs", 100000), (3, 5, 80, 20, [1, 2, 3, 4], "cycle", "halves", 1000), (300, 9, 64, 64, [16, 16], "cycle", "pairs", 64),
    (2, 4, 256, 256, [128], "blocks", "pairs", 1000000), (17, 1, 33, 10, [5], "blocks", "pairs", 77), (6, 3, 40, 8, [1, 3], "blocks", "halves", 5), (1000, 32, 128, 128, [22, 21, 21], "cycle", "halves", 130000),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("how", ["packed", "gaps", "odd"])
@pytest.mark.parametrize("case", ROPE, ids=str)
def test_rope_axes(paged, case, how, dtype):
    n, heads, size, rot, sections, order, layout, far = case
    g = gen(n + heads)
    x = torch.randn(n, heads, size, generator=g).to(dtype)
    pos = (far + torch.randint(0, 200, (len(sections), n), generator=g)).to(torch.int32)
    pos[:, 0] = torch.tensor([0, -3, 7, -far])[:len(sections)]
    rope = paged.RopeAxes.sections(rot, 10000.0, sections, order, layout)
    freq, axis = [10000.0 ** (-2.0 * j / rot) for j in range(rot // 2)], list(rope._c.axis[:rot // 2])
    want = oracle.turn(x, pos, freq, axis, layout)
    tol = oracle.turn_tolerance(x, want, freq, layout)
    tol += x.double().abs().amax(-1, keepdim=True) * float(pos.double().abs().max()) * 2.0 ** -51   # the 64-bit angles themselves
    xg, pg = laid_out(x, how), pos.cuda() if how == "packed" else pos.T.contiguous().cuda().T
    got = paged.rope_axes(xg, pg, rope)
    assert ((got.cpu().double() - want).abs() <= tol).all()
    assert torch.equal(xg.cpu(), x)
    assert torch.equal(got.cpu()[..., rot:], x[..., rot:])
    out = laid_out(torch.zeros_like(x), how)
    assert paged.rope_axes(xg, pg, rope, out=out) is out and torch.equal(out.contiguous(), got)
    paged.rope_axes(xg, pg, rope, out=xg)   # in place
    assert torch.equal(xg.contiguous(), got)
    if len(sections) == 1:
        assert torch.equal(paged.rope_axes(x.cuda(), pos[0].cuda(), rope), got)


def test_rope_axes_of_nothing(paged):
    rope = paged.RopeAxes([1.0])
    assert paged.rope_axes(torch.zeros(0, 3, 8, device="cuda"), torch.zeros(1, 0, dtype=torch.int32, device="cuda"), rope).shape == (0, 3, 8)
    assert paged.rope_axes(torch.zeros(2, 0, 8, device="cuda"), torch.zeros(1, 2, dtype=torch.int32, device="cuda"), rope).shape == (2, 0, 8)


def test_rope_axes_takes_non_finite_rows(paged):
    """a NaN or an infinity spoils its own pair only"""
    x = torch.randn(4, 2, 64, generator=gen(1))
    x[1, 0, 3], x[2, 1, 40] = math.nan, math.inf
    rope = paged.RopeAxes.sections(64, 1e4)
    got = paged.rope_axes(x.cuda(), torch.arange(4, dtype=torch.int32, device="cuda"), rope).cpu()
    bad = torch.zeros_like(x, dtype=torch.bool)
    bad[1, 0, [3, 35]] = bad[2, 1, [8, 40]] = True
    assert torch.isfinite(got[~bad]).all() and not torch.isfinite(got[bad]).any()


# ---- a batch: sequences of given lengths in a pool whose unused places hold NaN ------------------------------------------------------------------
class Made:
    def __init__(self, paged, seed, dtype, lens, counts, page, kv_heads, group, size, prefix=0, one_each=False, order="pshd", tail=0, bad=()):
        r = random.Random(seed)
        g = gen(seed)
        self.lens, self.dtype, self.prefix_len, self.one_each = lens, dtype, prefix, one_each
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
        self.k = torch.full((pages, page, kv_heads, size), math.nan, dtype=dtype)
        self.v = self.k.clone()
        self.page, self.heads, self.kv_heads, self.size, self.counts = page, kv_heads * group, kv_heads, size, counts
        for table, n in [(self.tables[b], n) for b, n in enumerate(lens)] + [(self.prefix, prefix)]:
            for x in range(max(0, n)):
                p = oracle.place(table, pages, page, x)
                if p:
                    self.k[p], self.v[p] = torch.randn(kv_heads, size, generator=g).to(dtype), torch.randn(kv_heads, size, generator=g).to(dtype)
        self.q = (1.5 * torch.randn(self.n, self.heads, size, generator=g)).to(dtype)
        self.order = order
        self.paged = paged

    def on_gpu(self):
        perm = ["pshd".index(c) for c in self.order]
        back = [self.order.index(c) for c in "pshd"]
        k, v = (t.permute(perm).contiguous().cuda().permute(back) for t in (self.k, self.v))
        pages = self.paged.KVPages(k, v)
        batch = self.paged.Batch(torch.tensor(self.lens, dtype=torch.int32).cuda(), self.tables.cuda(), rows=None if self.rows is None else self.rows.cuda(),
                                 max_rows=max([1] + self.counts) if self.rows is not None else 1, prefix=self.prefix.cuda() if self.prefix_len else None, prefix_len=self.prefix_len)
        return pages, batch

    def check(self, out, lse, scale=None, cap=0.0, q=None):
        scale = self.size ** -0.5 if scale is None else scale
        want, want_lse, tol, tol_lse = oracle.attention(self.k, self.v, self.lens, self.tables, self.rows, self.prefix, self.prefix_len, self.q if q is None else q, scale, cap, P_EPS[self.dtype])
        seen = ~torch.isnan(want_lse)   # rows of some sequence
        got, got_lse = out.cpu().double(), lse.cpu().double()
        assert torch.equal(torch.isinf(got_lse)[seen], torch.isinf(want_lse)[seen])
        assert ((got - want).abs() <= tol)[seen].all(), float(((got - want).abs() - tol)[seen].max())
        finite = seen & torch.isfinite(want_lse)
        assert ((got_lse - want_lse).abs() <= tol_lse)[finite].all(), float(((got_lse - want_lse).abs() - tol_lse)[finite].max())


SINGLE = [  # tokens held, page, kv heads, group, size, prefix, order of the pool
    ([1], 16, 1, 1, 64, 0, "pshd"), ([1], 1, 2, 4, 64, 1, "pshd"), ([63, 64, 65], 16, 2, 4, 64, 0, "pshd"), ([130, 1, 17, 0, 255], 7, 3, 2, 128, 33, "pshd"), ([700], 64, 8, 4, 64, 0, "phsd"),
    ([5, 0, 0, 9], 5, 2, 5, 96, 129, "pshd"), ([200, 300], 128, 1, 16, 256, 64, "phsd"), ([33, 40], 3, 4, 1, 8, 70, "pshd"), ([90] * 20, 32, 2, 8, 128, 200, "spdh"[:2] + "hd"), ([257, 3], 48, 1, 20, 64, 100, "hpsd"),
    ([40, 41, 42], 16, 5, 3, 40, 513, "pshd"), ([64] * 3, 64, 2, 12, 200, 64, "pshd"), ([2000, 1], 16, 1, 6, 128, 0, "pshd"), ([10] * 70, 16, 1, 4, 64, 400, "pshd"), ([0, 0], 16, 1, 2, 64, 50, "pshd"),
    ([12] * 40, 8, 2, 8, 128, 1100, "phsd"), ([100] * 3, 16, 1, 64, 64, 300, "pshd"), ([150] * 9, 16, 2, 16, 256, 260, "pshd"),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("case", SINGLE, ids=lambda c: f"{len(c[0])}x{max(c[0])}-page{c[1]}-{c[2]}x{c[3]}x{c[4]}-prefix{c[5]}-{c[6]}")
def test_attention_of_single_tokens(paged, case, dtype):
    lens, page, kv, group, size, prefix, order = case
    m = Made(paged, len(lens) + size, dtype, lens, [1] * len(lens), page, kv, group, size, prefix, one_each=True, order=order)
    pages, batch = m.on_gpu()
    out, lse = paged.attention(pages, batch, m.q.cuda(), return_lse=True)
    m.check(out, lse)
    assert torch.equal(paged.attention(pages, batch, laid_out(m.q, "odd"), out=laid_out(m.q, "odd")).contiguous(), out)   # the same bits, wherever the rows lie
    assert torch.equal(paged.attention(pages, batch, laid_out(m.q, "gaps")), out)


MANY = [  # tokens held, rows of the call, page, kv heads, group, size, prefix
    ([3], [3], 16, 1, 1, 64, 0), ([100, 40, 9], [100, 3, 9], 16, 2, 4, 64, 0), ([70, 300, 65], [1, 130, 65], 7, 2, 3, 128, 35), ([20, 0, 90], [20, 1, 33], 32, 1, 8, 96, 200), ([150, 150], [64, 65], 64, 3, 2, 256, 64),
    ([5, 2, 40], [7, 0, 40], 4, 2, 2, 64, 65), ([260], [257], 48, 1, 2, 128, 0), ([9] * 30, [3] * 30, 16, 2, 2, 64, 130), ([33], [33], 1, 1, 5, 24, 10), ([130, 200], [128, 129], 16, 1, 4, 128, 700),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("case", MANY, ids=lambda c: f"{len(c[0])}x{max(c[0])}-rows{max(c[1])}-page{c[2]}-{c[3]}x{c[4]}x{c[5]}-prefix{c[6]}")
def test_attention_of_several_rows(paged, case, dtype):
    """(a sequence with more rows than tokens: the first ones are padding; rows behind the last sequence stay as they are)"""
    lens, counts, page, kv, group, size, prefix = case
    m = Made(paged, len(lens) + size, dtype, lens, counts, page, kv, group, size, prefix, tail=2)
    pages, batch = m.on_gpu()
    out = torch.full((m.n, m.heads, size), 7.0, dtype=dtype, device="cuda")
    got, lse = paged.attention(pages, batch, m.q.cuda(), out=out, return_lse=True)
    assert got is out
    m.check(out, lse)
    assert (out[-2:] == 7.0).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_attention_scale_and_cap(paged, dtype):
    m = Made(paged, 5, dtype, [100, 37, 200], [1, 37, 70], 16, 2, 4, 64, 90)
    pages, batch = m.on_gpu()
    for scale, cap in ((1.0, 0.0), (0.125, 20.0), (0.5, 1.5), (0.0, 0.0), (-0.125, 0.0), (4.0, 50.0)):
        out, lse = paged.attention(pages, batch, m.q.cuda(), scale=scale, softcap=cap, return_lse=True)
        m.check(out, lse, scale, cap)


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_entries_that_are_no_pages(paged, dtype):
    """what lies there is not seen, wherever the entry is; a row all of whose pages are missing sees nothing"""
    lens = [100, 64, 16, 40]
    bad = [(0, 2, -1), (0, 4, 2 ** 31 - 1), (1, 0, -2 ** 31), (1, 3, 1000), (2, 0, -5), (-1, 1, 99999), (-1, 3, -1)]
    for one, prefix in ((True, 80), (False, 80), (True, 0), (False, 0)):
        m = Made(paged, 3, dtype, lens, [1] * 4 if one else [1, 30, 16, 40], 16, 2, 4, 64, prefix, one_each=one, bad=[x for x in bad if prefix or x[0] >= 0])
        out, lse = paged.attention(*m.on_gpu(), m.q.cuda(), return_lse=True)
        m.check(out, lse)
        if not prefix:
            row = 2 if one else 31
            assert (out[row] == 0).all() and (lse[row] == -math.inf).all()


def test_tokens_beyond_the_table(paged):
    """a length that the table does not reach: what it does reach counts"""
    m = Made(paged, 4, BF16, [40, 70], [1, 1], 16, 1, 2, 64, 20, one_each=True)
    pages, batch = m.on_gpu()
    m.tables = m.tables[:, :3]
    batch = paged.Batch(batch.lens, m.tables.cuda(), prefix=batch.prefix, prefix_len=20)   # 48 tokens at most
    out, lse = paged.attention(pages, batch, m.q.cuda(), return_lse=True)
    m.check(out, lse)
    batch.lens.copy_(torch.tensor([2 ** 31 - 1, -2 ** 31], dtype=torch.int32))
    out, lse = paged.attention(pages, batch, m.q.cuda(), return_lse=True)
    assert (out[1] == 0).all() and (lse[1] == -math.inf).all()
    assert paged.append(pages, batch, *(torch.ones(2, 1, 64, dtype=BF16, device="cuda"),) * 2) is None   # nowhere to write to
    empty = paged.Batch(batch.lens, m.tables[:, :0].cuda(), prefix=batch.prefix, prefix_len=20)
    batch.lens.fill_(5)
    m.lens, m.tables = [5, 5], m.tables[:, :0]
    m.check(*paged.attention(pages, empty, m.q.cuda(), return_lse=True))


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_values_that_are_not_finite(paged, dtype):
    """a NaN or an infinity reaches the rows that see it, and no other: not those of other sequences, nor those before it in its own"""
    m = Made(paged, 6, dtype, [130, 80, 50], [100, 80, 1], 16, 2, 2, 64, 70)
    at = [oracle.place(m.tables[0], len(m.k), 16, x) for x in (60, 99)]
    m.v[at[0]][1, 3], m.k[at[1]][0, 5], m.v[oracle.place(m.tables[1], len(m.k), 16, 77)][0, 63] = math.inf, math.nan, math.nan
    out, lse = paged.attention(*m.on_gpu(), m.q.cuda(), return_lse=True)
    out, lse = out.cpu(), lse.cpu()
    want, want_lse, tol, tol_lse = oracle.attention(m.k, m.v, m.lens, m.tables, m.rows, m.prefix, 70, m.q, 0.125, 0.0, P_EPS[dtype])
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(torch.isinf(out), torch.isinf(want))
    fine = torch.isfinite(want)
    assert fine.sum() > 0.8 * fine.numel() and ((out.double() - want).abs() <= tol)[fine].all()
    assert torch.equal(torch.isnan(lse), torch.isnan(want_lse))


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_scores_of_minus_infinity(paged, dtype):
    """keys at -infinity along a query weigh nothing; a row with no other keys is 0 / 0, as the formula has it"""
    m = Made(paged, 7, dtype, [40, 20], [1, 1], 16, 1, 2, 64, 0, one_each=True)
    m.q[:, :, 0] = 1.0
    for x in range(20):
        m.k[oracle.place(m.tables[1], len(m.k), 16, x)][0, 0] = -math.inf
        m.k[oracle.place(m.tables[0], len(m.k), 16, 2 * x)][0, 0] = -math.inf
    out, lse = paged.attention(*m.on_gpu(), m.q.cuda(), return_lse=True)
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1]).all() and (lse[1] == -math.inf).all()
    want, want_lse, tol, _ = oracle.attention(m.k, m.v, m.lens, m.tables, None, m.prefix, 0, m.q, 0.125, 0.0, P_EPS[dtype])
    # (scores of -infinity have no size: the bound of a dot product comes from the finite keys)
    k = m.k.clone()
    k[k == -math.inf] = 0.0
    tol = oracle.attention(k, m.v, m.lens, m.tables, None, m.prefix, 0, m.q, 0.125, 0.0, P_EPS[dtype])[2] * 2
    assert ((out[0].cpu().double() - want[0]).abs() <= tol[0]).all()


def test_large_and_small_scores(paged):
    """scores far apart, far from zero, and at the end of the type"""
    for dtype, big in ((BF16, 1e4), (F16, 200.0), (F32, 1e4)):
        m = Made(paged, 8, dtype, [70, 90, 1], [1, 40, 1], 16, 2, 2, 64, 50)
        m.q = (m.q.float() * big).to(dtype)
        m.check(*paged.attention(*m.on_gpu(), m.q.cuda(), return_lse=True))
        m.q = (m.q.float() / big ** 2).to(dtype)
        m.check(*paged.attention(*m.on_gpu(), m.q.cuda(), return_lse=True))


# ---- appending -----------------------------------------------------------------------------------------------------------------------------------
APPEND = [  # tokens held, rows, page, kv heads, group, size, rot, sections, layout, prefix, positions given
    ([1], None, 16, 1, 1, 64, 64, [32], "halves", 0, False), ([9, 0, 33, 16], None, 16, 2, 4, 64, 32, [8, 8], "pairs", 20, False), ([700], None, 64, 8, 4, 128, 128, [16, 24, 24], "halves", 0, True),
    ([20, 5, 0, 60], [20, 2, 1, 33], 7, 2, 3, 96, 96, [20, 28], "halves", 33, True), ([300, 300], [257, 300], 16, 1, 2, 40, 20, [10], "pairs", 0, False), ([4, 9], [6, 9], 1, 3, 1, 256, 256, [128], "halves", 5, False),
    ([50] * 70, None, 48, 2, 2, 64, 64, [10, 11, 11], "pairs", 100, True), ([12, 30], [5, 5], 4, 1, 1, 33, 10, [5], "halves", 0, False), ([8] * 9, [3] * 9, 8, 5, 1, 8, 2, [1], "pairs", 0, True),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("how", ["packed", "gaps", "odd"])
@pytest.mark.parametrize("case", APPEND, ids=lambda c: f"{len(c[0])}x{max(c[0])}-page{c[2]}-{c[3]}x{c[5]}-rot{c[6]}{c[8]}")
def test_append(paged, case, how, dtype):
    lens, counts, page, kv, group, size, rot, sections, layout, prefix, given = case
    m = Made(paged, len(lens) + size, dtype, lens, counts or [1] * len(lens), page, kv, group, size, prefix, one_each=counts is None, order="phsd" if how == "gaps" else "pshd", tail=0 if counts is None else 3)
    g = gen(3)
    k, v = (torch.randn(m.n, kv, size, generator=g).to(dtype) for _ in range(2))
    pos = torch.randint(0, 100000, (len(sections), m.n), generator=g).to(torch.int32)
    rope = paged.RopeAxes.sections(rot, 10000.0, sections, "cycle", layout)
    freq, axis = [10000.0 ** (-2.0 * j / rot) for j in range(rot // 2)], list(rope._c.axis[:rot // 2])
    pages, batch = m.on_gpu()
    places, index = {}, torch.zeros(m.n, dtype=torch.int64)
    for b, (first, c, have) in enumerate(oracle.spans(lens, m.rows, m.n)):
        for i in range(c):
            index[first + i] = have - c + i
            places[first + i] = oracle.place(m.tables[b], len(m.k), page, have - c + i)
    use = pos if given else (prefix + index).to(torch.int32).expand(len(sections), -1)
    turned = oracle.turn(k, use, freq, axis, layout), oracle.turn(m.q, use, freq, axis, layout)
    args = [laid_out(t, how) for t in (k, v, m.q)]
    q_out = torch.full(m.q.shape, 7.0, dtype=dtype, device="cuda") if how == "packed" else laid_out(torch.full_like(m.q, 7.0), how)
    assert paged.append(pages, batch, args[0], args[1], rope=rope, pos=pos.cuda() if given else None, q=args[2], q_out=q_out) is q_out
    kp, vp = pages.k.cpu(), pages.v.cpu()
    slack = 100200 * 2.0 ** -51
    want_k, want_v, tol = m.k.double(), m.v.clone(), torch.zeros_like(m.k, dtype=torch.float64)
    k_tol = oracle.turn_tolerance(k, turned[0], freq, layout) + k.double().abs().amax(-1, keepdim=True) * slack
    for r, p in places.items():
        if p:
            want_k[p], want_v[p], tol[p] = turned[0][r], v[r], k_tol[r]
    same = torch.isnan(want_k)
    assert torch.equal(torch.isnan(kp), same) and ((kp.double() - want_k).abs() <= tol)[~same].all()
    assert torch.equal(vp.nan_to_num(9.0), want_v.nan_to_num(9.0))
    rows = sorted(places)
    q_tol = oracle.turn_tolerance(m.q, turned[1], freq, layout) + m.q.double().abs().amax(-1, keepdim=True) * slack
    assert ((q_out.cpu().double() - turned[1]).abs() <= q_tol)[rows].all()
    assert (q_out[len(rows):] == 7.0).all()
    # the same again, queries in place; and as it is, without rotation
    paged.append(pages, batch, args[0], args[1], rope=rope, pos=pos.cuda() if given else None, q=args[2], q_out=args[2])
    assert torch.equal(pages.k.cpu().nan_to_num(9.0), kp.nan_to_num(9.0)) and torch.equal(args[2][:len(rows)], q_out[:len(rows)])
    assert paged.append(pages, batch, args[0], args[1]) is None
    for r, p in places.items():
        if p:
            assert torch.equal(pages.k[p].cpu(), k[r]) and torch.equal(pages.v[p].cpu(), v[r])
    kp2 = pages.k.cpu()
    for p in places.values():
        if p:
            kp2[p] = math.nan
            kp[p] = math.nan
    assert torch.equal(kp2.nan_to_num(9.0), kp.nan_to_num(9.0))


def test_append_drops_rows_without_a_page(paged):
    m = Made(paged, 3, F32, [20, 40, 33], [20, 10, 1], 16, 1, 1, 8, bad=[(0, 0, -1), (1, 2, 77), (2, 1, 2 ** 31 - 1)])
    pages, batch = m.on_gpu()
    before = m.k.clone()
    k = torch.ones(m.n, 1, 8)
    paged.append(pages, batch, k.cuda(), k.cuda())
    for b, (first, c, have) in enumerate(oracle.spans(m.lens, m.rows, m.n)):
        for i in range(c):
            p = oracle.place(m.tables[b], len(m.k), 16, have - c + i)
            if p:
                before[p] = 1.0
    assert torch.equal(pages.k.cpu().nan_to_num(9.0), before.nan_to_num(9.0))


def test_places_beyond_2_to_the_31(paged):
    """a pool of more than 2^31 elements, its last pages in use"""
    pages_n, page, size = 4200, 4096, 128   # 2.2e9 elements a side
    k = torch.empty(pages_n, page, 1, size, dtype=BF16, device="cuda")
    v = torch.empty_like(k)
    pages = paged.KVPages(k, v)
    table = torch.tensor([[pages_n - 1, 5, pages_n - 2]], dtype=torch.int32)
    n = 2 * page + 40
    g = gen(4)
    kn, vn = (torch.randn(n, 1, size, generator=g).to(BF16) for _ in range(2))
    lens = torch.tensor([n], dtype=torch.int32).cuda()
    paged.append(pages, paged.Batch(lens, table.cuda(), rows=torch.tensor([0, n], dtype=torch.int32).cuda(), max_rows=n), kn.cuda(), vn.cuda())
    assert torch.equal(k[pages_n - 1, :, 0].cpu(), kn[:page, 0]) and torch.equal(v[pages_n - 2, :40, 0].cpu(), vn[2 * page:, 0])
    q = torch.randn(1, 4, size, generator=g).to(BF16)
    out = paged.attention(pages, paged.Batch(lens, table.cuda()), q.cuda()).cpu().double()
    s = torch.einsum("hd,kd->hk", q[0].double(), kn[:, 0].double()) * size ** -0.5
    want, A = torch.softmax(s, -1) @ vn[:, 0].double(), torch.softmax(s, -1) @ vn[:, 0].double().abs()
    assert ((out[0] - want).abs() <= A * (2.0 ** -8 + 2 * n * 2.0 ** -24 + 2.0 ** -14) + want.abs() * 2.0 ** -8).all()


def exact_on_gpu(k, v, lens, tables, counts, prefix, prefix_len, q, scale, cap):
    """the formula in 64 bits, a sequence and a KV head at a time on the GPU; out, lse and the sums of weighted sizes that bound what rounding does"""
    G, D = k.shape[2:]
    H, ps = q.shape[1], k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse, size = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda"), torch.zeros_like(out)
    first = 0
    for b, (have, c) in enumerate(zip(lens, counts)):
        x = torch.arange(have, device="cuda")
        pages = [prefix.long()[torch.arange(prefix_len, device="cuda") // ps] * ps + torch.arange(prefix_len, device="cuda") % ps] if prefix_len else []
        at = torch.cat(pages + [tables[b].long()[x // ps] * ps + x % ps])
        keys, values = k.reshape(-1, G, D)[at].double(), v.reshape(-1, G, D)[at].double()
        last = prefix_len + have - c + torch.arange(c, device="cuda")
        for g in range(G):
            heads = slice(g * (H // G), (g + 1) * (H // G))
            s = torch.einsum("rhd,kd->rhk", q[first:first + c, heads].double(), keys[:, g]) * scale
            s = cap * torch.tanh(s / cap) if cap else s
            s = s.masked_fill(torch.arange(at.numel(), device="cuda") > last[:, None, None], -math.inf)
            w = torch.softmax(s, -1)
            out[first:first + c, heads], size[first:first + c, heads] = w @ values[:, g], w @ values[:, g].abs()
            lse[first:first + c, heads] = torch.logsumexp(s, -1)
        first += c
    return out, lse, size


LONG = [  # sequences, rows of the longest, tokens before, prefix, page, kv heads, group, size, cap: CTAs that take many tiles, and parts of several units
    (16, 1, 40, 5120, 16, 8, 4, 128, 0.0), (64, 1, 40, 5120, 16, 8, 4, 128, 0.0), (64, 1, 300, 20000, 64, 8, 4, 64, 0.0), (70, 1, 100, 9001, 7, 4, 8, 128, 0.0), (32, 1, 77, 8200, 32, 8, 4, 256, 0.0),
    (100, 1, 500, 3001, 48, 4, 5, 96, 30.0), (12, 200, 900, 2050, 32, 8, 2, 128, 0.0), (12, 200, 900, 0, 32, 8, 2, 128, 50.0), (2, 1500, 4000, 0, 16, 4, 4, 64, 0.0), (5, 300, 700, 1000, 8, 2, 3, 256, 20.0), (3, 5, 30000, 0, 16, 2, 4, 128, 0.0),
    (40, 1, 3000, 0, 16, 8, 4, 128, 0.0), (2, 1, 50000, 0, 1, 2, 8, 64, 0.0),
    (9, 2, 50, 1111, 16, 8, 4, 256, 0.0), (17, 5, 900, 60, 16, 2, 4, 256, 0.0), (6, 17, 500, 130, 32, 2, 4, 64, 30.0), (33, 1, 20, 70000, 128, 1, 1, 80, 0.0),
    (8, 1, 3000, 200, 16, 1, 16, 256, 0.0), (5, 1, 700, 0, 16, 1, 64, 128, 0.0), (4, 3, 500, 300, 16, 1, 48, 64, 0.0), (3, 2, 400, 1500, 24, 1, 128, 128, 20.0),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("case", LONG, ids=lambda c: "x".join(map(str, c)))
def test_attention_of_many_tiles(paged, case, dtype):
    seqs, most, past, prefix, page, kv, group, size, cap = case
    r = random.Random(seqs + prefix)
    counts = [most] + [r.randint(max(1, most // 3), most) for _ in range(seqs - 1)]
    lens = [past + most] + [r.randint(past // 4, past) + c for c in counts[1:]]
    held, shared = [-(-n // page) for n in lens], -(-prefix // page)
    g = torch.Generator("cuda")
    g.manual_seed(seqs)
    pages = sum(held) + shared
    k, v = (torch.randn(pages, page, kv, size, generator=g, device="cuda").to(dtype) for _ in range(2))
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    tables = torch.full((seqs, max(held)), -1, dtype=torch.int32, device="cuda")
    at = shared
    for b, h in enumerate(held):
        tables[b, :h] = order[at:at + h]
        if lens[b] % page:   # what lies behind a sequence's last token is not read
            k[order[at + h - 1].item(), lens[b] % page:] = math.nan
            v[order[at + h - 1].item(), lens[b] % page:] = math.nan
        at += h
    if prefix % page:
        k[order[shared - 1].item(), prefix % page:] = math.nan
        v[order[shared - 1].item(), prefix % page:] = math.nan
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    q = (1.5 * torch.randn(starts[-1], kv * group, size, generator=g, device="cuda")).to(dtype)
    rows = torch.tensor(starts, dtype=torch.int32, device="cuda") if most > 1 else None
    batch = paged.Batch(torch.tensor(lens, dtype=torch.int32, device="cuda"), tables, rows=rows, max_rows=most, prefix=order[:shared].contiguous() if prefix else None, prefix_len=prefix)
    scale = size ** -0.5
    out, lse = paged.attention(paged.KVPages(k, v), batch, q, softcap=cap, return_lse=True)
    want, want_lse, sizes = exact_on_gpu(k, v, lens, tables, counts, order[:shared], prefix, q, scale, cap)
    # as in paged_oracle.attention: a dot product's error D u of the sum of sizes (at most |q| |k|: here 1.5 D E|x|^2 scale with room), the exponential, the weights' rounding, and
    # sums of n terms, which in 16-bit types run in accumulators that may truncate
    n, u = prefix + max(lens), 2.0 ** -24
    off = (size + 4) * u * 2.5 * size * scale + 8 * u * cap
    rel = 2 * (off + 4 * u * 64 + 2.0 ** -21) + (2 * n + 64) * u
    eps = torch.finfo(dtype).eps / 2
    assert ((out.double() - want).abs() <= sizes * (rel + P_EPS[dtype]) * (1 + eps) + want.abs() * eps + torch.finfo(dtype).tiny).all()
    assert ((lse.double() - want_lse).abs() <= rel + 4 * u * want_lse.abs()).all()


# ---- together, captured, on other streams -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_a_chat_of_many_steps(paged, dtype):
    """a prefix, prompts of different lengths in one call, then tokens one by one: every step rotates, appends and attends, and must see what the
    sequence's own history (kept here as it was handed in) gives in 64 bits.  The steps are one captured graph, replayed."""
    kv, group, size, page, prefix, B = 2, 4, 64, 16, 37, 3
    g = gen(11)
    rope = paged.RopeAxes.sections(64, 10000.0, [8, 12, 12])
    freq, axis = [10000.0 ** (-2.0 * j / 64) for j in range(32)], [0] * 8 + [1] * 12 + [2] * 12
    pool = [torch.full((40, page, kv, size), math.nan, dtype=dtype, device="cuda") for _ in range(2)]
    pages = paged.KVPages(*pool)
    ids = torch.randperm(40, generator=g).to(torch.int32)
    shared, tables = ids[:3].cuda(), ids[3:36].view(3, 11).cuda()

    def rows(n, heads):
        return torch.randn(n, heads, size, generator=g).to(dtype)

    pk, pv = rows(prefix, kv), rows(prefix, kv)
    one = paged.Batch(torch.tensor([prefix], dtype=torch.int32).cuda(), shared[None], rows=torch.tensor([0, prefix], dtype=torch.int32).cuda(), max_rows=prefix)
    paged.append(pages, one, pk.cuda(), pv.cuda(), rope=rope)
    history = [[(pk[i], pv[i], i) for i in range(prefix)] for _ in range(B)]

    def check(out, q, owner, upto):
        for r, (b, n) in enumerate(zip(owner, upto)):
            ks, vs = torch.stack([h[0] for h in history[b][:n]]), torch.stack([h[1] for h in history[b][:n]]).double()
            at = torch.tensor([h[2] for h in history[b][:n]]).expand(3, -1)
            ks = oracle.turn(ks, at, freq, axis, "halves")
            qq = oracle.turn(q[r:r + 1], torch.full((3, 1), n - 1), freq, axis, "halves")[0]
            s = torch.einsum("hd,khd->hk", qq, ks.repeat_interleave(group, 1)) * size ** -0.5
            w = torch.softmax(s, -1)
            want, A = torch.einsum("hk,khd->hd", w, vs.repeat_interleave(group, 1)), torch.einsum("hk,khd->hd", w, vs.repeat_interleave(group, 1).abs())
            # keys and queries were rounded to the type after turning: each moves a score by half a step of the sum of sizes
            moved = 2 * torch.einsum("hd,khd->hk", qq.abs(), ks.abs().repeat_interleave(group, 1)).amax(-1) * size ** -0.5 * (torch.finfo(dtype).eps / 2 + 2.0 ** -21)
            tol = A * (2 * moved[:, None] + P_EPS[dtype] + 2.0 ** -14 * (dtype != F32) + 2.0 ** -17) + want.abs() * torch.finfo(dtype).eps
            assert ((out[r].cpu().double() - want).abs() <= tol).all(), (r, float(((out[r].cpu().double() - want).abs() - tol).max()))

    counts = [5, 70, 1]
    k, v, q = rows(76, kv), rows(76, kv), rows(76, kv * group)
    lens = torch.tensor(counts, dtype=torch.int32).cuda()
    batch = paged.Batch(lens, tables, rows=torch.tensor([0, 5, 75, 76], dtype=torch.int32).cuda(), max_rows=70, prefix=shared, prefix_len=prefix)
    turned = paged.append(pages, batch, k.cuda(), v.cuda(), rope=rope, q=q.cuda())
    out = paged.attention(pages, batch, turned)
    owner, upto, r = [], [], 0
    for b, c in enumerate(counts):
        for i in range(c):
            history[b].append((k[r], v[r], prefix + i))
            owner.append(b)
            upto.append(prefix + i + 1)
            r += 1
    check(out, q, owner, upto)

    step = paged.Batch(lens, tables, prefix=shared, prefix_len=prefix)
    k, v, q = (torch.zeros(B, h, size, dtype=dtype, device="cuda") for h in (kv, kv, kv * group))

    def decode():
        lens.add_(1)
        return paged.attention(pages, step, paged.append(pages, step, k, v, rope=rope, q=q))

    held = lens.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode()
    torch.cuda.current_stream().wait_stream(side)
    lens.copy_(held)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = decode()
    for i in range(12):
        new = [rows(B, h) for h in (kv, kv, kv * group)]
        for t, x in zip((k, v, q), new):
            t.copy_(x)
        graph.replay()
        for b in range(B):
            history[b].append((new[0][b], new[1][b], prefix + counts[b] + i))
        check(out, new[2], range(B), [prefix + c + i + 1 for c in counts])
    assert lens.tolist() == [c + 12 for c in counts]


def test_calls_on_two_streams_and_two_graphs(paged):
    """two batches over one pool at the same time, eager and as captured graphs that are replayed together: each what it is alone"""
    made = [Made(paged, s, BF16, [400 + 50 * s] * 6, [1] * 6, 16, 2, 4, 128, 600 + 100 * s, one_each=True) for s in (1, 2)]
    calls = [(m.on_gpu(), m.q.cuda()) for m in made]
    alone = [paged.attention(p, b, q, return_lse=True) for (p, b), q in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in calls], [[], []]
    for _ in range(20):
        for i, ((p, b), q) in enumerate(calls):
            with torch.cuda.stream(streams[i]):
                got[i].append(paged.attention(p, b, q, return_lse=True))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i][0]) and torch.equal(l, alone[i][1]) for o, l in got[i])
    graphs, outs = [], []
    for i, ((p, b), q) in enumerate(calls):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged.attention(p, b, q, return_lse=True))
        graphs.append(graph)
    for _ in range(20):
        for o, l in outs:
            o.fill_(9.0)
            l.fill_(9.0)
        torch.cuda.synchronize()
        for i, graph in enumerate(graphs):
            with torch.cuda.stream(streams[i]):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(outs[i][j], alone[i][j]) for i in range(2) for j in range(2))


def test_refusals_of_tensors(paged):
    m = Made(paged, 1, BF16, [40, 50], [1, 1], 16, 2, 2, 64, 20, one_each=True)
    pages, batch = m.on_gpu()
    q = m.q.cuda()
    k = torch.zeros(2, 2, 64, dtype=BF16, device="cuda")
    rope = paged.RopeAxes.sections(64, 1e4)
    i32 = dict(dtype=torch.int32, device="cuda")
    long = torch.zeros(2, dtype=torch.int64, device="cuda")
    for call in (lambda: paged.attention(pages, batch, q.float()), lambda: paged.attention(pages, batch, q[:1]), lambda: paged.attention(pages, batch, q[:, :3]), lambda: paged.attention(pages, batch, q[..., :56]),
                 lambda: paged.attention(pages, batch, q.cpu()), lambda: paged.attention(pages, batch, q, out=q[:, :, :1].expand_as(q)), lambda: paged.attention(pages, batch, q, out=q[:1].expand_as(q)),
                 lambda: paged.attention(pages, batch, q, scale=math.nan), lambda: paged.attention(pages, batch, q, softcap=-1.0), lambda: paged.attention(pages, None, q), lambda: paged.attention(None, batch, q),
                 lambda: paged.attention(pages, batch, q[:, :0]), lambda: paged.append(pages, batch, k[:1], k), lambda: paged.append(pages, batch, k, k[:, :1]), lambda: paged.append(pages, batch, k, k, q=q),
                 lambda: paged.append(pages, batch, k, k, pos=torch.zeros(1, 2, **i32)), lambda: paged.append(pages, batch, k, k, rope=rope, pos=long), lambda: paged.append(pages, batch, k, k, rope=rope, q_out=q),
                 lambda: paged.append(pages, batch, k, k, rope=rope, pos=torch.zeros(1, 3, **i32)), lambda: paged.append(pages, batch, k, k, rope=paged.RopeAxes.sections(66, 1e4)),
                 lambda: paged.rope_axes(q, long, rope), lambda: paged.rope_axes(q, torch.zeros(3, **i32), rope), lambda: paged.rope_axes(q.to(torch.float64), torch.zeros(2, **i32), rope),
                 lambda: paged.rope_axes(q, torch.zeros(1, 2, **i32), paged.RopeAxes.sections(64, 1e4, [16, 16])), lambda: paged.rope_axes(q.transpose(1, 2), torch.zeros(2, **i32), rope),
                 lambda: paged.Batch(long, m.tables.cuda()), lambda: paged.Batch(batch.lens, m.tables), lambda: paged.Batch(batch.lens, m.tables[:1].cuda()), lambda: paged.Batch(batch.lens, m.tables.cuda(), max_rows=2),
                 lambda: paged.Batch(batch.lens, m.tables.cuda(), prefix_len=3), lambda: paged.Batch(batch.lens, m.tables.cuda(), rows=torch.zeros(2, **i32)), lambda: paged.KVPages(pages.k, pages.v[1:]),
                 lambda: paged.KVPages(pages.k, pages.v.float()), lambda: paged.KVPages(pages.k[:1].expand_as(pages.k), pages.v), lambda: paged.KVPages(pages.k.transpose(2, 3), pages.v.transpose(2, 3)),
                 lambda: paged.attention(pages, paged.Batch(batch.lens, m.tables.cuda(), prefix=batch.prefix[:1], prefix_len=20), q)):
        with pytest.raises(paged.LmrsError):
            call()
    odd = torch.zeros(pages.k.numel() + 8, dtype=BF16, device="cuda")[1:-7].view(pages.k.shape)   # pages off their 16-byte boundaries: appended to, not attended
    off = paged.KVPages(odd, odd.clone())
    paged.append(off, batch, k, k)
    with pytest.raises(paged.LmrsError, match="16-byte"):
        paged.attention(off, batch, q)
    m.check(*paged.attention(pages, batch, q, return_lse=True))   # and the next call is fine


def test_calls_of_no_rows(paged):
    m = Made(paged, 1, BF16, [40], [1], 16, 2, 2, 64, 20, one_each=True)
    pages, _ = m.on_gpu()
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    batch = paged.Batch(none, none.view(0, 3))
    q, k = torch.zeros(0, 4, 64, dtype=BF16, device="cuda"), torch.zeros(0, 2, 64, dtype=BF16, device="cuda")
    assert paged.attention(pages, batch, q).shape == (0, 4, 64) and paged.append(pages, batch, k, k) is None
    idle = paged.Batch(torch.tensor([5, 0], dtype=torch.int32).cuda(), torch.zeros(2, 3, dtype=torch.int32).cuda(), rows=torch.zeros(3, dtype=torch.int32).cuda())
    q = torch.ones(2, 4, 64, dtype=BF16, device="cuda")
    out = torch.full_like(q, 7.0)
    paged.attention(pages, idle, q, out=out)   # sequences without rows, rows without a sequence
    assert (out == 7.0).all()


def test_attention_into_its_queries_is_refused(paged):
    m = Made(paged, 1, BF16, [40, 50], [1, 1], 16, 2, 2, 64, 20, one_each=True)
    pages, batch = m.on_gpu()
    q = m.q.cuda()
    with pytest.raises(paged.LmrsError, match="lies where q does"):
        paged.attention(pages, batch, q, out=q)
    m.check(*paged.attention(pages, batch, q, return_lse=True))


# ---- batches made on the GPU ------------------------------------------------------------------------------------------------------------------------
class MadeThere:
    """sequences of given lengths and rows over pages in random order, values made on the GPU; what lies behind a list's last token holds NaN"""

    def __init__(self, paged, seed, dtype, lens, counts, page, kv, group, size, prefix=0):
        self.paged, self.dtype, self.lens, self.counts, self.prefix_len, self.size = paged, dtype, list(lens), list(counts), prefix, size
        g = torch.Generator("cuda")
        g.manual_seed(seed)
        held, shared = [-(-n // page) for n in lens], -(-prefix // page)
        pages = sum(held) + shared
        self.k, self.v = (torch.randn(pages, page, kv, size, generator=g, device="cuda").to(dtype) for _ in range(2))
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        self.tables = torch.full((len(lens), max(held)), -1, dtype=torch.int32, device="cuda")
        self.prefix = order[:shared].contiguous()
        at, ends = shared, [(self.prefix, prefix)]
        for b, h in enumerate(held):
            self.tables[b, :h] = order[at:at + h]
            at += h
            ends.append((self.tables[b, :h], lens[b]))
        for table, n in ends:
            if n % page:
                self.k[table[-1].item(), n % page:] = math.nan
                self.v[table[-1].item(), n % page:] = math.nan
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        self.q = (1.5 * torch.randn(starts[-1], kv * group, size, generator=g, device="cuda")).to(dtype)
        one = max(counts) == min(counts) == 1
        self.rows = None if one else torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.pages = paged.KVPages(self.k, self.v)
        self.batch = self.batch_of()

    def batch_of(self, max_rows=None):
        return self.paged.Batch(torch.tensor(self.lens, dtype=torch.int32, device="cuda"), self.tables, rows=self.rows, max_rows=max_rows or max(self.counts),
                                prefix=self.prefix if self.prefix_len else None, prefix_len=self.prefix_len)

    def exact(self, cap=0.0):
        """out, lse, and what a call may be off in either (as in test_attention_of_many_tiles)"""
        scale = self.size ** -0.5
        want, want_lse, sizes = exact_on_gpu(self.k, self.v, self.lens, self.tables, self.counts, self.prefix, self.prefix_len, self.q, scale, cap)
        n, u, eps = self.prefix_len + max(self.lens), 2.0 ** -24, torch.finfo(self.dtype).eps / 2
        off = (self.size + 4) * u * 2.5 * self.size * scale + 8 * u * cap
        rel = 2 * (off + 4 * u * 64 + 2.0 ** -21) + (2 * n + 64) * u
        return want, want_lse, sizes * (rel + P_EPS[self.dtype]) * (1 + eps) + want.abs() * eps + torch.finfo(self.dtype).tiny, rel + 4 * u * want_lse.abs()


def holds(got, exact):
    (out, lse), (want, want_lse, tol, tol_lse) = got, exact
    assert ((out.double() - want).abs() <= tol).all(), float(((out.double() - want).abs() - tol).max())
    assert ((lse.double() - want_lse).abs() <= tol_lse).all(), float(((lse.double() - want_lse).abs() - tol_lse).max())


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("group, size", [(3, 64), (6, 128), (7, 256), (5, 96), (12, 40)], ids=str)
@pytest.mark.parametrize("prefix", [0, 320], ids=["own", "prefix"])
def test_groups_that_do_not_divide_a_block(paged, group, size, prefix, dtype):
    """Tensor-core units whose queries no TMA box holds, several short ones a CTA, keys by TMA: the queries come from far away (the cache holds other things), the keys from near, and every call gives
    the same bits as the first."""
    if prefix:
        rows = (60 if size <= 128 else 15) // group   # (below the own keys' rule, so that the prefix is a line by itself)
        n = 300 * (256 if size <= 128 else 128) // (8 * group * rows)   # some 300 units of the prefix, 5 tiles each
        m = MadeThere(paged, group, dtype, [rows + 3] * n, [rows] * n, 16, 8, group, size, prefix)
    else:
        rows = -(-64 // group)
        m = MadeThere(paged, group, dtype, [rows + 70] * 60, [rows] * 60, 16, 8, group, size)   # 480 units, 2 or 3 tiles each
    exact = m.exact()
    first = paged.attention(m.pages, m.batch, m.q, return_lse=True)
    holds(first, exact)
    other = torch.empty(512 << 20, dtype=torch.uint8, device="cuda")
    for i in range(8):
        other.fill_(i)
        m.k.sum(), m.v.sum()
        out, lse = paged.attention(m.pages, m.batch, m.q, return_lse=True)
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])


def exact_of_repeats(k, v, times, n, kv, group, q, cap=0.0):
    """out, lse and sums of sizes in 64 bits for n rows at the end of `times` copies of the first page and one of the second: keys of the first count that often"""
    page, size = k.shape[1], k.shape[3]
    out, sizes = torch.empty(q.shape, dtype=torch.float64, device="cuda"), torch.empty(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(q.shape[:2], dtype=torch.float64, device="cuda")
    for h in range(kv):
        heads = slice(h * group, (h + 1) * group)
        s = torch.einsum("rgd,kd->rgk", q[:, heads].double(), k[:, :, h].reshape(-1, size).double()) * size ** -0.5
        s = cap * torch.tanh(s / cap) if cap else s
        s[..., :page] += math.log(times)
        s.masked_fill_(torch.arange(2 * page, device="cuda") > (2 * page - n + torch.arange(n, device="cuda"))[:, None, None], -math.inf)
        values, w = v[:, :, h].reshape(-1, size).double(), torch.softmax(s, -1)
        out[:, heads], sizes[:, heads], lse[:, heads] = w @ values, w @ values.abs(), torch.logsumexp(s, -1)
    return out, lse, sizes


def repeats(paged, seed, kv, group, size, page, times, n):
    """one sequence whose table names one page `times` times and then another, and its last n tokens' queries"""
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    k, v = (torch.randn(2, page, kv, size, generator=g, device="cuda").to(BF16) for _ in range(2))
    q = (1.5 * torch.randn(n, kv * group, size, generator=g, device="cuda")).to(BF16)
    batch = paged.Batch(torch.tensor([(times + 1) * page], dtype=torch.int32, device="cuda"), torch.tensor([[0] * times + [1]], dtype=torch.int32, device="cuda"),
                        rows=torch.tensor([0, n], dtype=torch.int32, device="cuda"), max_rows=n)
    return k, v, q, batch


def repeats_tolerance(want, want_lse, sizes, have, size, cap=0.0):
    """as in test_attention_of_many_tiles, but for the sums: 64 weights of a tile are added up before they join the running sum, and the tensor cores add 16 products at a time, in accumulators that
    may truncate (2 u); on CUDA cores 128 terms at a time"""
    eps, u = 2.0 ** -8, 2.0 ** -24
    rel = 2 * ((size + 4) * u * 2.5 * size * size ** -0.5 + 8 * u * cap + 4 * u * 64 + 2.0 ** -21) + (have // 64 + 2 * (have // 16) + 2 * 128 + 64) * u
    return sizes * (rel + eps) * (1 + eps) + want.abs() * eps + torch.finfo(BF16).tiny, rel + 4 * u * want_lse.abs()


def test_rows_summed_again_while_others_wait(paged):
    """An infinity in the last value of one KV head, behind 150 thousand keys, where 63 tokens x 4 heads do not see it: summing them again takes seconds, and what the same CTA has yet to do
    (the next head's keys) is as it would be otherwise."""
    kv, group, size, n, head = 75, 4, 64, 128, 1   # 150 units of 256 rows for 148 CTAs: one has the end of this head's second unit, then the begin of the next head's
    k, v, q, batch = repeats(paged, 5, kv, group, size, 1024, 146, n)
    v[1, -1, head, 7] = math.inf
    out, lse = paged.attention(paged.KVPages(k, v), batch, q, return_lse=True)
    seers = out.view(n, kv, group, size)[n - 1, head, :, 7]
    assert torch.isposinf(seers).all()
    v[1, -1, head, 7] = 0.0   # (for the comparison: a place that its seers' column alone has)
    want, want_lse, sizes = exact_of_repeats(k, v, 146, n, kv, group, q)
    tol, tol_lse = repeats_tolerance(want, want_lse, sizes, 147 * 1024, size)
    seers.copy_(want.view(n, kv, group, size)[n - 1, head, :, 7])
    holds((out, lse), (want, want_lse, tol, tol_lse))


def test_a_part_of_seconds(paged):
    """heads of 256, whose units have one block of rows: the CTA's second group waits for the end of the part, which here takes more than two seconds: 120 million keys (a page that the table names 234375 times)"""
    kv, size, n = 148, 256, 128
    k, v, q, batch = repeats(paged, 6, kv, 1, size, 512, 234375, n)
    out, lse = paged.attention(paged.KVPages(k, v), batch, q, softcap=30.0, return_lse=True)
    want, want_lse, sizes = exact_of_repeats(k, v, 234375, n, kv, 1, q, 30.0)
    holds((out, lse), (want, want_lse, *repeats_tolerance(want, want_lse, sizes, 234376 * 512, size, 30.0)))


def test_results_over_what_is_read(paged):
    """a result shifted against its input is refused; one that interleaves with it (a projection's queries, turned in place, and a place for the results beside them) is not"""
    m = Made(paged, 1, BF16, [40, 50, 3], [1, 1, 1], 16, 2, 2, 64, 20, one_each=True)
    pages, batch = m.on_gpu()
    buf = torch.zeros(4, 4, 64, dtype=BF16, device="cuda")
    buf[:3] = m.q.cuda()
    rope = paged.RopeAxes.sections(64, 1e4)
    pos, k = torch.tensor([3, 5, 7], dtype=torch.int32, device="cuda"), torch.zeros(3, 2, 64, dtype=BF16, device="cuda")
    for call in (lambda: paged.attention(pages, batch, buf[:3], out=buf[1:]), lambda: paged.rope_axes(buf[:3], pos, rope, out=buf[1:]), lambda: paged.append(pages, batch, k, k, rope=rope, q=buf[:3], q_out=buf[1:]),
                 lambda: paged.append(pages, batch, buf[:3, 1:3], k, rope=rope, q=m.q.cuda(), q_out=buf[:3])):
        with pytest.raises(paged.LmrsError, match="lies"):
            call()
    assert torch.equal(buf[:3], m.q.cuda())
    wide = torch.randn(3, 12, 64, generator=gen(2)).to(BF16).cuda()   # 4 heads of q, 2 of k, 2 of v, 4 of results
    q, kk, v, out = wide[:, :4], wide[:, 4:6], wide[:, 6:8], wide[:, 8:]
    want = paged.rope_axes(q.contiguous(), pos, rope)
    rest = wide[:, 4:8].clone()
    assert paged.append(pages, batch, kk, v, rope=rope, pos=pos, q=q, q_out=q) is q
    assert torch.equal(q, want) and torch.equal(wide[:, 4:8], rest)
    paged.attention(pages, batch, q, out=out)
    assert torch.equal(out, paged.attention(pages, batch, want)) and torch.equal(q, want)


def test_gradients_are_refused_not_dropped(paged):
    m = Made(paged, 1, F32, [40, 50], [1, 1], 16, 2, 2, 64, 20, one_each=True)
    pages, batch = m.on_gpu()
    q, k = m.q.cuda(), torch.randn(2, 2, 64, generator=gen(1)).cuda()
    rope, pos = paged.RopeAxes.sections(64, 1e4), torch.zeros(2, dtype=torch.int32, device="cuda")
    p, kp = q.clone().requires_grad_(), k.clone().requires_grad_()
    calls = (lambda t, u: paged.rope_axes(t, pos, rope), lambda t, u: paged.attention(pages, batch, t), lambda t, u: paged.append(pages, batch, u, k, rope=rope, q=q), lambda t, u: paged.append(pages, batch, k, u),
             lambda t, u: paged.append(pages, batch, k, k, rope=rope, q=t), lambda t, u: paged.KVPages(u[:, None], u[:, None]), lambda t, u: paged.rope_axes(t * 2.0, pos, rope))
    for call in calls:
        with pytest.raises(paged.LmrsError, match="gradient"):
            call(p, kp)
        with torch.no_grad():
            got = call(p, kp)
        want = call(q, k)
        assert not isinstance(want, torch.Tensor) or (torch.equal(got, want) and not got.requires_grad)
        call(p.detach(), kp.detach())
    with pytest.raises(paged.LmrsError, match="out requires a gradient"):
        paged.rope_axes(q, pos, rope, out=torch.zeros_like(q).requires_grad_())


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_caps_and_scales_at_the_ends_of_float32(paged, dtype):
    """a cap so small that every score is 0, one so large that none is capped, a scale at the end: keys of zeros among the others, and queries of zeros"""
    m = Made(paged, 9, dtype, [70, 90, 1], [1, 40, 1], 16, 2, 2, 64, 50)
    for b, x in ((0, 3), (0, 69), (1, 5), (1, 60)):
        m.k[oracle.place(m.tables[b], len(m.k), 16, x)] = 0.0
    m.q[[0, 7]] = 0.0
    pages, batch = m.on_gpu()
    q = m.q.cuda()
    for cap in (1e-45, 1e-40, 3e38):
        out, lse = paged.attention(pages, batch, q, softcap=cap, return_lse=True)
        m.check(out, lse, cap=cap if cap < 1 else 0.0)
    rows = (q == 0).flatten(1).all(1)   # whatever the scale, a row of zeros weighs all keys alike
    assert torch.equal(paged.attention(pages, batch, q, scale=3e38)[rows], paged.attention(pages, batch, q)[rows])


def longer_and_shorter(m, seed):
    """other lengths (none longer than its pages), the pages of two sequences of one length exchanged"""
    r = random.Random(seed)
    m.lens = [max(c, n - r.randrange(0, n // 2 + 1)) for n, c in zip(m.lens, m.counts)]
    return torch.tensor(m.lens, dtype=torch.int32, device="cuda"), m.tables[torch.randperm(len(m.lens), generator=gen(seed))]


@pytest.mark.parametrize("what", ["prefix", "own"])
def test_tensor_core_calls_on_two_streams_and_two_graphs(paged, what):
    """a prefix on the tensor cores, then the own keys on others, then the join, each launched before the one in front of it has ended; or own keys of many rows on the tensor cores, then the join.
    Two batches at the same time, eager and as graphs that are replayed together, lengths and pages changed between replays: each what it is alone, which is held against 64 bits"""
    if what == "prefix":
        made = [MadeThere(paged, s, BF16, [300] * 64, [1] * 64, 16, 8, 4, 64, 5120 + 100 * s) for s in (1, 2)]
    else:
        made = [MadeThere(paged, s, F16, [300] * 16, [20] * 16, 16, 8, 4, 128) for s in (3, 4)]
    for m in made:   # (pages change hands: every length fits every row of the table)
        m.k.nan_to_num_(0.5), m.v.nan_to_num_(0.5)
    lens, tables = [m.batch.lens for m in made], [m.tables for m in made]

    def call(i):
        return paged.attention(made[i].pages, made[i].batch, made[i].q, return_lse=True)

    streams, graphs, outs = [torch.cuda.Stream() for _ in made], [], []
    for i in range(2):
        call(i)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(i))
        graphs.append(graph)
    for step in range(6):
        if step:
            for i, m in enumerate(made):
                new_lens, new_tables = longer_and_shorter(m, 10 * step + i)
                lens[i].copy_(new_lens)
                tables[i].copy_(new_tables.clone())
        alone = [[t.clone() for t in call(i)] for i in range(2)]
        for i, m in enumerate(made):
            holds(alone[i], m.exact())
        torch.cuda.synchronize()
        got = [[], []]
        for _ in range(10):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    got[i].append(call(i))
        torch.cuda.synchronize()
        assert all(torch.equal(g[j], alone[i][j]) for i in range(2) for g in got[i] for j in range(2))
        for _ in range(10):
            for o, l in outs:
                o.fill_(9.0), l.fill_(9.0)
            torch.cuda.synchronize()
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(outs[i][j], alone[i][j]) for i in range(2) for j in range(2))


ROWS_AND_HEADS = [  # tokens before, rows of each sequence, page, kv heads, group, size, prefix, cap
    (60, [40, 17], 16, 2, 4, 24, 300, 0.0), (100, [70] * 3, 32, 3, 2, 40, 0, 0.0), (200, [33] * 4, 8, 2, 2, 8, 90, 0.0), (90, [64, 100], 16, 2, 8, 56, 700, 20.0), (30, [130], 64, 1, 1, 16, 0, 0.0),
    (500, [200] + [1] * 40, 16, 4, 4, 64, 0, 0.0), (500, [200] + [1] * 40, 16, 2, 4, 128, 600, 0.0), (300, [1, 1, 60, 1, 2, 90], 32, 2, 3, 96, 100, 0.0), (700, [512] + [1] * 20, 16, 2, 4, 64, 0, 0.0),
    (100, [128, 100, 300], 16, 8, 4, 64, 0, 0.0), (100, [128, 100, 300], 16, 4, 1, 96, 0, 0.0), (100, [128, 100, 300], 16, 2, 4, 128, 0, 0.0), (64, [16] * 9, 16, 2, 1, 256, 200, 0.0),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("case", ROWS_AND_HEADS, ids=lambda c: f"past{c[0]}-rows{'+'.join(map(str, sorted(set(c[1]))))}-page{c[2]}-{c[3]}x{c[4]}x{c[5]}-prefix{c[6]}")
def test_portions_beside_single_tokens_and_narrow_heads(paged, case, dtype):
    """prompts' portions by themselves and with single tokens of other sequences in the same call, heads that fill a part of a box; and the same with a max_rows that is wrong in either direction"""
    past, counts, page, kv, group, size, prefix, cap = case
    m = MadeThere(paged, size + page, dtype, [past + c for c in counts], counts, page, kv, group, size, prefix)
    exact = m.exact(cap)
    for max_rows in (None, 1, 7, 100000):
        holds(paged.attention(m.pages, m.batch_of(max_rows), m.q, softcap=cap, return_lse=True), exact)


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("counts, group, prefix", [([7, 2, 1], 2, 70), ([7, 2, 1], 2, 0), ([3, 15, 1], 1, 0), ([15, 8, 3], 4, 33)], ids=str)
def test_values_that_are_not_finite_in_few_rows(paged, dtype, counts, group, prefix):
    """as test_values_that_are_not_finite, in units of up to 16 rows: some rows of a sequence see the value, those before it do not"""
    m = Made(paged, 12, dtype, [130, 80, 50], counts, 16, 2, group, 64, prefix)
    for b, head, column, value, keys in ((0, 1, 3, math.inf, False), (0, 0, 5, math.nan, True), (1, 0, 63, math.nan, False), (1, 1, 0, -math.inf, False)):
        x = m.lens[b] - max(1, counts[b] // 2)   # (seen by the last half of the rows)
        (m.k if keys else m.v)[oracle.place(m.tables[b], len(m.k), 16, x)][head, column] = value
    out, lse = paged.attention(*m.on_gpu(), m.q.cuda(), return_lse=True)
    out, lse = out.cpu(), lse.cpu()
    want, want_lse, tol, _ = oracle.attention(m.k, m.v, m.lens, m.tables, m.rows, m.prefix, prefix, m.q, 0.125, 0.0, P_EPS[dtype])
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(torch.isinf(out), torch.isinf(want)) and torch.equal(torch.isnan(lse), torch.isnan(want_lse))
    fine = torch.isfinite(want)
    assert fine.sum() > 0.5 * fine.numel() and ((out.double() - want).abs() <= tol)[fine].all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("rows, prefix", [([1] * 20, 600), ([40, 17, 1], 0)], ids=str)
def test_strides_that_are_no_multiples_of_one_another(paged, dtype, rows, prefix):
    """keys and values in one array, page by page, with gaps that no other stride divides; queries and results with odd gaps between tokens: the same bits as packed"""
    m = MadeThere(paged, 3, dtype, [90 + c for c in rows], rows, 16, 8, 4, 64, prefix)
    want = paged.attention(m.pages, m.batch, m.q, return_lse=True)
    holds(want, m.exact())
    n, both = len(m.k), 16 * 8 * 64
    buf = torch.full((n * (2 * both + 24) + 8,), math.nan, dtype=dtype, device="cuda")
    k, v = (buf.as_strided(m.k.shape, (2 * both + 24, 8 * 64, 64, 1), at) for at in (0, both + 8))
    k.copy_(m.k), v.copy_(m.v)
    q, out = (torch.full((m.q.shape[0] * (32 * 72 + gap),), math.nan, dtype=dtype, device="cuda").as_strided(m.q.shape, (32 * 72 + gap, 72, 1)) for gap in (8, 16))
    q.copy_(m.q)
    got = paged.attention(paged.KVPages(k, v), m.batch, q, out=out, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.isnan(buf.as_strided((n, 8), (2 * both + 24, 1), both)).all()
