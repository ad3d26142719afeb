"""Many sequences at once: what needs no GPU -- the rotary tables, and every call that the library has to refuse (nothing is launched)."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def paged(gpu_lib):
    from lmrs_b200 import paged
    return paged


def test_turns_are_the_frequencies_modulo_a_turn(paged):
    freq = [1.0, 0.5, 1e-6, 0.0, 7.0, -0.25, 2 * math.pi]
    r = paged.RopeAxes(freq, [0, 1, 2, 0, 1, 2, 0], layout="pairs")
    assert (r.pairs, r.axes, r._c.pairs, r._c.axes, r._c.layout) == (7, 3, 7, 3, 1)
    for j, f in enumerate(freq):
        turns = r._c.turns[j] / 2.0 ** 64
        want = (f / (2 * math.pi)) % 1.0
        assert min(abs(turns - want), 1 - abs(turns - want)) < 2.0 ** -52
    assert list(r._c.axis[:7]) == [0, 1, 2, 0, 1, 2, 0]


def test_sections(paged):
    assert list(paged.RopeAxes.sections(16, 1e4, [2, 3, 3])._c.axis[:8]) == [0, 0, 1, 1, 1, 2, 2, 2]
    assert list(paged.RopeAxes.sections(16, 1e4, [1, 3, 4], order="cycle")._c.axis[:8]) == [0, 1, 2, 1, 2, 1, 2, 2]
    assert paged.RopeAxes.sections(64, 1e4).axes == 1
    for bad in (dict(rot=15), dict(rot=16, sections=[4, 5]), dict(rot=16, sections=[9, -1]), dict(rot=16, order="x"), dict(rot=0), dict(rot=258)):
        with pytest.raises(paged.LmrsError):
            paged.RopeAxes.sections(**{"theta": 1e4, **bad})
    for freq, axis, layout in (([], None, "halves"), ([1.0] * 129, None, "halves"), ([math.inf], None, "halves"), ([math.nan], None, "pairs"), ([1.0], [256], "halves"),
                               ([1.0], [-1], "halves"), ([1.0], [0, 0], "halves"), ([1.0], None, "thirds")):
        with pytest.raises(paged.LmrsError):
            paged.RopeAxes(freq, axis, layout)


def test_host_tensors_are_refused(paged):
    x, pos = torch.zeros(2, 3, 8), torch.zeros(2, dtype=torch.int32)
    rope = paged.RopeAxes([1.0])
    with pytest.raises(paged.LmrsError, match="GPU"):
        paged.rope_axes(x, pos, rope)
    with pytest.raises(paged.LmrsError, match="GPU"):
        paged.KVPages(torch.zeros(1, 1, 1, 8), torch.zeros(1, 1, 1, 8))
    with pytest.raises(paged.LmrsError, match="GPU"):
        paged.Batch(pos, pos[:, None])
    for bad in (lambda: paged.rope_axes(x.numpy(), pos, rope), lambda: paged.rope_axes(x, pos, None), lambda: paged.KVPages(None, None), lambda: paged.Batch(None, None)):
        with pytest.raises(paged.LmrsError):
            bad()


def test_disjoint(paged):
    t = torch.zeros(4, 6, 8)
    assert paged._disjoint(t) and paged._disjoint(t.transpose(0, 1)) and paged._disjoint(t[:, ::2]) and paged._disjoint(t[:1].expand(1, 6, 8)) and paged._disjoint(t[:0])
    assert not paged._disjoint(t[:1].expand(4, 6, 8)) and not paged._disjoint(torch.zeros(100).as_strided((4, 6, 8), (4, 8, 1)))


# ---- the C entry points: pointers that nothing may follow, because every one of these calls is refused before a launch ----
P = 4096   # an aligned address


def _pages(paged, **kw):
    p = paged._Pages(P, P, 16 * 2 * 64, 2 * 64, 64, 16 * 2 * 64, 2 * 64, 64, 8, 16, 2, 64, 0)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _batch(paged, **kw):
    b = paged._Batch(P, None, P, None, 4, 3, 4, 1, 0)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


BAD_PAGES = [dict(k=None), dict(v=None), dict(dtype=3), dict(dtype=-1), dict(pages=0), dict(page_size=0), dict(kv_heads=0), dict(head_size=0), dict(head_size=257), dict(k_slot=-1), dict(v_head=-64)]
BAD_BATCH = [dict(seqs=-1), dict(lens=None), dict(tables=None), dict(table_len=-1), dict(table_stride=-1), dict(prefix_len=-1), dict(prefix_len=1), dict(table_len=1 << 30),
             dict(prefix_len=2 ** 31 - 1, prefix=P), dict(max_rows=0), dict(seqs=2), dict(seqs=4)]


@pytest.mark.parametrize("pages, batch", [(p, {}) for p in BAD_PAGES] + [({}, b) for b in BAD_BATCH], ids=str)
def test_bad_pages_and_batches(paged, gpu_lib, pages, batch):
    L = gpu_lib.lib()
    pg, bt, rows = _pages(paged, **pages), _batch(paged, **batch), paged._Rows(P, 256, 64)
    r, size = C.byref(rows), C.c_size_t()
    assert L.lmrs_b200_paged_append(C.byref(pg), C.byref(bt), 3, r, r, None, None, None, None, 0, None)
    assert b"no CUDA device" not in L.lmrs_b200_last_error()
    assert L.lmrs_b200_paged_attention(C.byref(pg), C.byref(bt), 3, r, r, 4, 0.125, 0.0, None, P, 1 << 30, None)
    assert b"no CUDA device" not in L.lmrs_b200_last_error()
    assert L.lmrs_b200_paged_attention_workspace(C.byref(pg), C.byref(bt), 3, 4, C.byref(size))


def test_bad_attention(paged, gpu_lib):
    L = gpu_lib.lib()
    rows, size = paged._Rows(P, 256, 64), C.c_size_t()
    r = C.byref(rows)

    def attend(heads=4, scale=0.125, cap=0.0, n=3, **pages):
        pg, bt = _pages(paged, **pages), _batch(paged)
        assert L.lmrs_b200_paged_attention(C.byref(pg), C.byref(bt), n, r, r, heads, scale, cap, None, P, 1 << 30, None)
        return L.lmrs_b200_last_error()

    for kw in (dict(heads=0), dict(heads=3), dict(heads=-2), dict(scale=math.inf), dict(scale=math.nan), dict(cap=-1.0), dict(cap=math.nan), dict(cap=math.inf), dict(head_size=60), dict(k=P + 2),
               dict(v=P + 8), dict(k_slot=132), dict(v_head=4), dict(v_page=2049), dict(n=-1), dict(n=2 ** 31)):
        assert b"no CUDA device" not in attend(**kw), kw
    assert L.lmrs_b200_paged_attention_workspace(None, None, 3, 4, C.byref(size)) and L.lmrs_b200_paged_attention(None, None, 3, r, r, 4, 1.0, 0.0, None, None, 0, None)
    pg, bt = _pages(paged), _batch(paged)
    assert L.lmrs_b200_paged_attention_workspace(C.byref(pg), C.byref(bt), 3, 4, None)
    assert L.lmrs_b200_paged_attention_workspace(C.byref(pg), C.byref(bt), 3, 4, C.byref(size)) == 0   # needs no GPU


def test_bad_appends_and_rotations(paged, gpu_lib):
    L = gpu_lib.lib()
    rope, wide = paged.RopeAxes([1.0] * 32)._c, paged.RopeAxes([1.0] * 33)._c
    pg, bt, rows, pos = _pages(paged), _batch(paged), paged._Rows(P, 256, 64), paged._Positions(P, 3, 1)
    r, empty = C.byref(rows), paged._Rope()

    def append(rope, q, q_out, heads):
        assert L.lmrs_b200_paged_append(C.byref(pg), C.byref(bt), 3, r, r, rope, None, q, q_out, heads, None)
        return L.lmrs_b200_last_error()

    for args in ((C.byref(rope), r, None, 4), (C.byref(rope), None, r, 4), (None, r, r, 4), (C.byref(rope), r, r, 0), (C.byref(wide), None, None, 0), (C.byref(empty), None, None, 0)):
        assert b"no CUDA device" not in append(*args)

    def turn(rope=C.byref(rope), dtype=0, x=r, out=r, n=3, heads=4, size=64, pos=C.byref(pos)):
        assert L.lmrs_b200_rope_axes(rope, dtype, x, out, n, heads, size, pos, None)
        return L.lmrs_b200_last_error()

    for kw in (dict(rope=None), dict(rope=C.byref(wide)), dict(rope=C.byref(empty)), dict(dtype=3), dict(x=None), dict(out=None), dict(pos=None), dict(n=-1), dict(heads=-1), dict(size=0), dict(size=257),
               dict(size=63)):
        assert b"no CUDA device" not in turn(**kw), kw


def test_every_refusal_without_a_gpu_says_so(paged, gpu_lib):
    if torch.cuda.is_available():
        pytest.skip("a GPU is there")
    L = gpu_lib.lib()
    pg, bt, rows, pos, rope = _pages(paged), _batch(paged), paged._Rows(P, 256, 64), paged._Positions(P, 3, 1), paged.RopeAxes([1.0] * 32)._c
    r = C.byref(rows)
    assert L.lmrs_b200_paged_attention(C.byref(pg), C.byref(bt), 3, r, r, 4, 0.125, 0.0, None, P, 1 << 30, None) and b"no CUDA device" in L.lmrs_b200_last_error()
    assert L.lmrs_b200_paged_append(C.byref(pg), C.byref(bt), 3, r, r, C.byref(rope), None, None, None, 0, None) and b"no CUDA device" in L.lmrs_b200_last_error()
    assert L.lmrs_b200_rope_axes(C.byref(rope), 0, r, r, 3, 4, 64, C.byref(pos), None) and b"no CUDA device" in L.lmrs_b200_last_error()


def test_every_asynchronous_copy_belongs_to_a_group():
    """A wait for groups waits for committed copies only.  In the tensor-core kernel, whatever asks for copies by threads (queries, operand tiles without TMA) commits them before it says that they are on
    their way: read from the source, since a copy that is late shows itself by chance only."""
    import os
    import re
    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lm.rs_b200", "csrc", "paged_tensor.cuh")).read()
    asked = [m.start() for m in re.finditer(r"copy16\(", src)]
    handed_on = [m.start() for m in re.finditer(r"asked = true;|next_slot\(\);", src)]
    assert len(asked) == 3 and "asked = true;" in src
    for at in asked:
        end = min(p for p in handed_on if p > at)
        assert "copy_commit();" in src[at:end], src[at:at + 80]


# q (or x, k) and a result: data in elements from one place, row and head strides, n_rows, heads; is it refused?
LIE = [
    ((0, 256, 64), (0, 256, 64), 3, 4, "itself"), ((0, 256, 64), (256, 256, 64), 3, 4, True), ((0, 256, 64), (768, 256, 64), 3, 4, False), ((768, 256, 64), (0, 256, 64), 3, 4, False),
    ((0, 256, 64), (8, 256, 64), 3, 4, True), ((767, 256, 64), (0, 256, 64), 3, 4, True), ((0, 512, 64), (256, 512, 64), 3, 4, False), ((0, 512, 64), (255, 512, 64), 3, 4, True), ((256, 512, 64), (0, 512, 64), 3, 4, False),
    ((0, 512, 128), (64, 512, 128), 3, 4, False), ((0, 512, 128), (63, 512, 128), 3, 4, True), ((0, 64, 64 * 9), (64 * 3, 64, 64 * 9), 3, 4, False), ((0, 64, 64 * 9), (64 * 2, 64, 64 * 9), 3, 4, True),
    ((0, 256, 64), (0, 64, 192), 3, 4, True), ((0, 256, 64), (0, 7, 64), 1, 4, "itself"), ((0, 999, 64), (256, 1, 64), 1, 4, False), ((0, 999, 64), (192, 1, 64), 1, 4, True), ((0, 64, 5), (0, 64, 7), 3, 1, "itself"),
    ((0, 128, 5), (64, 128, 7), 3, 1, False), ((0, 128, 5), (32, 128, 7), 3, 1, True), ((0, 0, 64), (512, 256, 64), 3, 4, False), ((0, 0, 64), (128, 256, 64), 3, 4, True), ((0, 300, 64), (60 * 300, 300, 64), 60, 4, False),
    ((0, 300, 64), (59 * 300, 300, 64), 60, 4, True), ((0, 2 ** 40, 2 ** 35), (2 ** 20, 2 ** 40, 2 ** 35), 60, 4, False),
    ((0, 600, 64), (256, 600, 70), 5, 4, False), ((256, 600, 70), (0, 600, 64), 5, 4, False), ((0, 600, 64), (255, 600, 70), 5, 4, True), ((0, 600, 64), (326, 600, 70), 5, 4, False), ((0, 600, 64), (327, 600, 70), 5, 4, True),
]


@pytest.mark.parametrize("a, b, n, heads, lies", LIE, ids=str)
def test_results_that_lie_over_what_is_read(paged, gpu_lib, a, b, n, heads, lies):
    """a shifted result is refused, an interleaved one is not, wherever rows and heads lie (held against the elements themselves where they are few)"""
    L = gpu_lib.lib()
    base = 1 << 44
    x, y = (paged._Rows(base + 2 * t[0], t[1], t[2]) for t in (a, b))
    if max(a + b) < 10 ** 6:
        places = [{t[0] + r * t[1] + h * t[2] + e for r in range(n) for h in range(heads) for e in range(64)} for t in (a, b)]
        meet = bool(places[0] & places[1])
        assert meet == bool(lies)
    rope, pos = paged.RopeAxes([1.0] * 32)._c, paged._Positions(P, n, 1)
    L.lmrs_b200_rope_axes(C.byref(rope), 0, C.byref(x), C.byref(y), n, heads, 64, C.byref(pos), None)
    assert (b"lies over x" in L.lmrs_b200_last_error()) == (lies is True)
    pg, bt = _pages(paged, kv_heads=1), _batch(paged, seqs=n)
    far = paged._Rows(1 << 50, 64, 64)
    L.lmrs_b200_paged_attention(C.byref(pg), C.byref(bt), n, C.byref(x), C.byref(y), heads, 0.125, 0.0, None, P, 1 << 30, None)
    if a[0] != b[0] or torch.cuda.is_available():   # (in one place: asked for behind the device)
        assert (b"lies where q does" in L.lmrs_b200_last_error()) == bool(lies)
    L.lmrs_b200_paged_append(C.byref(pg), C.byref(bt), n, C.byref(far), C.byref(far), C.byref(rope), None, C.byref(x), C.byref(y), heads, None)
    assert (b"lies over q" in L.lmrs_b200_last_error()) == (lies is True)
    if heads > 1:
        pg = _pages(paged, kv_heads=heads)
        for k, v in ((x, far), (far, x)):
            L.lmrs_b200_paged_append(C.byref(pg), C.byref(bt), n, C.byref(k), C.byref(v), C.byref(rope), None, C.byref(y), C.byref(y), heads, None)
            assert (b"lies over k or v" in L.lmrs_b200_last_error()) == bool(lies)


def test_one_projection_of_queries_keys_and_values(paged, gpu_lib):
    """q, k and v beside one another in the rows of one array, queries turned in place"""
    L = gpu_lib.lib()
    base, n = 1 << 44, 5
    for heads, kv in ((8, 2), (4, 4), (6, 1), (1, 1)):
        width = (heads + 2 * kv) * 64
        q, k, v = (paged._Rows(base + 2 * 64 * at, width, 64) for at in (0, heads, heads + kv))
        pg, bt, rope = _pages(paged, kv_heads=kv), _batch(paged, seqs=n), paged.RopeAxes([1.0] * 32)._c
        L.lmrs_b200_paged_append(C.byref(pg), C.byref(bt), n, C.byref(k), C.byref(v), C.byref(rope), None, C.byref(q), C.byref(q), heads, None)
        assert b"lies" not in L.lmrs_b200_last_error()


def test_a_torch_without_cuda_imports(paged):
    """(it has no name for the raw stream; what needs a GPU says so)"""
    import os
    import subprocess
    import sys
    code = ("import sys, torch; sys.path.insert(0, sys.argv[1])\n"
            "if hasattr(torch._C, '_cuda_getCurrentRawStream'): del torch._C._cuda_getCurrentRawStream\n"
            "from lmrs_b200 import paged\n"
            "try: paged.rope_axes(torch.zeros(2, 3, 8), torch.zeros(2, dtype=torch.int32), paged.RopeAxes([1.0]))\n"
            "except paged.LmrsError as e: print(e)\n")
    lib = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lm.rs_b200")
    r = subprocess.run([sys.executable, "-c", code, lib], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "must be a tensor on a GPU" in r.stdout, r.stderr[-500:]


def test_numbers_that_32_bits_do_not_hold(paged, monkeypatch):
    """refused, and not taken for their lower 32 bits (tensors without memory stand for those of a GPU)"""
    monkeypatch.setattr(paged, "_gpu", lambda t, name, device: None)
    i32 = dict(dtype=torch.int32)
    lens, tables, prefix = torch.zeros(2, **i32), torch.zeros(2, 3, **i32), torch.zeros(4, **i32)
    paged.Batch(lens, tables, rows=torch.zeros(3, **i32), max_rows=2 ** 31 - 1, prefix=prefix, prefix_len=2 ** 31 - 1)
    for kw in (dict(max_rows=2 ** 32 + 1), dict(max_rows=2 ** 31), dict(prefix_len=2 ** 32 + 5), dict(tables=torch.empty(2, 2 ** 32 + 1, dtype=torch.int32, device="meta"))):
        with pytest.raises(paged.LmrsError, match="2\\^31"):
            paged.Batch(lens, **{"tables": tables, "rows": torch.zeros(3, **i32), "prefix": prefix, **kw})
    for shape in ((2 ** 32 + 5, 1, 1, 1), (1, 2 ** 31, 1, 8)):
        big = torch.empty(shape, dtype=torch.bfloat16, device="meta")
        with pytest.raises(paged.LmrsError, match="2\\^31"):
            paged.KVPages(big, big)
    with pytest.raises(paged.LmrsError, match="heads"):
        paged.rope_axes(torch.empty(1, 2 ** 32 + 4, 1, dtype=torch.bfloat16, device="meta"), torch.zeros(1, **i32), paged.RopeAxes([1.0]))


def test_keys_up_to_the_end_of_32_bits(paged, gpu_lib):
    """a tile's end is a number of 32 bits, too"""
    L, size = gpu_lib.lib(), C.c_size_t()
    most = 2 ** 31 - 129
    for page, table, prefix, ok in ((most, 1, 0, True), (most + 1, 1, 0, False), (2 ** 31 - 1, 1, 0, False), (16, 4, most - 64, True), (16, 4, most - 63, False), (16, 4, 2 ** 31 - 1 - 64, False)):
        pg, bt = _pages(paged, page_size=page), _batch(paged, table_len=table, prefix=P, prefix_len=prefix)
        assert (L.lmrs_b200_paged_attention_workspace(C.byref(pg), C.byref(bt), 3, 4, C.byref(size)) == 0) == ok, (page, table, prefix)


def test_sequences_up_to_2_to_the_30(paged, gpu_lib):
    L, size, pg = gpu_lib.lib(), C.c_size_t(), _pages(paged)
    for seqs, ok in ((1 << 30, True), ((1 << 30) + 1, False), (2 ** 31 - 1, False)):
        bt = _batch(paged, seqs=seqs, rows=P)
        assert (L.lmrs_b200_paged_attention_workspace(C.byref(pg), C.byref(bt), 3, 4, C.byref(size)) == 0) == ok


def test_turns_to_the_last_bit(paged):
    """against pi in whole numbers (Machin's formula): half a step of 2^-64, and what the 128 bits of 1 / 2 pi leave of large frequencies"""
    import random
    from fractions import Fraction
    one = 1 << 1300

    def arctan(x):
        total, term, n = 0, one // x, 1
        while term:
            total += term // n if n % 4 == 1 else -(term // n)
            term, n = term // (x * x), n + 2
        return total

    two_pi = Fraction(8 * (4 * arctan(5) - arctan(239)), one)
    r = random.Random(1)
    freq = [1.0, 0.5, 7.0, -0.25, 2 * math.pi, -2 * math.pi, 1e-6, 5e-324, 1e-300, 0.0, -0.0, 1e6, 1e15, 2.0 ** 60, 2.0 ** 64 + 2.0 ** 12, -3e17, 1e300, -1e300, 2.0 ** 128]
    freq += [10000.0 ** (-2.0 * j / 128) for j in range(64)] + [math.ldexp(r.uniform(-1, 1), r.randint(-70, 70)) for _ in range(40)]
    for at in range(0, len(freq), 100):
        part = freq[at:at + 100]
        c = paged.RopeAxes(part)._c
        for j, f in enumerate(part):
            off = (Fraction(int(c.turns[j]), 2 ** 64) - Fraction(f) / two_pi) % 1
            assert min(off, 1 - off) * 2 ** 64 <= Fraction(1, 2) + Fraction(abs(f)) / 2 ** 65 + Fraction(1, 10 ** 6), f
