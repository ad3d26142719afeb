"""Pages of 8-bit codes and norms of heads: what needs no GPU -- every call that the library has to refuse (nothing is launched)."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")
P = 4096   # an aligned address, that nothing may follow


@pytest.fixture(scope="module")
def paged(gpu_lib):
    from lmrs_b200 import paged
    return paged


def _pages(paged, **kw):
    p = paged._Pages8(P, P, P, P, 16 * 2 * 64, 2 * 64, 64, 16 * 2 * 64, 2 * 64, 64, 8, 2, 1, 8, 2, 1, 8, 16, 2, 64, 4, 0)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _batch(paged, **kw):
    b = paged._Batch(P, None, P, None, 4, 3, 4, 1, 0)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


BAD_PAGES = [dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(form=2), dict(form=-1), dict(pages=0), dict(page_size=0), dict(kv_heads=0), dict(kv_heads=65536), dict(head_size=0),
             dict(head_size=257), dict(k_slot=-1), dict(v_head=-64), dict(ks_block=-1), dict(vs_page=-1), dict(block=0), dict(block=3), dict(block=32), dict(k_scale=P + 2), dict(v_scale=P + 1)]
BAD_BATCH = [dict(seqs=-1), dict(lens=None), dict(tables=None), dict(table_len=-1), dict(table_stride=-1), dict(prefix_len=-1), dict(prefix_len=1), dict(table_len=1 << 30),
             dict(prefix_len=2 ** 31 - 1, prefix=P), dict(max_rows=0), dict(seqs=2), dict(seqs=4)]


@pytest.mark.parametrize("pages, batch, dtype", [(p, {}, 0) for p in BAD_PAGES] + [({}, b, 0) for b in BAD_BATCH] + [({}, {}, 3), ({}, {}, -1)], ids=str)
def test_bad_pages_and_batches(paged, gpu_lib, pages, batch, dtype):
    L = gpu_lib.lib()
    pg, bt, rows, other = _pages(paged, **pages), _batch(paged, **batch), paged._Rows(P, 256, 64), paged._Rows(1 << 30, 256, 64)
    r, o, size = C.byref(rows), C.byref(other), C.c_size_t()
    for rc in (lambda: L.lmrs_b200_paged8_append(C.byref(pg), C.byref(bt), dtype, 3, r, r, None, None, None, None, 0, None, None),
               lambda: L.lmrs_b200_paged8_read(C.byref(pg), C.byref(bt), dtype, 3, r, o, None),
               lambda: L.lmrs_b200_paged8_attention(C.byref(pg), C.byref(bt), dtype, 3, r, o, 4, 0.125, 0.0, None, P, 1 << 30, None),
               lambda: L.lmrs_b200_paged8_attention_workspace(C.byref(pg), C.byref(bt), dtype, 3, 4, C.byref(size))):
        assert rc()
        assert b"no CUDA device" not in L.lmrs_b200_last_error()


def test_bad_attention(paged, gpu_lib):
    L = gpu_lib.lib()
    rows, other, size = paged._Rows(P, 256, 64), paged._Rows(1 << 30, 256, 64), C.c_size_t()

    def attend(heads=4, scale=0.125, cap=0.0, n=3, out=other, **pages):
        pg, bt = _pages(paged, **pages), _batch(paged)
        assert L.lmrs_b200_paged8_attention(C.byref(pg), C.byref(bt), 0, n, C.byref(rows), C.byref(out), heads, scale, cap, None, P, 1 << 30, None)
        return L.lmrs_b200_last_error()

    for kw in (dict(heads=0), dict(heads=3), dict(heads=-2), dict(heads=65536), dict(scale=math.inf), dict(scale=math.nan), dict(cap=-1.0), dict(cap=math.nan), dict(cap=math.inf), dict(head_size=56), dict(k=P + 8),
               dict(v=P + 1), dict(k_slot=136), dict(v_head=4), dict(v_page=2049), dict(n=-1), dict(n=2 ** 31), dict(out=rows)):
        assert b"no CUDA device" not in attend(**kw), kw
    assert L.lmrs_b200_paged8_attention_workspace(None, None, 0, 3, 4, C.byref(size)) and L.lmrs_b200_paged8_attention(None, None, 0, 3, None, None, 4, 1.0, 0.0, None, None, 0, None)
    pg, bt = _pages(paged), _batch(paged)
    assert L.lmrs_b200_paged8_attention_workspace(C.byref(pg), C.byref(bt), 0, 3, 4, None)
    assert L.lmrs_b200_paged8_attention_workspace(C.byref(pg), C.byref(bt), 0, 3, 4, C.byref(size)) == 0   # needs no GPU
    far = _batch(paged, table_len=(2 ** 31 - 129) // 16 + 1)
    assert L.lmrs_b200_paged8_attention_workspace(C.byref(pg), C.byref(far), 0, 3, 4, C.byref(size)) and b"2^31 - 129" in L.lmrs_b200_last_error()


def test_bad_appends_reads_and_norms(paged, gpu_lib):
    L = gpu_lib.lib()
    rope, wide = paged.RopeAxes([1.0] * 32)._c, paged.RopeAxes([1.0] * 33)._c
    pg, bt, rows, pos = _pages(paged), _batch(paged), paged._Rows(P, 256, 64), paged._Positions(P, 3, 1)
    far, near, empty = paged._Rows(1 << 30, 256, 64), paged._Rows(P + 2, 256, 64), paged._Rope()
    r, f, o, turn = C.byref(rows), C.byref(far), C.byref(near), C.byref(rope)

    def append(rope=turn, q=None, q_out=None, heads=4, eps=1e-6, k=None, w=None):
        norms = paged._Norms(k, w, 64, 64, eps)
        assert L.lmrs_b200_paged8_append(C.byref(pg), C.byref(bt), 0, 3, r, r, rope, None, q, q_out, heads, C.byref(norms), None)
        return L.lmrs_b200_last_error()

    for kw in (dict(q=r), dict(q_out=r), dict(rope=None, q=f, q_out=f), dict(q=f, q_out=f, heads=0), dict(q=f, q_out=f, heads=65536), dict(rope=C.byref(wide)), dict(rope=C.byref(empty)), dict(eps=-1.0), dict(eps=math.nan),
               dict(eps=math.inf), dict(q=r, q_out=o), dict(q=f, q_out=r), dict(q=f, q_out=f, w=(1 << 30) + 100), dict(q=f, q_out=f, k=(1 << 30) - 60)):
        assert b"no CUDA device" not in append(**kw), kw
    for args in ((None, f), (r, None), (r, o), (r, r)):
        assert L.lmrs_b200_paged8_read(C.byref(pg), C.byref(bt), 0, 3, *args, None) and b"no CUDA device" not in L.lmrs_b200_last_error()

    def norm(rope=turn, dtype=0, x=r, out=r, n=3, heads=4, size=64, w=None, eps=1e-6, pos=C.byref(pos)):
        assert L.lmrs_b200_norm_rope(rope, dtype, x, out, n, heads, size, w, 0, eps, pos, None)
        return L.lmrs_b200_last_error()

    for kw in (dict(rope=None), dict(rope=C.byref(wide)), dict(rope=C.byref(empty)), dict(dtype=3), dict(x=None), dict(out=None), dict(pos=None), dict(n=-1), dict(heads=-1), dict(heads=65536), dict(size=0), dict(size=257),
               dict(size=63), dict(out=o), dict(eps=-1e-9), dict(eps=math.nan), dict(w=P + 64), dict(w=P - 252)):
        assert b"no CUDA device" not in norm(**kw), kw
    if not torch.cuda.is_available():   # calls in order say that there is no GPU
        assert b"no CUDA device" in norm() and b"no CUDA device" in norm(rope=None, pos=None) and b"no CUDA device" in norm(w=P - 256) and b"no CUDA device" in append()
        assert b"no CUDA device" in append(q=f, q_out=f) and b"no CUDA device" in append(rope=None, q=f, q_out=f, w=P)
        assert L.lmrs_b200_paged8_read(C.byref(pg), C.byref(bt), 0, 3, r, f, None) and b"no CUDA device" in L.lmrs_b200_last_error()
        assert L.lmrs_b200_paged8_attention(C.byref(pg), C.byref(bt), 0, 3, r, f, 4, 0.125, 0.0, None, P, 1 << 30, None) and b"no CUDA device" in L.lmrs_b200_last_error()


def test_pools_that_are_refused(paged, monkeypatch):
    monkeypatch.setattr(paged, "_gpu", lambda t, name, device: None)

    def make(k=(3, 16, 2, 64), v=None, ks=(3, 4, 2), vs=None, form=torch.int8, v_form=None, kind=torch.float32):
        return paged.QuantPages(torch.zeros(k).to(form), torch.zeros(v or k).to(v_form or form), torch.zeros(ks, dtype=kind), torch.zeros(vs or ks))

    assert make().block == 4 and make(form=torch.float8_e4m3fn, ks=(3, 16, 2)).block == 1 and make(ks=(3, 1, 2)).block == 16
    for kw in (dict(k=(3, 16, 64)), dict(v=(3, 16, 2, 32)), dict(ks=(3, 5, 2)), dict(ks=(3, 0, 2)), dict(ks=(2, 4, 2)), dict(ks=(3, 4, 1)), dict(vs=(3, 2, 2)), dict(form=torch.uint8), dict(form=torch.bfloat16),
               dict(form=torch.float8_e5m2), dict(v_form=torch.float8_e4m3fn), dict(kind=torch.float16), dict(ks=(3, 32, 2)), dict(ks=(3, 4))):
        with pytest.raises(paged.LmrsError):
            make(**kw)
    c, s = torch.zeros(3, 16, 2, 64, dtype=torch.int8), torch.zeros(3, 4, 2)
    for bad in ((c[..., ::2], c[..., ::2], s, s), (c[:1].expand(3, 16, 2, 64), c, s, s), (c, c, s[:1].expand(3, 4, 2), s), (c, c, s, s.clone().requires_grad_())):
        with pytest.raises(paged.LmrsError):
            paged.QuantPages(*bad)


def test_host_tensors_and_other_arguments_are_refused(paged):
    x = torch.zeros(2, 3, 64)
    c, s = torch.zeros(3, 16, 2, 64, dtype=torch.int8), torch.zeros(3, 4, 2)
    for bad in (lambda: paged.norm_rope(x), lambda: paged.norm_rope(x[0]), lambda: paged.norm_rope(x.double()), lambda: paged.norm_rope(None), lambda: paged.QuantPages(c, c, s, s), lambda: paged.QuantPages(None, c, s, s),
                lambda: paged.read(None, None), lambda: paged.norm_rope(x, rope=paged.RopeAxes([1.0])), lambda: paged.norm_rope(x, pos=x), lambda: paged.norm_rope(x, rope=3, pos=x)):
        with pytest.raises(paged.LmrsError):
            bad()


def test_reading_without_the_number_of_rows(paged, monkeypatch):
    """a batch with rows of its own does not say here how many they are: fewer would be other tokens"""
    monkeypatch.setattr(paged, "_gpu", lambda t, name, device: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)
    asked = []
    monkeypatch.setattr(paged, "lib", lambda: type("Lib", (), {"lmrs_b200_paged8_read": staticmethod(lambda pages, batch, dtype, n, k, v, stream: asked.append(n) or 0)}))
    monkeypatch.setattr(paged, "_stream", lambda index: None)
    monkeypatch.setattr(paged, "_heads", lambda t, name, device, dtype, *shape, out=False: paged._Rows(t.data_ptr(), *t.stride()[:2]) if t.shape == shape else paged._need(False, name))
    ints = dict(dtype=torch.int32)
    codes, scales = torch.zeros(3, 16, 2, 64, dtype=torch.int8), torch.zeros(3, 4, 2)
    pages, lens, tables = paged.QuantPages(codes, codes, scales, scales), torch.tensor([10, 20], **ints), torch.zeros(2, 2, **ints)
    each, several = paged.Batch(lens, tables), paged.Batch(lens, tables, rows=torch.tensor([0, 4, 9], **ints), max_rows=5)
    with pytest.raises(paged.LmrsError, match="rows"):
        paged.read(pages, several)
    assert not asked
    k, v = (torch.zeros(9, 2, 64) for _ in range(2))
    assert paged.read(pages, each)[0].shape == (2, 2, 64) and paged.read(pages, several, rows=9)[0].shape == (9, 2, 64) and paged.read(pages, several, k=k, v=v)[0] is k
    assert asked == [2, 9, 9]
    with pytest.raises(paged.LmrsError):
        paged.read(pages, several, rows=8, k=k, v=v)
