"""Many sequences at once: rotary positions with several axes, keys and values in pages, and attention over the pages with a prefix that all
sequences share (include/lmrs_b200.h, "many sequences at once").  Torch tensors on a GPU, the current stream of their device; nothing is copied to
the host, and calls can be captured into CUDA graphs.  Nothing here has a backward pass: tensors that require gradients are refused while torch records them.

    rope  = RopeAxes(freq, axis)                        # which axis' position turns which pair, and how fast
    pages = KVPages(k, v)                               # [pages, page_size, kv_heads, head_size] each
    batch = Batch(lens, tables, prefix=..., prefix_len=...)
    q     = append(pages, batch, k_new, v_new, rope=rope, q=q)
    out   = attention(pages, batch, q)
"""
import ctypes as C

import torch

from ._lib import LmrsError, check, lib

_DTYPES = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}


class _Rope(C.Structure):
    _fields_ = [("turns", C.c_uint64 * 128), ("axis", C.c_uint8 * 128), ("pairs", C.c_int32), ("axes", C.c_int32), ("layout", C.c_int32)]


class _Rows(C.Structure):
    _fields_ = [("data", C.c_void_p), ("row", C.c_int64), ("head", C.c_int64)]


class _Positions(C.Structure):
    _fields_ = [("data", C.c_void_p), ("axis", C.c_int64), ("row", C.c_int64)]


class _Pages(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p)] + [(n, C.c_int64) for n in ("k_page", "k_slot", "k_head", "v_page", "v_slot", "v_head")] + \
               [(n, C.c_int32) for n in ("pages", "page_size", "kv_heads", "head_size", "dtype")]


class _Batch(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("lens", "rows", "tables", "prefix")] + [("table_stride", C.c_int64)] + \
               [(n, C.c_int32) for n in ("seqs", "table_len", "max_rows", "prefix_len")]


def _need(ok, why):
    if not ok:
        raise LmrsError(why)


def _disjoint(t):
    """no two elements of t in one place (as far as strides in falling order show it)"""
    reach = 0
    for stride, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride <= reach:
            return False
        reach += stride * (n - 1)
    return True


def _gpu(t, name, device):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise LmrsError(f"{name} must be a tensor on a GPU (this library has no CPU fallback)")
    if t.device != device:
        raise LmrsError(f"{name} lies on {t.device}, other arrays of the call on {device}")


def _no_gradients(t, name):
    """nothing here has a backward pass: a history that a call would drop is refused"""
    if torch.is_grad_enabled():
        raise LmrsError(f"{name} requires a gradient, and nothing here has a backward pass: call under torch.no_grad(), or pass {name}.detach()")


# (these run in every call: messages are made only where one is raised)
def _heads(t, name, device, dtype, rows, heads, size, out=False):
    """t as the library takes it, checked: [rows, heads, size]"""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.device != device:
        _gpu(t, name, device)
    if t.requires_grad:
        _no_gradients(t, name)
    if t.dtype != dtype:
        raise LmrsError(f"{name} is {t.dtype}, other arrays of the call {dtype}")
    if t.shape != (rows, heads, size):
        raise LmrsError(f"{name} must be [{rows}, {heads}, {size}], not {list(t.shape)}")
    row, head, one = t.stride()
    if one != 1 and size != 1:
        raise LmrsError(f"the elements of a head of {name} must lie next to each other")
    if out and not t.is_contiguous() and not _disjoint(t):
        raise LmrsError(f"elements of {name} share their places")
    return _Rows(t.data_ptr(), row, head)


def _new(like):
    """a result for a call, and the same as the library takes it"""
    t = torch.empty_like(like)
    row, head, one = t.stride()
    if one != 1:   # (only where a head has one element)
        t = torch.empty(like.shape, dtype=like.dtype, device=like.device)
        row, head, one = t.stride()
    return t, _Rows(t.data_ptr(), row, head)


def _ints(t, name, device):
    _gpu(t, name, device)
    if t.dtype != torch.int32:
        raise LmrsError(f"{name} must be int32, not {t.dtype}")


def _positions(pos, axes, rows, device):
    _ints(pos, "pos", device)
    shape = pos.shape
    if len(shape) == 2 and shape[0] >= axes and shape[1] == rows:
        return _Positions(pos.data_ptr(), *pos.stride())
    if len(shape) == 1 and axes == 1 and shape[0] == rows:
        return _Positions(pos.data_ptr(), 0, pos.stride(0))
    raise LmrsError(f"pos must be [{axes}, {rows}], not {list(shape)}")


# torch.cuda.current_stream(device).cuda_stream without the objects (2 us of a call's 10), where torch has it: a build without CUDA imports this and is refused by the calls
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_byref = C.byref


class RopeAxes:
    """Pair j of a head turns by pos[axis[j]] * freq[j] radians.  layout "halves": pair j is elements j and j + pairs; "pairs": elements
    2j and 2j + 1.  Elements from 2 * len(freq) on are left as they are.  axis None: one axis."""

    def __init__(self, freq, axis=None, layout="halves"):
        freq = [float(f) for f in freq]
        axis = [0] * len(freq) if axis is None else [int(a) for a in axis]
        _need(len(axis) == len(freq), f"{len(freq)} frequencies, {len(axis)} axes")
        _need(all(0 <= a < 256 for a in axis), "an axis is not in 0 .. 255")
        _need(layout in ("halves", "pairs"), f"layout must be 'halves' or 'pairs', not {layout!r}")
        self._c = _Rope()
        check(lib().lmrs_b200_rope_init(C.byref(self._c), (C.c_double * max(1, len(freq)))(*freq), (C.c_uint8 * max(1, len(axis)))(*axis), len(freq), int(layout == "pairs")))
        self.pairs, self.axes, self.layout, self._ref = len(freq), self._c.axes, layout, C.byref(self._c)

    @classmethod
    def sections(cls, rot, theta, sections=None, order="blocks", layout="halves"):
        """The usual frequencies theta^(-2j / rot) of `rot` elements; sections[a] of the pairs belong to axis a, one block after the other, or
        (order "cycle") turn by turn as long as an axis has pairs left."""
        pairs = rot // 2
        left = [pairs] if sections is None else [int(n) for n in sections]
        _need(rot > 0 and rot % 2 == 0, "rot must be positive and even")
        _need(all(n >= 0 for n in left) and sum(left) == pairs, f"sections must add up to {pairs}, not {left}")
        _need(order in ("blocks", "cycle"), f"order must be 'blocks' or 'cycle', not {order!r}")
        axis = []
        if order == "blocks":
            axis = [a for a, n in enumerate(left) for _ in range(n)]
        else:
            while any(left):
                for a, n in enumerate(left):
                    if n:
                        axis.append(a)
                        left[a] -= 1
        return cls([float(theta) ** (-2.0 * j / rot) for j in range(pairs)], axis, layout)


class KVPages:
    """The pool: keys and values [pages, page_size, kv_heads, head_size], in any order of the first three dimensions."""

    def __init__(self, k, v):
        _gpu(k, "k", k.device if isinstance(k, torch.Tensor) else None)
        _gpu(v, "v", k.device)
        _need(k.dim() == 4 and k.shape == v.shape, f"k and v must be [pages, page_size, kv_heads, head_size] alike, not {list(k.shape)} and {list(v.shape)}")
        _need(k.dtype in _DTYPES and k.dtype == v.dtype, f"k and v must both be bfloat16, float16 or float32, not {k.dtype} and {v.dtype}")
        for t, name in ((k, "k"), (v, "v")):
            if t.requires_grad:
                _no_gradients(t, name)
            _need(t.stride(3) == 1 or t.shape[3] == 1, f"the elements of a head of {name} must lie next to each other")
            _need(_disjoint(t), f"elements of {name} share their places")
        _need(max(k.shape) < 1 << 31, f"a dimension of {list(k.shape)} is beyond 2^31 - 1")   # (ctypes would keep its lower 32 bits)
        self.k, self.v, self.device, self.dtype = k, v, k.device, k.dtype
        self.pages, self.page_size, self.kv_heads, self.head_size = k.shape
        self._c = _Pages(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), v.stride(0), v.stride(1), v.stride(2), *k.shape, _DTYPES[k.dtype])
        self._ref = C.byref(self._c)


class Batch:
    """The sequences of a call.  lens [seqs]: tokens that each holds, those of the call included (which are its last).  tables [seqs, n]: the pages of
    each, in order.  rows [seqs + 1]: the first row of each in the call's arrays (None: one row each); max_rows: most rows of one sequence.  A
    row whose place would be before the first token (so the row of a sequence with lens 0) is padding; rows from rows[seqs] on are not touched, and in a
    result that a call allocates they hold anything.  prefix: the pages of the prefix_len tokens that come before every sequence's own.
    All int32 on the GPU and read there: what a program writes into them counts from the next call on, replays of captured calls included."""

    def __init__(self, lens, tables, rows=None, max_rows=1, prefix=None, prefix_len=0):
        device = lens.device if isinstance(lens, torch.Tensor) else None
        _ints(lens, "lens", device)
        _ints(tables, "tables", device)
        _need(lens.dim() == 1 and (lens.stride(0) == 1 or lens.numel() < 2), "lens must be [seqs], its elements next to each other")
        _need(tables.dim() == 2 and tables.shape[0] == lens.shape[0] and (tables.stride(1) == 1 or tables.shape[1] < 2), f"tables must be [{lens.shape[0]}, pages], the pages of a sequence next to each other")
        if rows is not None:
            _ints(rows, "rows", device)
            _need(rows.dim() == 1 and rows.shape[0] == lens.shape[0] + 1 and (rows.stride(0) == 1 or rows.numel() < 2), f"rows must be [{lens.shape[0] + 1}], its elements next to each other")
        _need(int(max_rows) >= 1 and (rows is not None or int(max_rows) == 1), "max_rows must be positive, and 1 without rows")
        _need(prefix_len >= 0 and (prefix is not None or prefix_len == 0), "prefix_len without prefix")
        _need(max(*tables.shape, int(max_rows), int(prefix_len)) < 1 << 31, "seqs, pages of a sequence, max_rows or prefix_len beyond 2^31 - 1")
        if prefix is not None:
            _ints(prefix, "prefix", device)
            _need(prefix.dim() == 1 and (prefix.stride(0) == 1 or prefix.numel() < 2), "prefix must be [pages], its elements next to each other")
        self.lens, self.tables, self.rows, self.max_rows, self.prefix, self.prefix_len, self.device = lens, tables, rows, int(max_rows), prefix, int(prefix_len), device
        self.seqs = lens.shape[0]
        self._c = _Batch(lens.data_ptr(), 0 if rows is None else rows.data_ptr(), tables.data_ptr(), 0 if not self.prefix_len else prefix.data_ptr(), tables.stride(0), self.seqs,
                         tables.shape[1], self.max_rows, self.prefix_len)
        self._ref = C.byref(self._c)
        self._bytes = {}   # workspaces' sizes

    def _for(self, pages, n_rows):
        if not isinstance(pages, KVPages):
            raise LmrsError("pages must be KVPages")
        if self.device != pages.device:
            raise LmrsError(f"the batch lies on {self.device}, the pages on {pages.device}")
        if self.prefix_len and self.prefix.shape[0] * pages.page_size < self.prefix_len:
            raise LmrsError(f"prefix lists too few pages for {self.prefix_len} tokens")
        if self.rows is None and n_rows != self.seqs:
            raise LmrsError(f"{n_rows} rows for {self.seqs} sequences of one row each")


def rope_axes(x, pos, rope, out=None):
    """x [rows, heads, head_size] turned by pos [axes, rows] (or [rows] for one axis); out may be x, and not lie over a part of it."""
    if not isinstance(rope, RopeAxes):
        raise LmrsError("rope must be RopeAxes")
    if not isinstance(x, torch.Tensor) or x.dim() != 3 or x.dtype not in _DTYPES:
        raise LmrsError("x must be a [rows, heads, head_size] tensor of bfloat16, float16 or float32")
    n, heads, size = x.shape
    if heads > 65535:
        raise LmrsError(f"{heads} heads: at most 65535")
    device, dtype = x.device, x.dtype
    if x.is_cuda and device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return rope_axes(x, pos, rope, out)
    xr = _heads(x, "x", device, dtype, n, heads, size)
    p = _positions(pos, rope.axes, n, device)
    if out is None:
        out, o = _new(x)
    else:
        o = _heads(out, "out", device, dtype, n, heads, size, out=True)
    rc = lib().lmrs_b200_rope_axes(rope._ref, _DTYPES[dtype], _byref(xr), _byref(o), n, heads, size, _byref(p), _stream(device.index))
    if rc:
        check(rc)
    return out


def append(pages, batch, k, v, rope=None, pos=None, q=None, q_out=None):
    """Writes k and v [rows, kv_heads, head_size] to the places in the pages that the batch gives their rows, k turned by pos [axes, rows] (None: by its
    place, the prefix included, on every axis); rope None: k as it is.  Returns q [rows, heads, head_size] turned alike (q_out may be q), or None."""
    if not isinstance(batch, Batch):
        raise LmrsError("batch must be a Batch")
    if not isinstance(k, torch.Tensor) or k.dim() != 3:
        raise LmrsError("k must be a [rows, kv_heads, head_size] tensor")
    n = k.shape[0]
    batch._for(pages, n)
    device, dtype, size = pages.device, pages.dtype, pages.head_size
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return append(pages, batch, k, v, rope, pos, q, q_out)
    kr = _heads(k, "k", device, dtype, n, pages.kv_heads, size)
    vr = _heads(v, "v", device, dtype, n, pages.kv_heads, size)
    if rope is None:
        if pos is not None or q is not None or q_out is not None:
            raise LmrsError("pos and q go with rope")
    elif not isinstance(rope, RopeAxes):
        raise LmrsError("rope must be RopeAxes")
    p = None if pos is None else _byref(_positions(pos, rope.axes, n, device))
    qr = qo = None
    heads = 0
    if q is not None:
        if not isinstance(q, torch.Tensor) or q.dim() != 3:
            raise LmrsError("q must be a [rows, heads, head_size] tensor")
        heads = q.shape[1]
        if heads > 65535:
            raise LmrsError(f"{heads} heads: at most 65535")
        qr = _byref(_heads(q, "q", device, dtype, n, heads, size))
        if q_out is None:
            q_out, qo = _new(q)
        else:
            qo = _heads(q_out, "q_out", device, dtype, n, heads, size, out=True)
        qo = _byref(qo)
    elif q_out is not None:
        raise LmrsError("q_out without q")
    rc = lib().lmrs_b200_paged_append(pages._ref, batch._ref, n, _byref(kr), _byref(vr), None if rope is None else rope._ref, p, qr, qo, heads, _stream(device.index))
    if rc:
        check(rc)
    return q_out


def attention(pages, batch, q, out=None, scale=None, softcap=0.0, return_lse=False):
    """softmax(scale * q . keys) . values for q [rows, heads, head_size]: every row over the prefix and over its own sequence up to its own place.
    heads: a multiple of kv_heads, neighbours share one.  scale None: head_size ** -0.5.  softcap > 0: scores s become softcap * tanh(s / softcap).  A row
    that sees nothing is 0.  return_lse: also the logarithms of the sums of exponentials, float32 [rows, heads] (-inf for a row that sees nothing).
    out may not overlap q.  16-bit types: the softmax' weights are rounded to the type before the product with the values, their sum is not."""
    if not isinstance(batch, Batch):
        raise LmrsError("batch must be a Batch")
    if not isinstance(q, torch.Tensor) or q.dim() != 3:
        raise LmrsError("q must be a [rows, heads, head_size] tensor")
    n, heads, size = q.shape
    if heads > 65535:
        raise LmrsError(f"{heads} heads: at most 65535")
    batch._for(pages, n)
    device, dtype = pages.device, pages.dtype
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return attention(pages, batch, q, out, scale, softcap, return_lse)
    qr = _heads(q, "q", device, dtype, n, heads, pages.head_size)
    if out is None:
        out, o = _new(q)
    else:
        o = _heads(out, "out", device, dtype, n, heads, size, out=True)
    lse = torch.empty(n, heads, dtype=torch.float32, device=device) if return_lse else None
    L = lib()
    key = (n, heads, pages.kv_heads, size, pages.page_size, dtype)
    need = batch._bytes.get(key)
    if need is None:   # (it goes by the numbers of the call alone)
        got = C.c_size_t()
        check(L.lmrs_b200_paged_attention_workspace(pages._ref, batch._ref, n, heads, C.byref(got)))
        if len(batch._bytes) > 64:
            batch._bytes.clear()
        need = batch._bytes[key] = got.value
    work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    rc = L.lmrs_b200_paged_attention(pages._ref, batch._ref, n, _byref(qr), _byref(o), heads, size ** -0.5 if scale is None else scale, softcap,
                                     lse.data_ptr() if return_lse and n and heads else None, work.data_ptr() if need else None, need, _stream(device.index))
    if rc:
        check(rc)
    return (out, lse) if return_lse else out
