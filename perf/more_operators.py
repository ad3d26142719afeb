"""Operators around a cache that holds keys and values in 8 bits, as cases that can be timed and compared.

  norm    norms of queries and keys for each head and their rotary positions, in one pass
  append  keys and values of new tokens quantised into pages as they are written (keys, and the queries beside them, normed and turned on the way), and all that the sequences hold read back
  read    tokens of 8-bit pages read back as 16- or 32-bit rows
  attend  attention of every sequence's new tokens over its own 8-bit pages and over a prefix that all sequences share

run() computes them in plain torch (32 bits; 64 where angles are formed and where a value is rounded to 8 bits, since it may lie next to a border), or, with `own`, through lmrs_b200.paged.
exact() computes them again in 64 bits from the definition.

A cache is two arrays of codes [pages, page_size, kv_heads, head_size], int8 or float8_e4m3fn, and two of scales [pages, page_size / block, kv_heads], float32: a code stands for
code * scale, one scale for `block` tokens of a page and a head.  Tokens that a call appends to a block that it begins get the scale a / Q, a the largest size among them and Q the
format's largest number; where the block held tokens before, the larger of that and the old scale, to which the old codes are rounded again.  Scales stay within 2^-60 .. 2^60.
"""
import math
import os
import random
import sys
from fractions import Fraction

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
MOST = {"int8": 127.0, "e4m3": 448.0}
EPS = 1e-6
PI = Fraction(31415926535897932384626433832795028841971693993751, 10 ** 49)


def _paged():
    path = os.path.join(os.getcwd(), "lm.rs_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from lmrs_b200 import paged
    return paged


def listed():
    return [
        # one token of one chat: queries and keys of the 1B layer shape as they come out of one projection (nothing but latency)
        dict(name="norm_step", kind="norm", dtype="bfloat16", rows=1, heads=40, kv_heads=8, dim=64, rot=64, sections="32", order="blocks", layout="halves", theta=500000.0, far=8192),
        # queries and keys of an image prompt, positions in time, height and width
        dict(name="norm_image", kind="norm", dtype="bfloat16", rows=4099, heads=40, kv_heads=8, dim=128, rot=128, sections="16+24+24", order="blocks", layout="halves", theta=1000000.0,
             far=131072),
        # one token of one chat that becomes the 14th of its block
        dict(name="append_step", kind="append", dtype="bfloat16", form="int8", seqs=1, idle=0, rows=1, past=701, heads=32, kv_heads=8, dim=64, rot=64, page=16, block=16, norms=True,
             sections="32", order="blocks", layout="halves", theta=500000.0, far=0, mix=1),
        # one token of each of 64 chats, some places of the batch empty, positions counted apart from the cache, a scale for each token
        dict(name="append_batch", kind="append", dtype="float16", form="e4m3", seqs=64, idle=3, rows=1, past=300, heads=32, kv_heads=8, dim=128, rot=128, page=64, block=1, norms=False,
             sections="16+24+24", order="blocks", layout="halves", theta=1000000.0, far=100000, mix=2),
        # prompts of many chats in one call, that go on where others ended
        dict(name="append_prompts", kind="append", dtype="bfloat16", form="int8", seqs=24, idle=0, rows=700, past=300, heads=32, kv_heads=8, dim=128, rot=64, page=32, block=16, norms=True,
             sections="32", order="blocks", layout="pairs", theta=10000.0, far=0, mix=3),
        # a few short chats taken out of the cache in full precision
        dict(name="read_chats", kind="read", dtype="float32", form="int8", seqs=9, idle=1, past=500, kv_heads=8, dim=64, page=16, block=8, mix=4),
        # long sessions taken out of the cache
        dict(name="read_sessions", kind="read", dtype="bfloat16", form="e4m3", seqs=6, idle=0, past=20000, kv_heads=8, dim=128, page=64, block=64, mix=5),
        # one token of one chat
        dict(name="attend_step", kind="attend", dtype="bfloat16", form="int8", seqs=1, idle=0, rows=1, past=1000, prefix=0, heads=32, kv_heads=8, dim=64, page=16, block=16, cap=0.0, mix=6),
        # one token of each of 61 chats that begin with the same instructions
        dict(name="attend_shared", kind="attend", dtype="bfloat16", form="e4m3", seqs=64, idle=3, rows=1, past=1000, prefix=8200, heads=32, kv_heads=8, dim=128, page=64, block=32, cap=0.0,
             mix=7),
        # four long chats with nothing in common: the cache is read once, and that is all there is to it
        dict(name="attend_long", kind="attend", dtype="float16", form="int8", seqs=4, idle=0, rows=1, past=100000, prefix=0, heads=32, kv_heads=8, dim=128, page=32, block=1, cap=0.0, mix=8),
        # portions of prompts that follow the same instructions, scores held down
        dict(name="attend_prompts", kind="attend", dtype="bfloat16", form="e4m3", seqs=12, idle=0, rows=200, past=900, prefix=2050, heads=16, kv_heads=8, dim=256, page=32, block=16, cap=50.0,
             mix=9),
        # full precision beside the cache
        dict(name="attend_float32", kind="attend", dtype="float32", form="int8", seqs=16, idle=1, rows=1, past=900, prefix=4096, heads=32, kv_heads=8, dim=64, page=16, block=4, cap=0.0,
             mix=10),
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    """a case of the same ranges, no dearer than the dearest of the list"""
    top = [work(c) for c in listed()]
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= max(t["bytes"] for t in top) and w["flops"] <= max(t["flops"] for t in top):
            return case


def _draw_rope(rng, dim):
    rot = rng.choice((dim, dim // 2))
    axes, pairs = rng.choice((1, 1, 2, 3)), rot // 2
    cuts = sorted(rng.sample(range(1, pairs), axes - 1))
    parts = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
    return dict(rot=rot, sections="+".join(map(str, parts)), order=rng.choice(("blocks", "cycle")), layout=rng.choice(("halves", "pairs")), theta=rng.choice((10000.0, 500000.0, 1000000.0)))


def _draw(rng):
    kind = rng.choice(("norm", "append", "append", "read", "attend", "attend", "attend"))
    dtype, form = rng.choice(("bfloat16", "bfloat16", "float16", "float32")), rng.choice(("int8", "e4m3"))
    dim = rng.choice((64, 64, 96, 128, 128, 256))
    kv_heads, group = rng.choice((1, 2, 4, 5, 8)), rng.choice((1, 2, 3, 4, 6, 8))
    if kind == "norm":
        return dict(kind=kind, dtype=dtype, rows=_log(rng, 1, 3000), heads=kv_heads * (group + 1), kv_heads=kv_heads, dim=dim, far=_log(rng, 64, 1000000), **_draw_rope(rng, dim))
    page = rng.choice((1, 8, 16, 16, 32, 48, 64, 128))
    block = rng.choice([b for b in (1, 2, 4, 8, 12, 16, 24, 32, 64, 128) if page % b == 0])
    mix = rng.randrange(1 << 30)
    many = rng.random() < 0.35   # prompts rather than single tokens
    base = dict(kind=kind, dtype=dtype, form=form, kv_heads=kv_heads, dim=dim, page=page, block=block, mix=mix)
    if kind == "read":
        seqs = _log(rng, 1, 64)
        return dict(base, seqs=seqs, idle=rng.choice((0, seqs // 8)), past=_log(rng, 1, 8000))
    base["heads"] = kv_heads * group
    if kind == "append":
        seqs, rows = (_log(rng, 1, 16), _log(rng, 2, 400)) if many else (_log(rng, 1, 128), 1)
        return dict(base, seqs=seqs, idle=rng.choice((0, 0, seqs // 8)), rows=rows, past=_log(rng, 1, 500), far=rng.choice((0, 100000)), norms=rng.choice((True, False)), **_draw_rope(rng, dim))
    prefix = 0 if rng.random() < 0.25 else _log(rng, 30, 16000)
    if many:
        seqs, rows, past = _log(rng, 1, 8), _log(rng, 2, 160), _log(rng, 1, 1200)
        prefix = min(prefix, 4000)
    else:
        seqs, rows, past = _log(rng, 1, 100), 1, _log(rng, 1, 6000)
    return dict(base, seqs=seqs, idle=rng.choice((0, 0, seqs // 8)), rows=rows, past=past, prefix=prefix, cap=rng.choice((0.0, 0.0, 30.0)))


def _shape(case):
    """tokens of this call and tokens held, of every sequence: from the case, not from the seed"""
    rng = random.Random(case["mix"])
    counts, lens, rows = [], [], case.get("rows", 0)
    for b in range(case["seqs"]):
        n = rows if b == 0 else rng.randint(max(1, rows // 3), rows) if rows else 0
        past = case["past"] if b == 0 else rng.randint(case["past"] // 4, case["past"])
        counts.append(n)
        lens.append(past + n)
    for b in rng.sample(range(case["seqs"]), case["idle"]):
        counts[b], lens[b] = min(1, rows), 0
    return counts, lens


def _axes(case):
    """the axis of every pair"""
    left = [int(s) for s in case["sections"].split("+")]
    if case["order"] == "blocks":
        return [a for a, n in enumerate(left) for _ in range(n)]
    out = []
    while any(left):   # turn by turn, as long as an axis has pairs left
        for a, n in enumerate(left):
            if n:
                out.append(a)
                left[a] -= 1
    return out


def _freq(case):
    return [case["theta"] ** (-2.0 * j / case["rot"]) for j in range(case["rot"] // 2)]


def _turns(freq):
    """freq / 2 pi modulo a turn, in 2^-64 turns, as signed numbers of 64 bits: products with positions wrap to what is left of them modulo a turn"""
    t = [round(Fraction(f) / (2 * PI) * 2 ** 64) % 2 ** 64 for f in freq]
    return [x - 2 ** 64 if x >= 2 ** 63 else x for x in t]


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=gen, device=DEV).mul_(scale).to(dt)

    def heads(n, count, dim):   # rows as a projection leaves them: some heads and some columns larger than others
        x = torch.randn((n, count, dim), generator=gen, device=DEV)
        x *= torch.exp(0.5 * torch.randn((1, count, dim), generator=gen, device=DEV))
        return x.to(dt)

    def weight(count):
        return 1.0 + 0.2 * torch.randn((count, case["dim"]) if count else (case["dim"],), generator=gen, device=DEV)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    def positions(n):
        """[axes, n]: a walk through rows and columns of images that lie somewhere before `far`"""
        start = torch.randint(0, case["far"], (1,), generator=gen, device=DEV)
        pos = torch.randint(0, max(2, min(case["far"], 200)), (len(case["sections"].split("+")), n), generator=gen, device=DEV) + start
        return pos.to(torch.int32)

    st, kind, dim = dict(case=case), case["kind"], case["dim"]
    if kind in ("norm", "append"):
        st["turns"] = torch.tensor(_turns(_freq(case)), dtype=torch.int64, device=DEV)
        st["axis"] = torch.tensor(_axes(case), dtype=torch.int64, device=DEV)
    if kind == "norm":   # queries and keys lie in the rows of one projection, values behind them
        st["x"] = heads(case["rows"], case["heads"] + case["kv_heads"], dim)[:, :case["heads"]]
        st["weight"] = weight(case["heads"])
        st["pos"] = positions(case["rows"])
    else:
        form = CODES[case["form"]]
        counts, lens = _shape(case)
        n, page, kv, block = sum(counts), case["page"], case["kv_heads"], case["block"]
        held, prefix = [-(-x // page) for x in lens], case.get("prefix", 0)
        shared = -(-prefix // page)
        pages = sum(held) + shared + 2
        order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
        tables = torch.full((case["seqs"], max(1, max(held))), -1, dtype=torch.int32, device=DEV)
        at = shared
        for b, h in enumerate(held):
            tables[b, :h] = order[at:at + h]
            at += h

        def codes():   # a block's largest is some 2.5 to 4 of the others' root mean square
            x = torch.randn((pages, page, kv, dim), generator=gen, device=DEV)
            return (x * 40).round_().clamp_(-127, 127).to(form) if case["form"] == "int8" else (x * 120).clamp_(-448, 448).to(form)

        def scales():
            x = torch.rand((pages, page // block, kv), generator=gen, device=DEV)
            return (0.5 + x) / (40 if case["form"] == "int8" else 120)

        starts = [sum(counts[:b]) for b in range(case["seqs"] + 1)]
        st.update(tables=tables, shared=order[:shared].contiguous(), prefix=prefix, lens=ints(lens), rows=ints(starts) if case.get("rows", 1) > 1 else None,
                  k_pages=codes(), v_pages=codes(), k_scale=scales(), v_scale=scales())
        # the sequence of every row and its index there, which a program that forms batches knows; and the same for all that the sequences hold
        index, size = torch.tensor([x - c for c, x in zip(counts, lens)], device=DEV), torch.tensor(counts, device=DEV)
        all_size = st["lens"].long()
        st["seq"] = torch.repeat_interleave(size)
        st["index"] = torch.arange(n, device=DEV) + (index - size.cumsum(0) + size)[st["seq"]]
        st["all_seq"] = torch.repeat_interleave(all_size)
        st["all_index"] = torch.arange(sum(lens), device=DEV) - (all_size.cumsum(0) - all_size)[st["all_seq"]]
        st["all_rows"] = ints([sum(lens[:b]) for b in range(case["seqs"] + 1)])
        st["held"], st["counts"], st["starts"] = lens, counts, starts
        if kind == "append":
            st["real"] = torch.nonzero(st["index"] >= 0)[:, 0]
            st["q"], st["k"], st["v"] = heads(n, case["heads"], dim), heads(n, kv, dim), heads(n, kv, dim)
            st["pos"] = positions(n) if case["far"] else None
            st["q_norm"], st["k_norm"] = (weight(0), weight(0)) if case["norms"] else (None, None)
        if kind == "attend":
            st["q"] = normal(n, case["heads"], dim, scale=1.5)
            st["slot"] = st["seq"] * case["rows"] + torch.arange(n, device=DEV) - (size.cumsum(0) - size)[st["seq"]]   # rows in a batch of equal lengths
    if own:
        paged = _paged()
        if kind in ("norm", "append"):
            st["rope"] = paged.RopeAxes(_freq(case), _axes(case), layout=case["layout"])
        if kind != "norm":
            st["pages"] = paged.QuantPages(st["k_pages"], st["v_pages"], st["k_scale"], st["v_scale"])
        if kind in ("append", "attend"):
            st["batch"] = paged.Batch(st["lens"], tables, rows=st["rows"], max_rows=case["rows"], prefix=st["shared"] if prefix else None, prefix_len=prefix)
        if kind in ("append", "read"):
            st["all"] = paged.Batch(st["lens"], tables, rows=st["all_rows"], max_rows=max(1, max(lens)))
    return st


# ---- plain forms ---------------------------------------------------------------------------------------------------------------------------
def _normed(x, weight):
    return x if weight is None else x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.to(x.dtype)


def _turned(st, x, pos):
    """x [n, heads, dim] (32 or 64 bits) turned by pos [axes, n]"""
    half = st["turns"].numel()
    angle = (pos.to(torch.int64).T[:, st["axis"]] * st["turns"]).to(torch.float64) * (math.pi / 2 ** 63)
    c, s = torch.cos(angle).to(x.dtype)[:, None], torch.sin(angle).to(x.dtype)[:, None]
    out = x.clone()
    if st["case"]["layout"] == "halves":
        a, b = x[..., :half], x[..., half:2 * half]
        out[..., :half], out[..., half:2 * half] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = a * c - b * s, b * c + a * s
    return out


def _rounded(x, form):
    """x (64 bits, within the format's range) to the format's nearest numbers, ties to even"""
    if form == "int8":
        return torch.round(x)
    step = torch.ldexp(torch.ones_like(x), torch.frexp(x).exponent.clamp(min=-5) - 4)   # (x = m 2^e with m from 1/2 on: three bits behind the first)
    return torch.round(x / step) * step


def _write(case, pages, scale, x, page, place, fresh_rows):
    """x [n, kv_heads, dim] (64 bits) into the codes and scales of one of the cache's two arrays"""
    block, form, G = case["block"], case["form"], case["kv_heads"]
    blocks = scale.shape[1]
    at = page * blocks + place // block
    flat = scale.view(-1, G)
    a = torch.zeros(flat.shape, dtype=torch.float64, device=DEV).scatter_reduce(0, at[:, None].expand(-1, G), x.abs().amax(-1), "amax")
    touched = torch.zeros(flat.shape[0], dtype=torch.bool, device=DEV)
    fresh = touched.clone()
    touched[at] = True
    fresh[at[fresh_rows]] = True
    mine = (a / MOST[form]).clamp(2.0 ** -60, 2.0 ** 60).float()
    now = torch.where(touched[:, None], torch.where(fresh[:, None], mine, torch.maximum(mine, flat)), flat)
    old = torch.nonzero(touched & ~fresh)[:, 0]
    by_block, by_token = pages.view(-1, block, G, case["dim"]), pages.view(-1, G, case["dim"])
    again = by_block[old].to(torch.float64) * flat[old][:, None, :, None].double() / now[old][:, None, :, None].double()
    by_block[old] = _rounded(again, form).float().to(pages.dtype)   # (float32 holds both formats' numbers)
    code = (x / now[at][..., None].double()).clamp(-MOST[form], MOST[form])
    by_token[page * case["page"] + place] = _rounded(code, form).float().to(pages.dtype)
    scale.copy_(now.view_as(scale))


def _values(st, codes, scale, seq, index):
    """the values [n, kv_heads, dim], 32 bits, of these tokens"""
    case = st["case"]
    page, place = st["tables"][seq, index // case["page"]].long(), index % case["page"]
    return codes[page, place].float() * scale[page, place // case["block"]][..., None]


def _append(st):
    case = st["case"]
    seq, index, real = st["seq"], st["index"], st["real"]
    pos = st["pos"] if st["pos"] is not None else index.expand(len(case["sections"].split("+")), -1)
    q = _turned(st, _normed(st["q"].float(), st["q_norm"]), pos).to(st["q"].dtype)
    k, v = _turned(st, _normed(st["k"].double(), st["k_norm"]), pos)[real], st["v"].double()[real]   # rows of empty places go nowhere
    at = index[real]
    page, fresh = st["tables"][seq[real], at // case["page"]].long(), at % case["block"] == 0
    _write(case, st["k_pages"], st["k_scale"], k, page, at % case["page"], fresh)
    _write(case, st["v_pages"], st["v_scale"], v, page, at % case["page"], fresh)
    return (q,) + _read(st) + (st["k_scale"], st["v_scale"])


def _read(st):
    dt = TYPES[st["case"]["dtype"]]
    return tuple(_values(st, st[c], st[s], st["all_seq"], st["all_index"]).to(dt) for c, s in (("k_pages", "k_scale"), ("v_pages", "v_scale")))


def _scores(q, k, scale, cap):
    s = torch.matmul(q, k.transpose(-1, -2)) * scale
    return cap * torch.tanh(s / cap) if cap else s


def _attend(st):
    case = st["case"]
    B, R, H, G, D, P = case["seqs"], case["rows"], case["heads"], case["kv_heads"], case["dim"], st["prefix"]
    scale, cap, page, block = D ** -0.5, case["cap"], case["page"], case["block"]
    # everything in the batch of equal lengths [sequence, KV head, row x grouped head, .]
    q = torch.zeros(B * R, H, D, dtype=torch.float32, device=DEV)
    q[st["slot"]] = st["q"].float()
    q = q.view(B, R, G, H // G, D).permute(0, 2, 1, 3, 4).reshape(B, G, R * (H // G), D)
    keys = st["tables"].shape[1] * page
    table = st["tables"].clamp(min=0).long()
    place = torch.arange(page, device=DEV) // block
    k = (st["k_pages"][table].float() * st["k_scale"][table][:, :, place, :, None]).view(B, keys, G, D).permute(0, 2, 1, 3)
    v = (st["v_pages"][table].float() * st["v_scale"][table][:, :, place, :, None]).view(B, keys, G, D).permute(0, 2, 1, 3)
    index = torch.full((B * R,), -1, dtype=torch.int64, device=DEV)
    index[st["slot"]] = st["index"]
    index = index.view(B, 1, R, 1).expand(B, 1, R, H // G).reshape(B, 1, R * (H // G), 1)
    seen = torch.arange(keys, device=DEV).view(1, 1, 1, keys) <= index
    s = _scores(q, k, scale, cap).masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    if P:
        shared = st["shared"].long()
        pk = (st["k_pages"][shared].float() * st["k_scale"][shared][:, place, :, None]).view(-1, G, D)[:P].permute(1, 0, 2)
        pv = (st["v_pages"][shared].float() * st["v_scale"][shared][:, place, :, None]).view(-1, G, D)[:P].permute(1, 0, 2)
        qp = q.permute(1, 0, 2, 3).reshape(G, -1, D)
        sp = _scores(qp, pk, scale, cap).view(G, B, -1, P)
        sp = sp.masked_fill((index < 0).permute(1, 0, 2, 3), -math.inf)
        top = torch.maximum(top, sp.amax(-1, keepdim=True).permute(1, 0, 2, 3))
    base = torch.where(top == -math.inf, torch.zeros_like(top), top)
    w = torch.exp(s - base)
    total, out = w.sum(-1, keepdim=True), torch.matmul(w, v)
    if P:
        w = torch.exp(sp - base.permute(1, 0, 2, 3))
        total = total + w.sum(-1, keepdim=True).permute(1, 0, 2, 3)
        out = out + torch.matmul(w.reshape(G, -1, P), pv).view(G, B, -1, D).permute(1, 0, 2, 3)
    out = torch.where(total == 0, torch.zeros_like(out), out / total)
    lse = (torch.log(total) + base)[..., 0]
    out = out.view(B, G, R, H // G, D).permute(0, 2, 1, 3, 4).reshape(B * R, H, D)[st["slot"]]
    lse = lse.view(B, G, R, H // G).permute(0, 2, 1, 3).reshape(B * R, H)[st["slot"]]
    return out.to(st["q"].dtype), lse


def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        paged = _paged()
        if kind == "norm":
            return paged.norm_rope(st["x"], st["weight"], pos=st["pos"], rope=st["rope"], eps=EPS)
        if kind == "append":
            q = paged.append(st["pages"], st["batch"], st["k"], st["v"], rope=st["rope"], pos=st["pos"], q=st["q"], k_norm=st["k_norm"], q_norm=st["q_norm"], eps=EPS)
        if kind in ("append", "read"):
            k, v = paged.read(st["pages"], st["all"], rows=st["all_index"].shape[0], dtype=TYPES[case["dtype"]])
            return (q, k, v, st["k_scale"], st["v_scale"]) if kind == "append" else (k, v)
        return paged.attention(st["pages"], st["batch"], st["q"], scale=case["dim"] ** -0.5, softcap=case["cap"], return_lse=True)
    if kind == "norm":
        return _turned(st, _normed(st["x"].float(), st["weight"]), st["pos"]).to(st["x"].dtype)
    return _append(st) if kind == "append" else _read(st) if kind == "read" else _attend(st)


def work(case):
    size, D, kind = TYPES[case["dtype"]].itemsize, case["dim"], case["kind"]
    if kind == "norm":
        n = case["rows"] * case["heads"]
        return {"bytes": 2 * n * D * size + 4 * case["heads"] * D + 4 * len(case["sections"].split("+")) * case["rows"], "flops": n * (4 * D + 3 * case["rot"])}
    counts, lens = _shape(case)
    n, H, G = sum(counts), case.get("heads", 0), case["kv_heads"]
    blocks = sum(-(-x // case["block"]) for x in lens) + -(-case.get("prefix", 0) // case["block"])
    tables = 4 * (sum(-(-x // case["page"]) for x in lens) + -(-case.get("prefix", 0) // case["page"]))
    held = sum(lens) + case.get("prefix", 0)
    cache = 2 * held * G * D + 8 * blocks * G + tables
    if kind == "read":
        return {"bytes": cache + 2 * held * G * D * size, "flops": 2 * held * G * D}
    if kind == "append":   # new rows in, queries and codes out; then all codes in and their values out
        axes = len(case["sections"].split("+")) if case["far"] else 0
        return {"bytes": n * (2 * H + 2 * G) * D * size + 2 * n * G * D + 4 * axes * n + cache + 2 * held * G * D * size,
                "flops": n * (H + G) * (3 * case["rot"] + (4 * D if case["norms"] else 0)) + 4 * n * G * D + 2 * held * G * D}
    pairs = sum(c * (case["prefix"] + x - c) + c * (c + 1) // 2 for c, x in zip(counts, lens) if x)
    return {"bytes": 2 * n * H * D * size + 4 * n * H + cache, "flops": 4 * D * H * pairs}


# ---- the same from the definitions, in 64 bits -------------------------------------------------------------------------------------------
def _exact_angles(pos, freq):
    """pos * freq modulo 2 pi: the product in two parts, the first one exact, whole turns taken off in three parts of 2 pi"""
    parts, left = [], 2 * PI
    for bits in (28, 58):
        parts.append(float(Fraction(math.floor(left * 2 ** bits), 2 ** bits)))
        left -= Fraction(parts[-1])
    parts.append(float(left))
    high = math.ldexp(math.floor(math.ldexp(freq, 26)), -26)   # (positions have up to 21 bits, frequencies are 1 at most)
    a, b = pos.double() * high, pos.double() * (freq - high)
    turns = torch.round(a / parts[0])
    return (a - turns * parts[0]) - turns * parts[1] - turns * parts[2] + b


def _exact_turn(case, x, pos):
    """pair by pair of columns: (a, b) is a + ib, multiplied by e^(i angle)"""
    out, half = x.clone(), case["rot"] // 2
    for j, a in enumerate(_axes(case)):
        first, second = (j, j + half) if case["layout"] == "halves" else (2 * j, 2 * j + 1)
        angle = _exact_angles(pos[a], _freq(case)[j])
        z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.ones_like(angle), angle)[:, None]
        out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_norm(x, weight):
    x = x.double()
    if weight is None:
        return x
    return x * weight.double() * torch.rsqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / x.shape[-1] + EPS)


def _exact_numbers(form):
    """the format's numbers, rising, and whether each has an even code"""
    if form == "int8":
        return torch.arange(-127, 128, dtype=torch.float64, device=DEV), torch.arange(-127, 128, device=DEV) % 2 == 0
    up = [m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1]
    return torch.tensor([-x for x in up[:0:-1]] + up, dtype=torch.float64, device=DEV), torch.tensor([i % 2 == 0 for i in range(len(up) - 1, 0, -1)] + [i % 2 == 0 for i in range(len(up))], device=DEV)


def _exact_round(x, form):
    """the nearest of the format's numbers, of two as near the one with an even code"""
    numbers, even = _exact_numbers(form)
    above = torch.searchsorted(numbers, x.contiguous()).clamp(1, numbers.numel() - 1)
    below = above - 1
    up, down = numbers[above] - x, x - numbers[below]
    return torch.where((up < down) | ((up == down) & even[above]), numbers[above], numbers[below])


def _exact_write(case, codes, scale, x, have, first):
    """codes [held, G, D] (values of a sequence's codes, 64 bits) and scale [held, G] (of every token) with its last tokens x; first: index of the first of them"""
    block, form = case["block"], case["form"]
    i0 = first // block * block   # (the block that held tokens before, by itself)
    pieces = ([(i0, first, min(have, i0 + block))] if first > i0 else []) + [(i, i, min(have, i + block)) for i in range(-(-first // block) * block, have, block)]
    for start, new, end in pieces:
        a = x[new - first:end - first].abs().amax((0, 2))
        s = (a / MOST[form]).clamp(2.0 ** -60, 2.0 ** 60).float().double()
        if new > start:
            s = torch.maximum(s, scale[start])
            codes[start:new] = _exact_round(codes[start:new] * scale[start][None, :, None] / s[None, :, None], form)
        codes[new:end] = _exact_round(x[new - first:end - first] / s[None, :, None], form)
        scale[start:end] = s


def exact(case, seed):
    st = prepare(case, seed)
    kind, D = case["kind"], case["dim"]
    if kind == "norm":
        return _exact_turn(case, _exact_norm(st["x"], st["weight"]), st["pos"])
    page, block, G = case["page"], case["block"], case["kv_heads"]
    tables = st["tables"].cpu()

    def held(b, name):   # codes and scales of what sequence b holds
        i = torch.arange(st["held"][b])
        p, at = tables[b, i // page].long().to(DEV), (i % page).to(DEV)
        return st[name + "_pages"][p, at].double(), st[name + "_scale"][p, at // block].double()

    if kind in ("append", "read"):
        dt = torch.float64
        got = {"k": [torch.zeros(0, G, D, dtype=dt, device=DEV)], "v": [torch.zeros(0, G, D, dtype=dt, device=DEV)]}
        new, scales = {}, {}
        if kind == "append":
            n_axes = len(case["sections"].split("+"))
            pos = torch.stack([st["index"]] * n_axes) if st["pos"] is None else st["pos"]
            new = {"k": _exact_turn(case, _exact_norm(st["k"], st["k_norm"]), pos), "v": st["v"].double()}
        for name in ("k", "v"):
            if kind == "append":
                scales[name] = st[name + "_scale"].double()
            for b, (first, c) in enumerate(zip(st["starts"], st["counts"])):
                have = st["held"][b]
                if not have:
                    continue
                codes, s = held(b, name)
                if kind == "append":
                    _exact_write(case, codes, s, new[name][first:first + c], have, have - c)
                    i = torch.arange(0, have, block)
                    scales[name][tables[b, i // page].long().to(DEV), (i % page // block).to(DEV)] = s[::block]
                got[name].append(codes * s[..., None])
        k, v = torch.cat(got["k"]), torch.cat(got["v"])
        return (k, v) if kind == "read" else (_exact_turn(case, _exact_norm(st["q"], st["q_norm"]), pos), k, v, scales["k"], scales["v"])
    H, cap = case["heads"], case["cap"]
    n = st["q"].shape[0]
    out = torch.zeros(n, H, D, dtype=torch.float64, device=DEV)
    lse = torch.full((n, H), -math.inf, dtype=torch.float64, device=DEV)
    i = torch.arange(st["prefix"], device=DEV)
    front = [(st[x + "_pages"][st["shared"].long()[i // page], i % page], st[x + "_scale"][st["shared"].long()[i // page], i % page // block]) for x in ("k", "v")]
    front = [c.double() * s.double()[..., None] for c, s in front]
    for b, (first, c) in enumerate(zip(st["starts"], st["counts"])):
        have = st["held"][b]
        if not have:
            continue
        k, v = (torch.cat([f, x * s[..., None]]) for f, (x, s) in zip(front, (held(b, "k"), held(b, "v"))))
        last = st["prefix"] + have - c + torch.arange(c, device=DEV)
        hidden = torch.arange(k.shape[0], device=DEV) > last[:, None, None]
        for g in range(G):
            heads = slice(g * (H // G), (g + 1) * (H // G))
            s = torch.einsum("rhd,kd->rhk", st["q"][first:first + c, heads].double(), k[:, g]) / math.sqrt(D)
            if cap:
                s = cap * torch.tanh(s / cap)
            s = s.masked_fill(hidden, -math.inf)
            out[first:first + c, heads] = torch.softmax(s, -1) @ v[:, g]
            lse[first:first + c, heads] = torch.logsumexp(s, -1)
    return out, lse
