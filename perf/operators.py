"""Operators of serving many sequences at once, as cases that can be timed and compared.

  rope     rotary positions with several axes: rows of heads turned by the angles of their (time, height, width) positions
  append   keys and values of new tokens into a cache of pages, keys (and the queries beside them) turned on the way
  attend   attention of every sequence's new tokens over its own pages and over a prefix that all sequences share

run() computes them in plain torch (32 bits, 64 where angles are formed), or, with `own`, through lmrs_b200.paged.
exact() computes them again in 64 bits from the definition.

A cache is two arrays [pages, page_size, kv_heads, head_size].  Sequence b holds lens[b] tokens in the pages that its row of `tables` lists, the
tokens of the call included, which are the last of them; a sequence with no tokens is a place of the batch that stands empty, and its row comes out as 0.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def _paged():
    path = os.path.join(os.getcwd(), "lm.rs_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from lmrs_b200 import paged
    return paged


def listed():
    return [
        # one token of one chat: queries and keys of the 1B layer shape, one axis (nothing but latency)
        dict(name="rope_step", kind="rope", dtype="bfloat16", rows=1, heads=40, dim=64, rot=64, sections="32", order="blocks", layout="halves", theta=500000.0, far=8192),
        # the queries of an image prompt: positions in time, height and width, one block of the pairs for each
        dict(name="rope_image", kind="rope", dtype="bfloat16", rows=4099, heads=32, dim=128, rot=128, sections="16+24+24", order="blocks", layout="halves", theta=1000000.0, far=131072),
        # patch rows of a vision tower (577 for each of four crops), height and width turn by turn, full precision
        dict(name="rope_patches", kind="rope", dtype="float32", rows=2308, heads=16, dim=64, rot=64, sections="16+16", order="cycle", layout="pairs", theta=10000.0, far=64),
        # one token of one chat
        dict(name="append_step", kind="append", dtype="bfloat16", seqs=1, idle=0, rows=1, past=700, heads=32, kv_heads=8, dim=64, rot=64, page=16,
             sections="32", order="blocks", layout="halves", theta=500000.0, far=0, mix=1),
        # one token of each of 64 chats, some places of the batch empty, positions counted apart from the cache
        dict(name="append_batch", kind="append", dtype="float16", seqs=64, idle=3, rows=1, past=1500, heads=32, kv_heads=8, dim=128, rot=128, page=64,
             sections="16+24+24", order="blocks", layout="halves", theta=1000000.0, far=100000, mix=2),
        # prompts of many chats in one call
        dict(name="append_prompts", kind="append", dtype="bfloat16", seqs=24, idle=0, rows=700, past=300, heads=32, kv_heads=8, dim=128, rot=64, page=16,
             sections="32", order="blocks", layout="pairs", theta=10000.0, far=0, mix=3),
        # one token of one chat, everything in its own pages
        dict(name="attend_step", kind="attend", dtype="bfloat16", seqs=1, idle=0, rows=1, past=1000, prefix=0, heads=32, kv_heads=8, dim=64, page=16, cap=0.0, mix=4),
        # one token of each of 61 chats that begin with the same instructions
        dict(name="attend_shared", kind="attend", dtype="bfloat16", seqs=64, idle=3, rows=1, past=1000, prefix=8200, heads=32, kv_heads=8, dim=64, page=64, cap=0.0, mix=5),
        # the same with a whole document in front, wide heads
        dict(name="attend_document", kind="attend", dtype="bfloat16", seqs=128, idle=0, rows=1, past=600, prefix=32768, heads=32, kv_heads=8, dim=128, page=16, cap=0.0, mix=6),
        # four long chats with nothing in common: the cache is read once, and that is all there is to it
        dict(name="attend_long", kind="attend", dtype="float16", seqs=4, idle=0, rows=1, past=60000, prefix=0, heads=32, kv_heads=8, dim=128, page=32, cap=0.0, mix=7),
        # portions of prompts that follow the same instructions, scores held down
        dict(name="attend_prompts", kind="attend", dtype="bfloat16", seqs=12, idle=0, rows=200, past=900, prefix=2050, heads=16, kv_heads=8, dim=256, page=32, cap=50.0, mix=8),
        # full precision
        dict(name="attend_float32", kind="attend", dtype="float32", seqs=16, idle=1, rows=1, past=500, prefix=4096, heads=32, kv_heads=8, dim=64, page=16, cap=0.0, mix=9),
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _draw_rope(rng, dim, rot):
    axes, pairs = rng.choice((1, 2, 3, 3)), rot // 2
    cuts = sorted(rng.sample(range(1, pairs), axes - 1))
    parts = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
    order = rng.choice(("blocks", "cycle"))
    return dict(rot=rot, sections="+".join(map(str, parts)), order=order, layout=rng.choice(("halves", "pairs")), theta=rng.choice((10000.0, 500000.0, 1000000.0)))


def draw(rng):
    """a case of the same ranges, no dearer than the dearest of the list"""
    top = [work(c) for c in listed()]
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= max(t["bytes"] for t in top) and w["flops"] <= max(t["flops"] for t in top):
            return case


def _draw(rng):
    kind = rng.choice(("rope", "append", "attend", "attend"))
    dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
    dim = rng.choice((64, 64, 96, 128, 128, 256))
    if kind == "rope":
        return dict(kind=kind, dtype=dtype, rows=_log(rng, 1, 2000), heads=_log(rng, 1, 40), dim=dim, far=_log(rng, 64, 1000000),
                    **_draw_rope(rng, dim, rng.choice((dim, dim // 2))))
    kv_heads, group = rng.choice((1, 2, 4, 5, 8)), rng.choice((1, 2, 3, 4, 6, 8))
    page = rng.choice((1, 8, 16, 16, 32, 48, 64, 128))
    many = rng.random() < 0.35   # prompts rather than single tokens
    mix = rng.randrange(1 << 30)
    if kind == "append":
        seqs, rows = (_log(rng, 1, 16), _log(rng, 2, 200)) if many else (_log(rng, 1, 128), 1)
        return dict(kind=kind, dtype=dtype, seqs=seqs, idle=rng.choice((0, 0, seqs // 8)), rows=rows, past=_log(rng, 1, 1200), heads=kv_heads * group,
                    kv_heads=kv_heads, dim=dim, page=page, far=rng.choice((0, 100000)), mix=mix, **_draw_rope(rng, dim, rng.choice((dim, dim // 2))))
    prefix = 0 if rng.random() < 0.25 else _log(rng, 30, 16000)
    if many:
        seqs, rows, past = _log(rng, 1, 8), _log(rng, 2, 160), _log(rng, 1, 1200)
        prefix = min(prefix, 4000)
    elif dtype == "float32":
        seqs, rows, past = _log(rng, 1, 32), 1, _log(rng, 1, 4000)
    else:
        seqs, rows, past = _log(rng, 1, 100), 1, _log(rng, 1, 4000)
    return dict(kind=kind, dtype=dtype, seqs=seqs, idle=rng.choice((0, 0, seqs // 8)), rows=rows, past=past, prefix=prefix, heads=kv_heads * group, kv_heads=kv_heads,
                dim=dim, page=page, cap=rng.choice((0.0, 0.0, 30.0)), mix=mix)


def _shape(case):
    """tokens of this call and tokens held, of every sequence: from the case, not from the seed"""
    rng = random.Random(case["mix"])
    counts, lens = [], []
    for b in range(case["seqs"]):
        n = case["rows"] if b == 0 else rng.randint(max(1, case["rows"] // 3), case["rows"])
        past = case["past"] if b == 0 else rng.randint(case["past"] // 4, case["past"])
        counts.append(n)
        lens.append(past + n)
    for b in rng.sample(range(case["seqs"]), case["idle"]):
        counts[b], lens[b] = 1, 0
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


def _positions(case, n, gen):
    """[axes, n]: a walk through rows and columns of images that lie somewhere before `far`"""
    axes = len(case["sections"].split("+"))
    start = torch.randint(0, case["far"], (1,), generator=gen, device=DEV)
    pos = torch.randint(0, max(2, min(case["far"], 200)), (axes, n), generator=gen, device=DEV) + start
    return pos.to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=gen, device=DEV).mul_(scale).to(dt)

    st = dict(case=case)
    if case["kind"] == "rope":
        st["x"] = normal(case["rows"], case["heads"], case["dim"])
        st["pos"] = _positions(case, case["rows"], gen)
    else:
        counts, lens = _shape(case)
        n, page, kv, dim = sum(counts), case["page"], case["kv_heads"], case["dim"]
        held, prefix = [-(-x // page) for x in lens], case.get("prefix", 0)
        shared = -(-prefix // page)
        pages = sum(held) + shared + 2
        order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
        tables = torch.full((case["seqs"], max(1, max(held))), -1, dtype=torch.int32, device=DEV)
        at = shared
        for b, h in enumerate(held):
            tables[b, :h] = order[at:at + h]
            at += h
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        st.update(counts=counts, held=lens, tables=tables, shared=order[:shared].contiguous(), prefix=prefix, starts=starts,
                  lens=torch.tensor(lens, dtype=torch.int32, device=DEV), rows=torch.tensor(starts, dtype=torch.int32, device=DEV) if case["rows"] > 1 else None,
                  k_pages=normal(pages, page, kv, dim), v_pages=normal(pages, page, kv, dim),
                  q=normal(n, case["heads"], dim, scale=1.0 if case["kind"] == "append" else 1.5))
        # the sequence of every row and its index there, which a program that forms batches knows
        seq = [b for b, c in enumerate(counts) for _ in range(c)]
        index = [lens[b] - c + i for b, c in enumerate(counts) for i in range(c)]
        st["seq"] = torch.tensor(seq, dtype=torch.int64, device=DEV)
        st["index"] = torch.tensor(index, dtype=torch.int64, device=DEV)
        if case["kind"] == "append":
            st["real"] = torch.nonzero(st["index"] >= 0)[:, 0]
            st["k"], st["v"] = normal(n, kv, dim), normal(n, kv, dim)
            st["pos"] = _positions(case, n, gen) if case["far"] else None
        else:
            at = [(b, i) for b, c in enumerate(counts) for i in range(c)]
            st["slot"] = torch.tensor([b * case["rows"] + i for b, i in at], dtype=torch.int64, device=DEV)   # rows in a batch of equal lengths
    if case["kind"] != "attend":
        pairs = case["rot"] // 2
        st["freq"] = torch.tensor([case["theta"] ** (-j / pairs) for j in range(pairs)], dtype=torch.float64, device=DEV)
        st["axis"] = torch.tensor(_axes(case), dtype=torch.int64, device=DEV)
    if own:
        paged = _paged()
        if case["kind"] != "attend":
            st["rope"] = paged.RopeAxes([case["theta"] ** (-j / pairs) for j in range(pairs)], _axes(case), layout=case["layout"])
        if case["kind"] != "rope":
            st["pages"] = paged.KVPages(st["k_pages"], st["v_pages"])
            st["batch"] = paged.Batch(st["lens"], tables, rows=st["rows"], max_rows=case["rows"], prefix=st["shared"] if prefix else None, prefix_len=prefix)
    return st


def _turn(st, x, pos):
    """x [n, heads, dim] turned by pos [axes, n]"""
    half = st["freq"].numel()
    angle = pos.to(torch.float64).T[:, st["axis"]] * st["freq"]
    c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    y = x.float()
    out = y.clone()
    if st["case"]["layout"] == "halves":
        a, b = y[..., :half], y[..., half:2 * half]
        out[..., :half], out[..., half:2 * half] = a * c - b * s, b * c + a * s
    else:
        a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = a * c - b * s, b * c + a * s
    return out.to(x.dtype)


def _scores(q, k, scale, cap):
    s = torch.matmul(q, k.transpose(-1, -2)) * scale
    return cap * torch.tanh(s / cap) if cap else s


def _attend(st):
    case = st["case"]
    B, R, H, G, D, P = case["seqs"], case["rows"], case["heads"], case["kv_heads"], case["dim"], st["prefix"]
    scale, cap, page = D ** -0.5, case["cap"], case["page"]
    n = st["q"].shape[0]
    # everything in the batch of equal lengths [sequence, KV head, row x grouped head, .]
    q = torch.zeros(B * R, H, D, dtype=torch.float32, device=DEV)
    q[st["slot"]] = st["q"].float()
    q = q.view(B, R, G, H // G, D).permute(0, 2, 1, 3, 4).reshape(B, G, R * (H // G), D)
    keys = st["tables"].shape[1] * page
    table = st["tables"].clamp(min=0).long()
    k = st["k_pages"][table].view(B, keys, G, D).permute(0, 2, 1, 3).float()
    v = st["v_pages"][table].view(B, keys, G, D).permute(0, 2, 1, 3).float()
    index = torch.full((B * R,), -1, dtype=torch.int64, device=DEV)
    index[st["slot"]] = st["index"]
    index = index.view(B, 1, R, 1).expand(B, 1, R, H // G).reshape(B, 1, R * (H // G), 1)
    seen = torch.arange(keys, device=DEV).view(1, 1, 1, keys) <= index
    s = _scores(q, k, scale, cap).masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    if P:
        shared = st["shared"].long()
        pk = st["k_pages"][shared].view(-1, G, D)[:P].permute(1, 0, 2).float()
        pv = st["v_pages"][shared].view(-1, G, D)[:P].permute(1, 0, 2).float()
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
    if own:
        paged = _paged()
        if case["kind"] == "rope":
            return paged.rope_axes(st["x"], st["pos"], st["rope"])
        if case["kind"] == "append":
            q = paged.append(st["pages"], st["batch"], st["k"], st["v"], rope=st["rope"], pos=st["pos"], q=st["q"])
            return q, st["k_pages"], st["v_pages"]
        return paged.attention(st["pages"], st["batch"], st["q"], scale=case["dim"] ** -0.5, softcap=case["cap"], return_lse=True)
    if case["kind"] == "rope":
        return _turn(st, st["x"], st["pos"])
    if case["kind"] == "append":
        seq, index, page = st["seq"], st["index"], case["page"]
        pos = st["pos"] if st["pos"] is not None else index.expand(len(case["sections"].split("+")), -1)
        k, real = _turn(st, st["k"], pos), st["real"]   # rows of empty places go nowhere
        at = index[real]
        p = st["tables"][seq[real], at // page].long()
        st["k_pages"][p, at % page], st["v_pages"][p, at % page] = k[real], st["v"][real]
        return _turn(st, st["q"], pos), st["k_pages"], st["v_pages"]
    return _attend(st)


def work(case):
    size = TYPES[case["dtype"]].itemsize
    if case["kind"] == "rope":
        n = case["rows"] * case["heads"]
        return {"bytes": 2 * n * case["dim"] * size + 4 * len(case["sections"].split("+")) * case["rows"], "flops": 3 * n * case["rot"]}
    counts, lens = _shape(case)
    n, H, G, D = sum(counts), case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "append":
        axes = len(case["sections"].split("+")) if case["far"] else 0
        return {"bytes": 2 * n * (H + 2 * G) * D * size + 4 * axes * n, "flops": 3 * n * (H + G) * case["rot"]}
    pairs = sum(c * (case["prefix"] + x - c) + c * (c + 1) // 2 for c, x in zip(counts, lens) if x)
    held = sum(lens) + case["prefix"]
    pages = sum(-(-x // case["page"]) for x in lens) + -(-case["prefix"] // case["page"])
    return {"bytes": 2 * n * H * D * size + 4 * n * H + 2 * held * G * D * size + 4 * pages, "flops": 4 * D * H * pairs}


# ---- the same from the definitions, in 64 bits -------------------------------------------------------------------------------------------
def _exact_turn(case, x, pos):
    """pair by pair of columns: (a, b) is a + ib, multiplied by e^(i angle)"""
    x = x.double()
    out, half = x.clone(), case["rot"] // 2
    for j, a in enumerate(_axes(case)):
        first, second = (j, j + half) if case["layout"] == "halves" else (2 * j, 2 * j + 1)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), pos[a].double() * math.pow(case["theta"], -2.0 * j / case["rot"]))
        z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
        out[..., first], out[..., second] = z.real, z.imag
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_turn(case, st["x"], st["pos"])
    page, G = case["page"], case["kv_heads"]
    if case["kind"] == "append":
        n_axes = len(case["sections"].split("+"))
        pos = torch.stack([st["index"]] * n_axes) if st["pos"] is None else st["pos"]
        k, kp, vp = _exact_turn(case, st["k"], pos), st["k_pages"].double(), st["v_pages"].double()
        tables = st["tables"].cpu()
        for b, (first, c) in enumerate(zip(st["starts"], st["counts"])):
            have = st["held"][b]
            if not have:
                continue
            where = torch.arange(have - c, have)
            flat = (tables[b, where // page].long() * page + where % page).to(DEV)
            kp.view(-1, G, case["dim"])[flat] = k[first:first + c]
            vp.view(-1, G, case["dim"])[flat] = st["v"][first:first + c].double()
        return _exact_turn(case, st["q"], pos), kp, vp
    D, H, cap = case["dim"], case["heads"], case["cap"]
    n = st["q"].shape[0]
    out = torch.zeros(n, H, D, dtype=torch.float64, device=DEV)
    lse = torch.full((n, H), -math.inf, dtype=torch.float64, device=DEV)
    front = st["shared"].long()
    flat_k, flat_v = st["k_pages"].view(-1, G, D), st["v_pages"].view(-1, G, D)
    inside = torch.arange(page, device=DEV)
    front = (front[:, None] * page + inside).reshape(-1)[:st["prefix"]]
    for b, (first, c) in enumerate(zip(st["starts"], st["counts"])):
        have = st["held"][b]
        if not have:
            continue
        mine = (st["tables"][b, :-(-have // page)].long()[:, None] * page + inside).reshape(-1)[:have]
        at = torch.cat([front, mine])
        k, v = flat_k[at].double(), flat_v[at].double()
        for g in range(G):
            q = st["q"][first:first + c, g * (H // G):(g + 1) * (H // G)].double()
            s = torch.einsum("rhd,kd->rhk", q, k[:, g]) / math.sqrt(D)
            if cap:
                s = cap * torch.tanh(s / cap)
            last = st["prefix"] + have - c + torch.arange(c, device=DEV)
            s = torch.where(torch.arange(at.numel(), device=DEV) <= last[:, None, None], s, -math.inf)
            heads = slice(g * (H // G), (g + 1) * (H // G))
            out[first:first + c, heads] = torch.softmax(s, -1) @ v[:, g]
            lse[first:first + c, heads] = torch.logsumexp(s, -1)
    return out, lse
