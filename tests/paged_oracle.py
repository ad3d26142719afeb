"""Many sequences at once in 64 bits, one row and one head at a time, from the definitions: what lmrs_b200.paged is held against.  CPU tensors."""
import math

import torch


def turn(x, pos, freq, axis, layout):
    """x [rows, heads, size] (any dtype) -> float64; pos [axes, rows] integers"""
    out = x.double().clone()
    for j, (f, a) in enumerate(zip(freq, axis)):
        angle = pos[a].double() * f
        c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
        i0, i1 = (j, j + len(freq)) if layout == "halves" else (2 * j, 2 * j + 1)
        a0, a1 = x[..., i0].double(), x[..., i1].double()
        out[..., i0], out[..., i1] = a0 * c - a1 * s, a1 * c + a0 * s
    return out


def turn_tolerance(x, exact, freq, layout):
    """float32 angles: cosine and sine are off by 2^-22.4 at most (2 units in the last place of sincospi, 2^-23, and a quarter turn's argument rounded to
    24 bits, pi / 4 * 2^-24); two products and a sum, each 2^-24 of a value no larger than |a| + |b|; then the type's own half step"""
    n, size = len(freq), x.double().abs()
    total = torch.zeros_like(size)
    for j in range(n):
        i0, i1 = (j, j + n) if layout == "halves" else (2 * j, 2 * j + 1)
        total[..., i0] = total[..., i1] = size[..., i0] + size[..., i1]
    eps = torch.finfo(x.dtype).eps / 2
    return (total * (2 ** -22.4 + 3 * 2 ** -24)) * (1 + eps) + exact.abs() * eps * (0 if x.dtype == torch.float32 else 1) + torch.finfo(x.dtype).tiny


def spans(lens, rows, n_rows):
    """(first row, rows, tokens) of every sequence"""
    if rows is None:
        return [(b, 1, int(n)) for b, n in enumerate(lens)]
    return [(int(rows[b]), int(rows[b + 1]) - int(rows[b]), int(n)) for b, n in enumerate(lens)]


def place(table, pages, page_size, x):
    """(page, slot) of token x, or None"""
    i = x // page_size
    if x < 0 or i >= len(table) or not 0 <= int(table[i]) < pages:
        return None
    return int(table[i]), x % page_size


def attention(k, v, lens, tables, rows, prefix, prefix_len, q, scale, softcap, p_eps):
    """k, v [pages, page_size, kv_heads, size]; q [n, heads, size].  Returns out, lse (float64; NaN rows for rows of no sequence), and how far a kernel
    may be off in either, given that it rounds weights by p_eps and works in float32 otherwise."""
    pages, ps, G, D = k.shape
    n, H = q.shape[:2]
    out, lse = torch.full((n, H, D), math.nan, dtype=torch.float64), torch.full((n, H), math.nan, dtype=torch.float64)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    u = 2.0 ** -24
    front = [place(prefix, pages, ps, x) for x in range(prefix_len)]
    for b, (first, c, have) in enumerate(spans(lens, rows, n)):
        own = [place(tables[b], pages, ps, x) for x in range(max(have, 0))]
        for i in range(c):
            index = have - c + i
            at = [] if index < 0 else [p for p in front + own[:index + 1] if p is not None]
            if not at:
                out[first + i], lse[first + i] = 0.0, -math.inf
                continue
            pg, sl = torch.tensor([p for p, _ in at]), torch.tensor([s for _, s in at])
            keys, values = k[pg, sl].double(), v[pg, sl].double()   # [keys, G, D]
            for h in range(H):
                g = h // (H // G)
                x = q[first + i, h].double()
                s = keys[:, g] @ x * scale
                # a dot product of D terms in f32 is off by D u of the sum of their sizes; the factor and the exponent's argument round again
                size = (keys[:, g].abs() @ x.abs() * abs(scale)).max()
                off = (D + 4) * u * size
                if softcap:
                    s = softcap * torch.tanh(s / softcap)
                    off = off + 8 * u * softcap
                w = torch.exp(s - s.max())
                out[first + i, h] = (w / w.sum()) @ values[:, g]
                lse[first + i, h] = torch.logsumexp(s, 0)
                # weights: the score's error, the exponent's argument (at most the spread of the scores, in f32 powers of two) and 2^-21 for the exponential;
                # numerator and denominator alike; sums of len(at) terms, rescaled on the way; the rounding of the weights
                spread = float((s.max() - s.min()).clamp(max=200.0)) if torch.isfinite(s).all() else 200.0
                rel = 2 * (off + 4 * u * (spread + float(s.abs().max().clamp(max=1e4))) + 2.0 ** -21) + (2 * len(at) + 64) * u
                A = (w / w.sum()) @ values[:, g].abs()
                tol[first + i, h] = A * (rel + p_eps)
                tol_lse[first + i, h] = rel + 4 * u * lse[first + i, h].abs()
    eps = torch.finfo(q.dtype).eps / 2
    tol = tol * (1 + eps) + out.nan_to_num(0.0).abs() * eps + torch.finfo(q.dtype).tiny * (0.5 if q.dtype != torch.float16 else 2.0 ** -10)
    return out, lse, tol, tol_lse
