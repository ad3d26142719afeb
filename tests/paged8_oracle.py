"""Pages of 8-bit codes in 64 bits, from the definitions: what lmrs_b200.paged is held against where the pool is QuantPages, and for norms of heads.  CPU tensors."""
import math

import torch
from paged_oracle import place, spans, turn  # noqa: F401

MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
U = 2.0 ** -24


def numbers(form):
    """the format's numbers, rising, and whether each has an even code"""
    if form == torch.int8:
        up = [float(i) for i in range(128)]
    else:
        up = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8)][:-1]
    even = [i % 2 == 0 for i in range(len(up))]
    return torch.tensor([-x for x in up[:0:-1]] + up, dtype=torch.float64), torch.tensor(even[:0:-1] + even)


def nearest(x, form):
    """the format's number nearest to x (float64), of two as near the one with an even code"""
    all_numbers, even = numbers(form)
    above = torch.searchsorted(all_numbers, x.contiguous()).clamp(1, len(all_numbers) - 1)
    up, down = all_numbers[above] - x, x - all_numbers[above - 1]
    return torch.where((up < down) | ((up == down) & even[above]), all_numbers[above], all_numbers[above - 1])


def norm(x, weight, eps):
    """x [.., heads, size] -> float64; weight [size], [heads, size] or None"""
    y = x.double()
    y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / x.shape[-1] + eps)
    return y if weight is None else y * weight.double()


def norm_tolerance(normed, exact, freq, layout, dtype):
    """Of a norm and a rotation in float32.  The sum of D squares is off by D U of itself, so its root by half of that; the mean, the sum with eps, the root, the quotient and two products round once each.
    Cosine and sine are off by 2^-22.4 at most; two products and a sum of the rotation.  Then the type's own half step."""
    D, n, size = normed.shape[-1], len(freq), normed.abs()
    total = size.clone()
    for j in range(n):
        i0, i1 = (j, j + n) if layout == "halves" else (2 * j, 2 * j + 1)
        total[..., i0] = total[..., i1] = size[..., i0] + size[..., i1]
    eps = torch.finfo(dtype).eps / 2
    return total * ((D / 2 + 6) * U + (2 ** -22.4 + 3 * U if n else 0.0)) * (1 + eps) + exact.abs() * eps + torch.finfo(dtype).tiny


def put(codes, scales, block, form, x, where, slack, got_scale):
    """One array's heads: x [tokens, heads, size] (float64, off by `slack` at most) goes to places where[t] = (page, slot, in the call's block at its beginning?) or None, all of one sequence and in order.  codes (float64)
    [pages, page_size, heads, size] and scales (float64) [pages, blocks, heads] are changed; where a value within `slack` of a border may go to either side, the code is NaN.  got_scale: the scales that
    the call left, which are taken where they are within half a step (and the slack) of the exact ones."""
    done = 0
    while done < len(where):
        if where[done] is None:
            done += 1
            continue
        page, slot, index = where[done]
        start = index // block * block
        n = 1
        while done + n < len(where) and where[done + n] is not None and where[done + n][2] // block * block == start:
            n += 1
        at, in_page = slot - (index - start), (slot - (index - start)) // block
        a = x[done:done + n].abs().amax((0, 2))
        a = torch.where(torch.isfinite(x[done:done + n]).all(0).all(-1), a, math.nan)
        s = (a / MOST[form]).clamp(2.0 ** -60, 2.0 ** 60)
        old = scales[page, in_page].clone()
        if index > start:
            s = torch.where(torch.isnan(old) | torch.isnan(s), math.nan, torch.maximum(s, old))
        got = got_scale[page, in_page].double()
        assert torch.equal(torch.isnan(got), torch.isnan(s))
        fine = ~torch.isnan(s)
        assert ((got - s).abs() <= s * (U + slack))[fine].all(), (got, s)
        scales[page, in_page] = got
        if index > start:
            again = nearest(codes[page, at:slot] * old[None, :, None] / got[None, :, None], form)
            codes[page, at:slot] = torch.where((fine & (got > old))[None, :, None], again, codes[page, at:slot])
        y, off = x[done:done + n] / got[None, :, None], slack * MOST[form]
        low, high = nearest(y - off, form), nearest(y + off, form)
        codes[page, slot:slot + n] = torch.where(low == high, low, math.nan)
        codes[page, slot:slot + n][:, ~fine] = 0.0   # (of a scale that is NaN: any)
        done += n


def attention(k, v, k_scale, v_scale, block, lens, tables, rows, prefix, prefix_len, q, scale, softcap, p_eps):
    """Codes k, v [pages, page_size, kv_heads, size] and scales [pages, blocks, kv_heads], float64; q [n, heads, size].  Returns out, lse (float64; NaN rows for rows of no sequence), and how far a kernel
    may be off in either, given that it rounds weights (times the values' scales) by p_eps, to 2^-32 of the largest of them at least, and works in float32 otherwise."""
    pages, ps, G, D = k.shape
    n, H = q.shape[:2]
    out, lse = torch.full((n, H, D), math.nan, dtype=torch.float64), torch.full((n, H), math.nan, dtype=torch.float64)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    front = [place(prefix, pages, ps, x) for x in range(prefix_len)]
    most = float(torch.nan_to_num(v.abs()).max())
    for b, (first, c, have) in enumerate(spans(lens, rows, n)):
        own = [place(tables[b], pages, ps, x) for x in range(max(have, 0))]
        for i in range(c):
            index = have - c + i
            at = [] if index < 0 else [p for p in front + own[:index + 1] if p is not None]
            if not at:
                out[first + i], lse[first + i] = 0.0, -math.inf
                continue
            pg, sl = torch.tensor([p for p, _ in at]), torch.tensor([s for _, s in at])
            ks, vs = k_scale[pg, sl // block], v_scale[pg, sl // block].clamp(2.0 ** -60, 2.0 ** 60)   # [keys, G]
            for h in range(H):
                g = h // (H // G)
                keys, values = k[pg, sl, g] * ks[:, g, None], v[pg, sl, g] * vs[:, g, None]
                x = q[first + i, h].double()
                s = keys @ x * scale
                # a dot product of D terms in f32 is off by D U of the sum of their sizes; the key's scale, the factors and the exponent's argument round again
                off = (D + 8) * U * (keys.abs() @ x.abs() * abs(scale)).max()
                if softcap:
                    s = softcap * torch.tanh(s / softcap)
                    off = off + 8 * U * softcap
                w = torch.softmax(s, 0)
                out[first + i, h] = w @ values
                lse[first + i, h] = torch.logsumexp(s, 0)
                # weights: the score's error, the exponent's argument (the spread of the scores and of the scales, in f32 powers of two), 2^-21 each for the exponential and for the scale's logarithm and
                # reciprocal; numerator and denominator alike; sums of len(at) terms, rescaled on the way; the rounding of the weights
                spread = float((s.max() - s.min()).clamp(max=200.0)) if torch.isfinite(s).all() else 200.0
                logs = float(torch.log2(vs[:, g]).abs().nan_to_num(0.0).max())
                rel = 2 * (off + 4 * U * (spread + logs + float(s.abs().max().clamp(max=1e4))) + 2 * 2.0 ** -21) + (2 * len(at) + 64) * U
                tol[first + i, h] = (w @ values.abs()) * (rel + p_eps) + len(at) * 2.0 ** -32 * most * float((w * vs[:, g]).max())
                tol_lse[first + i, h] = rel + 4 * U * lse[first + i, h].abs()
    eps = torch.finfo(q.dtype).eps / 2
    tol = tol * (1 + eps) + out.nan_to_num(0.0).abs() * eps + torch.finfo(q.dtype).tiny * (0.5 if q.dtype != torch.float16 else 2.0 ** -10)
    return out, lse, tol, tol_lse
