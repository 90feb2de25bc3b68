"""Plain statements, in 64 bits, of the operators over a cache in 8 bits, and what their results may be off by.

The bounds.  A weight is held in float16: half a step is 2^-12 of it, at least 2^-25 of a row's largest weight (its smallest step
there is 2^-24).  The output is rounded to bfloat16: 2^-8 of its value at most.  A score is a sum of products in the tensor cores' 32-bit
accumulators: off by at most 2^-20 of the sum of the products' sizes (16 steps of 16 products each, every step off by a few 2^-24), and by
2^-22 of its own size in the exponent's arithmetic; a score's error is a weight's relative error, once in the numerator and once in
the denominator."""
import math

import torch

D = torch.float64
LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def grid(kind):
    """The codes' values, ascending, and whether each has an even last bit."""
    if kind == torch.int8:
        v = torch.arange(-127, 128, dtype=D)
        return v, v % 2 == 0
    v = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).to(D)
    even = torch.arange(0, 127) % 2 == 0
    return torch.cat([-v[1:].flip(0), v]), torch.cat([even[1:].flip(0), even])


def nearest(x, kind):
    g, even = grid(kind)
    x = x.clamp(-LARGEST[kind], LARGEST[kind]).contiguous()
    hi = torch.searchsorted(g, x).clamp(1, g.numel() - 1)
    a, b = x - g[hi - 1], g[hi] - x
    return torch.where((a < b) | ((a == b) & even[hi - 1]), g[hi - 1], g[hi])


def exponent(top, kind):
    """Least e in -100 .. 100 with top <= largest * 2^e."""
    e = -100
    while e < 100 and top > LARGEST[kind] * 2.0 ** e:
        e += 1
    return e


def write(x, pages, scales, table, cu_q, ctx_before):
    """Keys (or values) x [N, nKV * hd] into CPU copies of pages (values of the codes, float64) and scales (float64)."""
    kind, values, factors = pages.dtype, pages.to(D), scales.to(D)
    _, n_kv, page, hd = pages.shape
    block = page // scales.shape[2]
    for e in range(len(ctx_before)):
        ctx, q0, n = int(ctx_before[e]), int(cu_q[e]), int(cu_q[e + 1] - cu_q[e])
        rows = x[q0:q0 + n].to(D).view(n, n_kv, hd)
        for b in range(ctx // block, -(-(ctx + n) // block) if n else 0):
            lo, hi = max(ctx, b * block), min(ctx + n, (b + 1) * block)
            p, at = int(table[e, b * block // page]), b * block % page
            if p < 0:
                continue
            for h in range(n_kv):
                part = rows[lo - ctx:hi - ctx, h]
                finite = part[torch.isfinite(part)]
                f = 2.0 ** exponent(float(finite.abs().max()) if finite.numel() else 0.0, kind)
                old = float(factors[p, h, at // block])
                if lo > b * block and old > f:
                    f = old
                front = values[p, h, at:at + lo - b * block]
                if lo > b * block and f > old:
                    values[p, h, at:at + lo - b * block] = nearest(front * (old / f), kind)
                codes = nearest(torch.nan_to_num(part / f, nan=0.0, posinf=1e300, neginf=-1e300), kind)
                if kind != torch.int8:
                    codes = torch.where(torch.isnan(part), part, codes)
                values[p, h, at + lo - b * block:at + hi - b * block] = codes
                factors[p, h, at // block] = f
    return values, factors


def attention(q, k_pages, v_pages, k_scales, v_scales, table, cu_q, ctx_before, n_heads, window, scale, slopes=None):
    """(out, bound) [N, nH * hd] in float64 on the CPU for every row of every entry; rows of no entry are zero with a bound of zero."""
    k_pages, v_pages, k_scales, v_scales, table, q = (t.cpu() for t in (k_pages, v_pages, k_scales, v_scales, table, q))
    _, n_kv, page, hd = k_pages.shape
    block = page // k_scales.shape[2]
    out = torch.zeros(q.shape, dtype=D)
    bound = torch.zeros(q.shape, dtype=D)
    group = n_heads // n_kv
    for e in range(len(ctx_before)):
        ctx, q0, n = int(ctx_before[e]), int(cu_q[e]), int(cu_q[e + 1] - cu_q[e])
        if n == 0:
            continue
        j = torch.arange(ctx + n)
        p, at = table[e][j // page].long(), j % page
        for h in range(n_heads):
            g = h // group
            ks, vs = k_scales[p, g, at // block].to(D)[:, None], v_scales[p, g, at // block].to(D)[:, None]
            k = k_pages[:, g].view(torch.uint8)[p, at].view(k_pages.dtype).to(D) * ks
            v = v_pages[:, g].view(torch.uint8)[p, at].view(v_pages.dtype).to(D) * vs
            qq = q[q0:q0 + n, h * hd:(h + 1) * hd].to(D)
            pos = torch.arange(ctx, ctx + n)[:, None]
            s = qq @ k.T * scale
            if slopes is not None:
                s = s - float(slopes[h]) * (pos - j).to(D)
            seen = (j <= pos) & ((j > pos - window) if window else torch.ones_like(j, dtype=torch.bool))
            s = s.masked_fill(~seen, -math.inf)
            w = torch.softmax(s, -1)
            # keys that no row sees may hold anything
            some = seen.any(0)[:, None]
            k, v, vs = torch.where(some, k, 0.0), torch.where(some, v, 0.0), torch.where(some, vs, 0.0)
            o = w @ v
            size = (qq.abs() @ k.T.abs() * scale).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            far = s.masked_fill(~seen, 0.0).abs().amax(-1, keepdim=True)
            rel = 2.0 ** -11 + 2 * (2.0 ** -20 * size + 2.0 ** -22 * (1.5 * far + 128))
            small = 2.0 ** -25 * seen.sum(-1, keepdim=True) * LARGEST[k_pages.dtype] * vs.max()
            out[q0:q0 + n, h * hd:(h + 1) * hd] = o
            bound[q0:q0 + n, h * hd:(h + 1) * hd] = 2.0 ** -8 * o.abs() + rel * (w @ v.abs()) + small
    return out, bound
