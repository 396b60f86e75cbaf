"""64-bit definitions of the serving operators, and bounds on what fp32 arithmetic may add, for their tests.

Everything runs on the CPU in float64 with plain torch.  u = 2^-24 is the rounding of one fp32
operation, `half_step(dtype)` that of the output's type.
"""
import math

import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def norm_rope(x, w, positions, inv_freq, eps, interleaved):
    """(y, b): the rotated rows, and the sum of magnitudes that each element is made of."""
    x, w = x.double(), w.double()
    pairs = inv_freq.numel()
    y = x * (x.square().mean(-1, keepdim=True) + eps) ** -0.5 * w
    angle = positions.double()[..., None, None] * inv_freq.double()
    c, s = angle.cos(), angle.sin()
    if interleaved:
        i, j = torch.arange(pairs) * 2, torch.arange(pairs) * 2 + 1
    else:
        i, j = torch.arange(pairs), torch.arange(pairs) + pairs
    a, b = y[..., i], y[..., j]
    out, size = y.clone(), y.abs()
    out[..., i], out[..., j] = a * c - b * s, b * c + a * s
    size[..., i] = size[..., j] = a.abs() + b.abs()
    return out, size


def norm_rope_backward(dy, x, w, positions, inv_freq, eps, interleaved):
    """(dx, dw, bound of dx, bound of dw): bounds in units of u."""
    D = x.shape[-1]
    g, g_size = norm_rope_rotate_back(dy.double(), positions, inv_freq, interleaved)
    x, w = x.double(), w.double()
    r = (x.square().mean(-1, keepdim=True) + eps) ** -0.5
    xh = x * r
    h = g * w
    dx = r * (h - xh * (h * xh).mean(-1, keepdim=True))
    h_size = g_size * w.abs()
    dx_size = r * (h_size + xh.abs() * (h_size * xh.abs()).mean(-1, keepdim=True))
    lead = tuple(range(x.dim() - 1))
    terms = x.numel() // D
    # rows: D products and their sum, twice; weights: a sum of `terms` products in any order
    return dx, (g * xh).sum(lead), 64 * dx_size, (terms + 64) * (g_size * xh.abs()).sum(lead)


def norm_rope_rotate_back(dy, positions, inv_freq, interleaved):
    pairs = inv_freq.numel()
    angle = positions.double()[..., None, None] * inv_freq.double()
    c, s = angle.cos(), -angle.sin()
    if interleaved:
        i, j = torch.arange(pairs) * 2, torch.arange(pairs) * 2 + 1
    else:
        i, j = torch.arange(pairs), torch.arange(pairs) + pairs
    a, b = dy[..., i], dy[..., j]
    g, size = dy.clone(), dy.abs()
    g[..., i], g[..., j] = a * c - b * s, b * c + a * s
    size[..., i] = size[..., j] = a.abs() + b.abs()
    return g, size


# the 127 magnitudes of e4m3, in code order
E4M3 = torch.tensor([(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
                     for e in range(16) for m in range(8)][:127], dtype=torch.float64)


def quantise(x):
    """(codes, exponents) of rows [..., D] as a cache stores them; NaN and infinity have code 127."""
    x = x.double()
    finite = torch.isfinite(x)
    y = torch.where(finite, x, torch.zeros_like(x))
    amax = y.abs().amax(-1)
    e = torch.full(amax.shape, -126, dtype=torch.int64)
    big = amax > 448 * 2.0 ** -126
    e[big] = torch.ceil(torch.log2(amax[big] / 448)).long()  # log2 of a ratio of fp32 numbers, exact at powers of two
    e = e.clamp(min=-126)
    y = y.abs() / (2.0 ** e.double())[..., None]
    hi = torch.searchsorted(E4M3, y.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = E4M3[hi] - y, y - E4M3[lo]
    code = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = torch.where(finite, code, torch.full_like(code, 127))
    return code.to(torch.uint8) | (torch.signbit(x) & finite).to(torch.uint8) * 128, (e + 127).to(torch.uint8)


def dequantise(codes, exponents):
    c = (codes & 127).long()
    v = torch.cat((E4M3, torch.tensor([math.nan], dtype=torch.float64)))[c]
    v = torch.where(codes >= 128, -v, v)
    return v * (2.0 ** (exponents.double() - 127))[..., None]


def fmha_cache(q, k, v, table, context, drafts, tree, scale, before):
    """(out, bound for fp32 arithmetic, bound per unit of relative error of the weights).

    k, v: [pages, heads, page, D] in float64; table [B, width]; lists of lengths; tree [B, N] ints or None;
    `before`: what the output holds.  Keys in pages that the cache does not have are not seen.
    """
    B, N, Hq, D = q.shape
    pages, heads, page, _ = k.shape
    out, arith, weight = before.double().clone(), torch.zeros(q.shape, dtype=torch.float64), torch.zeros(
        q.shape, dtype=torch.float64)
    room = table.shape[1] * page
    for b in range(B):
        queries = min(max(int(drafts[b]) if drafts is not None else N, 0), N)
        ctx = min(max(int(context[b]), 0), room)
        nd = min(queries, room - ctx)
        for n in range(queries):
            word = int(tree[b, n]) if tree is not None else (2 << n) - 1
            keys = list(range(ctx)) + [ctx + j for j in range(nd) if (word >> j) & 1]
            where = [(int(table[b, j // page]), j % page) for j in keys]
            where = [(p, o) for p, o in where if 0 <= p < pages]
            for h in range(Hq):
                if not where:
                    out[b, n, h] = 0
                    continue
                p, o = (torch.tensor(t) for t in zip(*where))
                kk, vv = k[p, h // (Hq // heads), o], v[p, h // (Hq // heads), o]
                x = q[b, n, h].double()
                s = kk @ x * scale
                w = torch.softmax(s, 0)
                y = w @ vv
                size = w @ vv.abs() + y.abs()
                out[b, n, h] = y
                weight[b, n, h] = size
                # a score is off by at most (D + 8) u times the sum of its products' magnitudes, and by
                # a few u of itself in the exponent; weights by twice that relatively; sums by their length
                off = (D + 8) * abs(scale) * (kk.abs() @ x.abs()).max() + 8 * s.abs().max() + 8
                arith[b, n, h] = U * (2 * off + len(where) + 64) * size + 1e-30
    return out, arith, weight
