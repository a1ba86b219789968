"""The attention side of a layer in 64 bits on the CPU, from its formulas: what the GPU tests compare with."""
import math

import torch


def slots(table, page, lo, hi):
    at = torch.arange(lo, hi)
    return table[at // page].long(), at % page


def visible(ntok, ctx, keys, tree_rows=None, words=0):
    """[ntok, keys] bool: the whole context, then rows 0 .. i or the bits of tree_rows."""
    see = torch.zeros((ntok, keys), dtype=torch.bool)
    see[:, :ctx] = True
    for i in range(ntok):
        for j in range(min(ntok, keys - ctx)):
            if tree_rows is None:
                see[i, ctx + j] = j <= i
            else:
                see[i, ctx + j] = j < 32 * words and bool((int(tree_rows[i, j // 32]) >> (j % 32)) & 1)
    return see


def attention(k, v, q, row_start, context, table, scale, tree=None):
    """k, v [pages, kv_heads, page, dim] (one layer), q [rows, heads, dim], CPU tensors of any float type ->
    (out f64, lse f64, and sum_j p_j |v_j|, the scale of the products' rounding)."""
    rows, heads, dim = q.shape
    kvh, page = k.shape[1], k.shape[2]
    out = torch.zeros((rows, heads, dim), dtype=torch.float64)
    mass = torch.zeros((rows, heads, dim), dtype=torch.float64)
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64)
    for s in range(len(context)):
        a, b, ctx = row_start[s], row_start[s + 1], context[s]
        n = b - a
        if n == 0:
            continue
        pg, of = slots(table[s], page, 0, ctx + n)
        kk, vv = k[pg, :, of].double(), v[pg, :, of].double()  # [keys, kvh, dim]
        see = visible(n, ctx, ctx + n, None if tree is None else tree[a:b], 0 if tree is None else tree.shape[1])
        for h in range(heads):
            kh = h // (heads // kvh)
            for i in range(n):
                ok = see[i]
                if not bool(ok.any()):
                    continue
                z = (kk[ok, kh] @ q[a + i, h].double()) * scale
                lse[a + i, h] = torch.logsumexp(z, 0)
                p = torch.exp(z - lse[a + i, h])
                out[a + i, h] = p @ vv[ok, kh]
                mass[a + i, h] = p @ vv[ok, kh].abs()
    return out, lse, mass


def norm_rotate(x, weight, pos, inv_freq, eps, adjacent, offset=0.0):
    """x [rows, heads, dim] -> f64."""
    y = x.double().clone()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * (weight.double() + offset)
    if inv_freq is None or inv_freq.numel() == 0:
        return y
    half = inv_freq.numel()
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if adjacent else (i, i + half)
    t = pos.double()[:, None, None] * inv_freq
    x0, x1 = y[..., a].clone(), y[..., b].clone()
    y[..., a] = x0 * torch.cos(t) - x1 * torch.sin(t)
    y[..., b] = x1 * torch.cos(t) + x0 * torch.sin(t)
    return y
