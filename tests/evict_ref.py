"""Accumulated attention weights in 64 bits, and eviction by them slot by slot, on the CPU: what the GPU tests of
exl3_attention_weight and exl3_cache_evict compare with."""
import math

import torch

import attention_ref as R


def weights(k, q, lse, row_start, context, table, scale, decay, old, tree=None):
    """k [pages, kv_heads, page, dim] (one layer), q [rows, heads, dim], lse [rows, heads], old [nseq, kv_heads, slots]:
    CPU tensors -> (the new weights f64, how far f32 arithmetic may be off).

    The bound, term by term: the scores' D products are exact in f32 and each of their additions is off by at most 2^-23 of
    what is summed, sum |q k| (a tensor core may cut instead of rounding); the score in units of log 2, the rounded
    scale and log-sum-exp and their difference by 2^-22 (|score| + |lse|); a power of two by 2^-21.  A sum of n terms is
    off by n 2^-24 of itself, the update by two roundings."""
    kvh, page, heads, dim = k.shape[1], k.shape[2], q.shape[1], q.shape[2]
    out, off = old.double().clone(), torch.zeros(old.shape, dtype=torch.float64)
    for s in range(len(context)):
        a, b, ctx = row_start[s], row_start[s + 1], context[s]
        n = b - a
        if n == 0:
            continue
        pg, of = R.slots(table[s], page, 0, ctx + n)
        kk = k[pg, :, of].double()
        see = R.visible(n, ctx, ctx + n, None if tree is None else tree[a:b], 0 if tree is None else tree.shape[1])
        for g in range(kvh):
            w = torch.zeros(ctx + n, dtype=torch.float64)
            err = torch.zeros_like(w)
            count = 0
            for h in range(g * (heads // kvh), (g + 1) * (heads // kvh)):
                l = lse[a:b, h].double()[:, None]
                z = q[a:b, h].double() @ kk[:, g].T * scale
                some = see & (l != -math.inf)
                e = torch.where(some, torch.exp(z - l), 0.0)
                each = dim * 2.0 ** -23 * scale * (q[a:b, h].double().abs() @ kk[:, g].abs().T) + \
                    2.0 ** -22 * (z.abs() + l.abs()) + 2.0 ** -21
                w += e.sum(0)
                err += torch.where(some, e * each, 0.0).sum(0)
                count += n
            err += count * 2.0 ** -24 * w
            if decay:
                w[:ctx] += out[s, g, :ctx] * decay
            out[s, g, :ctx + n] = w
            off[s, g, :ctx + n] = err + 2.0 ** -23 * w.abs()
    return out, off


def key(w):
    """Heavier first; NaN is the heaviest of all."""
    return math.inf if math.isnan(w) else w


def kept_slots(w, n, keep, sink, recent):
    """Of n slots with weights w, the `keep` that stay, ascending."""
    always = [j for j in range(n) if j < sink or j >= n - recent]
    rest = [j for j in range(n) if sink <= j < n - recent]
    # (NaN before +inf: a second key tells them apart)
    rest.sort(key=lambda j: (-key(w[j]), not math.isnan(w[j]), j))
    return sorted((always + rest)[:keep])


def evict(k, v, weight, refs, table, held, lens, budget, sink, recent, after=None):
    """k, v [layers, pages, kv_heads, page, dim], weight [layers, nseq, kv_heads, slots], the page state as lists -> the new
    (k, v, weights, refs, table, held, lens, missing); `after`: what the weights' result held before (default: weight)."""
    layers, pages, kvh, page = k.shape[:4]
    nseq = len(lens)
    keep = [min(lens[i], max(budget[i], sink + recent)) if budget[i] >= 0 else lens[i] for i in range(nseq)]
    cut = [keep[i] < lens[i] for i in range(nseq)]
    free = [p for p in range(pages) if refs[p] == 0]
    refs2, table2, held2 = list(refs), [list(t) for t in table], list(held)
    asked = 0
    for i in range(nseq):
        if not cut[i]:
            continue
        held2[i] = -(-keep[i] // page)
        for j in range(held[i]):
            p = table[i][j]
            if j >= held2[i]:
                refs2[p] -= 1
                table2[i][j] = -1
            elif refs[p] > 1:
                refs2[p] -= 1
                if asked < len(free):
                    table2[i][j] = free[asked]
                    refs2[free[asked]] = 1
                asked += 1
    k2, v2 = k.clone(), v.clone()
    w2 = (weight if after is None else after).clone()
    if asked > len(free):
        for i in range(nseq):
            w2[:, i, :, :lens[i]] = weight[:, i, :, :lens[i]]
        return k2, v2, w2, list(refs), [list(t) for t in table], list(held), list(lens), asked - len(free)
    for i in range(nseq):
        if not cut[i]:
            w2[:, i, :, :lens[i]] = weight[:, i, :, :lens[i]]
            continue
        for la in range(layers):
            for h in range(kvh):
                for d, j in enumerate(kept_slots(weight[la, i, h].tolist(), lens[i], keep[i], sink, recent)):
                    a, b = (table[i][j // page], h, j % page), (table2[i][d // page], h, d % page)
                    k2[la][b], v2[la][b] = k[la][a], v[la][a]
                    w2[la, i, h, d] = weight[la, i, h, j]
    return k2, v2, w2, refs2, table2, held2, keep, 0
