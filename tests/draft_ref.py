"""Verification of drafted tokens in 64 bits on the CPU, one sequence and one child at a time: what the GPU tests of
exl3_draft_verify compare with."""
import math

import torch


def probabilities(logits, temperature):
    """softmax(logits / temperature) of one row, f64; None for a row without a logit above -inf."""
    x = logits.double()
    x = torch.where(torch.isnan(x), -math.inf, x).clamp(max=torch.finfo(torch.float32).max)
    top = x.max()
    if top == -math.inf:
        return None
    if temperature == 0:
        p = torch.zeros_like(x)
        p[int((x == top).nonzero()[0])] = 1.0
        return p
    z = (x - top) / temperature / math.log(2.0)
    p = torch.where(z >= -100, torch.exp2(z), 0.0)
    return p / p.sum()


def verify_one(logits, tokens, parent, uniform, temperature, draft, depth):
    """One sequence's rows -> (path, token, near): near is the least distance of a decision (an acceptance, a place in the
    cumulative sums) from its border, in units of what f32 exponentials may move it by.

    An exponential is within 2^-22 + 2^-24 |x - m| / T of itself, in its slice and the slice in the row together within twice
    the first and once the second; weighted by p, |x - m| / T sums to at most ln(vocab) + 1 < 14.  So p's sums are within
    2^-21 + 14 2^-24 of themselves, p (divided by one) within twice that, < 2^-18.6.  With k rejections behind it, A_k = sum
    Z_i: each Z_i = sum max(p - A_i q, 0) is off by at most that + err(A_i) (sum q = 1), so err(A_k) <= (2^k - 1) 2^-18.6;
    u q Z - r and cumsum r - u Z are then within 2 (2^-18.6 + err(A_k)) < 2^(k - 17).  Without draft nothing is subtracted
    but whole tokens, and it stays 2^-17."""
    n, vocab = logits.shape
    path, at, near = [0], 0, math.inf
    while True:
        p = probabilities(logits[at], temperature)
        if p is None:
            return path, -1, near
        r, z, child, unit = p, 1.0, None, 2.0 ** -17
        for c in range(at + 1, n) if len(path) < depth else ():
            x = int(tokens[c])
            if int(parent[c]) != at or not 0 <= x < vocab:
                continue
            if draft is None or temperature == 0:
                q = torch.zeros(vocab, dtype=torch.float64)
                q[x] = 1.0
            else:
                q = torch.nan_to_num(draft[at].double(), nan=0.0).clamp(min=0)
            border = float(uniform[c, 0]) * float(q[x]) * z
            if temperature:
                near = min(near, abs(float(r[x]) - border) / unit)
            if border < float(r[x]):
                child = c
                break
            less = (r - z * q).clamp(min=0)
            r, z = (less, float(less.sum())) if float(less.sum()) > 0 else (p, 1.0)
            unit *= 1 if draft is None else 2
        if child is None:
            break
        path.append(child)
        at = child
    upto = r.cumsum(0)
    goal = float(uniform[at, 1]) * z
    over = (upto > goal).nonzero()
    token = int(over[0]) if len(over) else int((r > 0).nonzero()[-1])
    if temperature:
        near = min(near, float((upto - goal).abs().min()) / unit)
    return path, token, near


def verify(row_start, logits, tokens, parent, uniform, temperature, draft, depth):
    """-> (paths, tokens, near) of every sequence; parent None: chains."""
    paths, out, near = [], [], []
    for s in range(len(row_start) - 1):
        a, b = row_start[s], row_start[s + 1]
        if a == b:
            paths.append([]), out.append(-1), near.append(math.inf)
            continue
        par = torch.arange(-1, b - a - 1) if parent is None else parent[a:b]
        got = verify_one(logits[a:b], tokens[a:b], par, uniform[a:b], 1.0 if temperature is None else float(temperature[s]),
                         None if draft is None else draft[a:b], depth)
        paths.append(got[0]), out.append(got[1]), near.append(got[2])
    return paths, out, near
