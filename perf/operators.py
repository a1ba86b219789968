"""The attention side of a decode step over a paged key/value cache, as measured work.

Three operators of :mod:`plugins_b200.attention`:

* ``norm_rope`` -- per-head RMS norms of queries and keys and the position rotation, keys and values written to their
  cache slots in the same pass;
* ``attention`` -- attention of every sequence's new tokens (one token, a tree of drafted tokens, a prompt chunk) over
  the paged cache;
* ``fork_grow`` / ``compact`` / ``keep`` -- the cache's pages: forking and freeing rows and growing them with copy on
  write, defragmentation, and keeping a drafted tree's accepted path (after the pass that wrote the tree).

The plain forms are elementary torch operations in 32 bits, rounded once at the end.
"""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6
THETA = 1000000.0


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one layer's q|k|v of one token: the latency of a decode step's smallest launch
        dict(name="rope_token", op="norm_rope", nseq=1, rows_lo=1, rows_hi=1, ctx_lo=700, ctx_hi=700, heads=32,
             kv_heads=8, dim=128, rot=128, page=16, dtype="f16", cache="f16", pairs="halves"),
        # 19 sequences' drafted trees in 32-bit activations, two of the model seam's wide heads, a quarter rotated
        dict(name="rope_trees_d256_f32", op="norm_rope", nseq=19, rows_lo=17, rows_hi=64, ctx_lo=33, ctx_hi=5000,
             heads=16, kv_heads=8, dim=256, rot=64, page=64, dtype="f32", cache="bf16", pairs="halves"),
        # the q|k|v of an 8192-row prompt pass
        dict(name="rope_prompt_8192", op="norm_rope", nseq=3, rows_lo=2200, rows_hi=3300, ctx_lo=0, ctx_hi=911,
             heads=32, kv_heads=8, dim=128, rot=128, page=64, dtype="bf16", cache="bf16", pairs="adjacent"),
        # one sequence, one token, a short chat: latency
        dict(name="attn_token_short", op="attention", nseq=1, rows_lo=1, rows_hi=1, ctx_lo=301, ctx_hi=301, heads=32,
             kv_heads=8, dim=128, page=16, dtype="f16", tree=False),
        # a batch of eight decoding, ragged contexts
        dict(name="attn_decode_8", op="attention", nseq=8, rows_lo=1, rows_hi=1, ctx_lo=1500, ctx_hi=9001, heads=32,
             kv_heads=8, dim=128, page=16, dtype="f16", tree=False),
        # 32 sequences verifying 16-token trees over long contexts: the bandwidth-bound middle
        dict(name="attn_trees_32x16", op="attention", nseq=32, rows_lo=16, rows_hi=16, ctx_lo=4000, ctx_hi=8190,
             heads=32, kv_heads=8, dim=128, page=64, dtype="bf16", tree=True),
        # wide heads, small ragged trees over 32k contexts
        dict(name="attn_trees_d256_32k", op="attention", nseq=5, rows_lo=3, rows_hi=9, ctx_lo=20011, ctx_hi=32749,
             heads=16, kv_heads=8, dim=256, page=128, dtype="f16", tree=True),
        # wide trees (64 drafted tokens): many rows per key
        dict(name="attn_trees_8x64", op="attention", nseq=8, rows_lo=63, rows_hi=64, ctx_lo=12000, ctx_hi=16301,
             heads=32, kv_heads=8, dim=128, page=64, dtype="bf16", tree=True),
        # a prompt's second 4096-row chunk, causal: the largest, bound by the matrix products
        dict(name="attn_prompt_4096", op="attention", nseq=1, rows_lo=4096, rows_hi=4096, ctx_lo=4096, ctx_hi=4096,
             heads=32, kv_heads=8, dim=128, page=64, dtype="bf16", tree=False),
        # 24 conversations forked to 48 rows (some dropped), each grown by a tree's pages, shared last pages copied in
        # all 36 layers
        dict(name="pages_fork_grow", op="fork_grow", nseq=24, nout=48, layers=36, ctx_lo=100, ctx_hi=1300, rows=33,
             kv_heads=8, dim=128, page=16, dtype="bf16", spare=256),
        # a pool half emptied by ended conversations, its live pages moved together
        dict(name="pages_compact", op="compact", nseq=40, layers=36, ctx_lo=40, ctx_hi=800, kv_heads=8, dim=128,
             page=16, dtype="f16", spare=900),
        # one verification's end in a 36-layer cache: the trees' keys and values written, the accepted paths kept
        dict(name="keep_paths", op="keep", nseq=32, rows_lo=9, rows_hi=16, layers=36, ctx_lo=65, ctx_hi=700, heads=32,
             kv_heads=8, dim=128, rot=128, page=16, dtype="bf16", cache="bf16", pairs="halves"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] < 1.8e9 and w["flops"] < 4e11:  # at most the largest listed cases
            return c


def _draw(rng):
    op = rng.choice(["norm_rope", "attention", "attention", "attention", "fork_grow", "compact", "keep"])
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (16, 8, 256), (16, 16, 128), (24, 4, 128), (8, 1, 64),
                                       (10, 2, 128)])
    dtype = rng.choice(["f16", "bf16"])
    page = rng.choice([16, 32, 64, 128])
    if op == "norm_rope":
        rows = _log(rng, 1, 8000)
        nseq = min(rows, _log(rng, 1, 40))
        hi = max(1, rows // nseq)
        return dict(op=op, nseq=nseq, rows_lo=max(1, hi // 2), rows_hi=hi, ctx_lo=0, ctx_hi=_log(rng, 1, 4000),
                    heads=heads, kv_heads=kv_heads, dim=dim, rot=rng.choice([dim, dim // 2, dim // 4]), page=page,
                    dtype=rng.choice(["f16", "bf16", "f32"]), cache=dtype, pairs=rng.choice(["halves", "adjacent"]))
    if op == "attention":
        kind = rng.choice(["token", "tree", "prompt"])
        rows = 1 if kind == "token" else _log(rng, 2, 64) if kind == "tree" else _log(rng, 65, 3000)
        nseq = _log(rng, 1, 48) if kind != "prompt" else _log(rng, 1, 3)
        ctx = _log(rng, 1, 16000) if kind != "prompt" else rng.choice([0, _log(rng, 1, 2000)])
        while nseq > 1 and nseq * (ctx + rows) * kv_heads * dim > 32 * 8200 * 8 * 128:
            nseq = (nseq + 1) // 2
        return dict(op=op, nseq=nseq, rows_lo=max(1, rows // 2), rows_hi=rows, ctx_lo=ctx // 3, ctx_hi=ctx, heads=heads,
                    kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, tree=kind == "tree")
    layers = rng.choice([1, 4, 36])
    kv_heads, dim = rng.choice([(8, 128), (8, 256), (4, 128), (1, 64)])
    ctx = _log(rng, 8, 1400 if layers == 36 else 6000)
    page = rng.choice([16, 32, 64])
    nseq = _log(rng, 2, 40)
    if op == "fork_grow":
        return dict(op=op, nseq=nseq, nout=nseq + rng.randrange(0, nseq + 1), layers=layers, ctx_lo=ctx // 2, ctx_hi=ctx,
                    rows=_log(rng, 1, 60), kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, spare=rng.randrange(50, 300))
    if op == "compact":
        return dict(op=op, nseq=nseq, layers=layers, ctx_lo=ctx // 2, ctx_hi=ctx, kv_heads=kv_heads, dim=dim, page=page,
                    dtype=dtype, spare=rng.randrange(10, 600))
    rows = _log(rng, 1, 40)
    return dict(op=op, nseq=nseq, rows_lo=max(1, rows // 2), rows_hi=rows, layers=layers, ctx_lo=ctx // 2, ctx_hi=ctx,
                heads=4 * kv_heads, kv_heads=kv_heads, dim=dim, rot=dim, page=page, dtype=dtype, cache=dtype,
                pairs="halves")


def _spread(lo, hi, n):
    """n whole numbers over [lo, hi], the ends among them, in a mixed order; the same for the same case."""
    if n == 1:
        return [hi]
    v = [lo + (hi - lo) * i // (n - 1) for i in range(n)]
    random.Random(n).shuffle(v)
    return v


def _sizes(c):
    rows = _spread(c["rows_lo"], c["rows_hi"], c["nseq"]) if "rows_lo" in c else [0] * c["nseq"]
    return rows, _spread(c["ctx_lo"], c["ctx_hi"], c["nseq"])[::-1]


def _trees(c):
    """Each drafted token's ancestors (itself among them), by sequence: a token's parent is one before it."""
    out = []
    for b, n in enumerate(_sizes(c)[0]):
        r, anc = random.Random(1000 * b + n), []
        for i in range(n):
            parent = r.randrange(max(0, i - 6), i) if i else None
            anc.append((anc[parent] if i else []) + [i])
        out.append(anc)
    return out


def _pages_of(tokens, page):
    return -(-tokens // page)


def work(c):
    e = {"f16": 2, "bf16": 2, "f32": 4}
    if c["op"] in ("norm_rope", "keep"):
        rows = sum(_sizes(c)[0])
        ce = e[c["cache"]]
        n = rows * c["dim"]
        b = n * (c["heads"] * 2 * e[c["dtype"]] + 2 * c["kv_heads"] * (e[c["dtype"]] + ce))
        if c["op"] == "keep":  # the accepted tokens of every layer, read and written once
            b += sum(_kept(c)) * c["layers"] * c["kv_heads"] * c["dim"] * 2 * 2 * ce
        return {"bytes": b, "flops": 10 * n * (c["heads"] + c["kv_heads"])}
    if c["op"] == "attention":
        rows, ctx = _sizes(c)
        seen = sum(r + x for r, x in zip(rows, ctx))
        if c["tree"]:
            pairs = sum(r * x for r, x in zip(rows, ctx)) + sum(len(a) for t in _trees(c) for a in t)
        else:
            pairs = sum(r * x + r * (r + 1) // 2 for r, x in zip(rows, ctx))
        es = e[c["dtype"]]
        return {"bytes": es * c["dim"] * (2 * seen * c["kv_heads"] + 2 * sum(rows) * c["heads"]) + 4 * sum(rows) * c["heads"],
                "flops": 4 * c["dim"] * c["heads"] * pairs}
    es, plan = e[c["dtype"]], _plan(c)
    page_bytes = c["layers"] * 2 * c["kv_heads"] * c["page"] * c["dim"] * es
    small = 4 * (2 * plan["pages"] + plan["nout"] * plan["width"] + c["nseq"] * plan["width"])
    return {"bytes": 2 * page_bytes * plan["moved"] + small, "flops": 0}


def _kept(c):
    return [1 + (7 * b) % n for b, n in enumerate(max(len(a) for a in t) for t in _trees(c))]


def _plan(c):
    """The page state of a fork_grow or compact case: what a server's bookkeeping holds (ids in a mixed order)."""
    ctx = _sizes(c)[1]
    page = c["page"]
    held = [_pages_of(x, page) for x in ctx]
    pages = sum(held) + c["spare"]
    width = max(held) + (_pages_of(c["rows"], page) + 1 if c["op"] == "fork_grow" else 0)
    if c["op"] == "fork_grow":
        pages += c["nout"] * (_pages_of(c["rows"], page) + 2)
    ids = list(range(pages))
    random.Random(pages).shuffle(ids)
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-1] * (width - h))
        at += h
    plan = dict(pages=pages, width=width, held=held, lens=ctx, table=table, nout=c["nseq"], used=at, ids=ids)
    if c["op"] == "compact":
        plan["moved"] = sum(1 for p in ids[:at] if p >= at)
        return plan
    r = random.Random(c["nseq"])
    parent = [i if i < c["nseq"] and i % 7 != 3 else r.randrange(c["nseq"]) for i in range(c["nout"])]
    plan |= dict(nout=c["nout"], parent=parent)
    plan["moved"] = sum(n - 1 for p, n in ((p, parent.count(p)) for p in set(parent)) if ctx[p] % page)
    return plan


# ------------------------------------------------------------------ inputs

def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype).cuda()


def _cache(c, pages, g):
    """A pool in use: every slot holds keys and values, those no sequence owns stale ones."""
    shape = (c.get("layers", 2), pages, c["kv_heads"], c["page"], c["dim"])
    dt = DTYPES[c.get("cache", c["dtype"])]
    k = torch.empty(shape, dtype=dt, device="cuda")
    v = torch.empty(shape, dtype=dt, device="cuda")
    k.normal_(generator=g)
    v.normal_(generator=g)
    return k, v


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c, "op": c["op"]}
    if c["op"] in ("fork_grow", "compact"):
        p = _plan(c)
        refs = [0] * p["pages"]
        for i in p["ids"][:p["used"]]:
            refs[i] = 1
        s["k"], s["v"] = _cache(c, p["pages"], g)
        s |= dict(refs=_ints(refs), table=_ints(p["table"]), held=_ints(p["held"]), lens=_ints(p["lens"]))
        if c["op"] == "fork_grow":
            s["parent"] = _ints(p["parent"])
            s["need"] = _ints([p["lens"][i] + c["rows"] for i in p["parent"]])
    else:
        rows, ctx = _sizes(c)
        held = [_pages_of(r + x, c["page"]) for r, x in zip(rows, ctx)]
        pages, width = sum(held) + 5, max(held) + 1
        ids = list(range(pages))
        random.Random(seed).shuffle(ids)
        table, at = [], 0
        for h in held:
            table.append(ids[at:at + h] + [-1] * (width - h))
            at += h
        start = [0]
        for r in rows:
            start.append(start[-1] + r)
        dt = DTYPES[c["dtype"]]
        s |= dict(row_start=_ints(start), context=_ints(ctx), table=_ints(table), max_rows=max(rows),
                  max_context=max(r + x for r, x in zip(rows, ctx)))
        s["k"], s["v"] = _cache(c, pages, g)
        s["layer"] = s["k"].shape[0] - 1
        n, h, kh, d = start[-1], c["heads"], c["kv_heads"], c["dim"]
        s["tree"] = s["position"] = None
        if c.get("tree") or c["op"] == "keep":
            trees, words = _trees(c), -(-max(rows) // 32)
            bits = [[sum(1 << (j - 32 * w) for j in a if j // 32 == w) for w in range(words)] for t in trees for a in t]
            s["tree"] = _ints([[x - (1 << 32) if x >> 31 else x for x in r] for r in bits])
            s["position"] = _ints([ctx[b] + len(a) - 1 for b, t in enumerate(trees) for a in t])
            if c["op"] == "keep":
                deepest = [max(t, key=len) for t in trees]
                depth = max(map(len, deepest))
                s["path"] = _ints([a + [-1] * (depth - len(a)) for a in deepest])
                s["kept"] = _ints(_kept(c))
        if c["op"] == "attention":
            s["q"] = torch.randn((n, h, d), generator=g, device="cuda").to(dt)
        else:
            # q|k|v as one projection's rows: the heads are views into them
            qkv = torch.randn((n, (h + 2 * kh) * d), generator=g, device="cuda").mul_(2.5).to(dt)
            s["q"], s["key"], s["value"] = (t.unflatten(1, (-1, d)) for t in qkv.split([h * d, kh * d, kh * d], 1))
            s["q_weight"], s["k_weight"] = ((1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(dt) for _ in range(2))
            half = torch.arange(c["rot"] // 2, dtype=torch.float64, device="cuda")
            s["inv_freq"] = THETA ** (-2 * half / c["rot"])
    if own:
        from plugins_b200 import attention as A
        s["cache"] = A.KvCache(s["k"], s["v"])
        if "refs" in s:
            s["pages"] = A.PageState(s["refs"], s["table"], s["held"], s["lens"])
        else:
            s["batch"] = A.TreeBatch(s["row_start"], s["context"], s["table"], max_rows=s["max_rows"],
                                     max_context=s["max_context"], tree=s["tree"], position=s["position"])
        if "inv_freq" in s:
            s["rope"] = A.NormRope(s["inv_freq"], s["q_weight"], s["k_weight"], eps=EPS,
                                   adjacent=c["pairs"] == "adjacent")
    return s


# ------------------------------------------------------------------ one pass

def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return {"norm_rope": _norm_rope, "attention": _attention, "fork_grow": _fork_grow, "compact": _compact,
                "keep": _keep}[s["op"]](s)


def _run_own(s):
    from plugins_b200 import attention as A
    if s["op"] == "attention":
        return A.tree_attention(s["cache"], s["layer"], s["batch"], s["q"], lse=True)
    if s["op"] in ("norm_rope", "keep"):
        q = A.qk_norm_rope(s["cache"], s["layer"], s["batch"], s["q"], s["key"], s["value"], s["rope"])
        if s["op"] == "norm_rope":
            return q, s["k"], s["v"]
        return q, s["k"], s["v"], A.cache_keep(s["cache"], s["batch"], s["path"], s["kept"])
    if s["op"] == "fork_grow":
        p, missing = A.cache_grow(s["cache"], A.cache_fork(s["cache"], s["pages"], s["parent"]), s["need"])
        return s["k"], s["v"], p.refs, p.table, p.held, p.lens, missing
    p = A.cache_compact(s["cache"], s["pages"])
    return s["k"], s["v"], p.refs, p.table, p.held, p.lens


def _slots(s):
    """Every new row's sequence, place in it, page and offset in the page."""
    start, page = s["row_start"].long(), s["k"].shape[3]
    row = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(start, row, right=True) - 1
    place = row - start[seq]
    at = s["context"].long()[seq] + place
    return seq, place, s["table"].long()[seq, at // page], at % page


def _rms_rotate(x, w, pos, s):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    t = (pos.double()[:, None] * s["inv_freq"])[:, None]
    cos, sin = t.cos().float(), t.sin().float()
    rot = 2 * s["inv_freq"].numel()
    if s["case"]["pairs"] == "adjacent":
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        r = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        r = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((r, x[..., rot:]), -1)


def _norm_rope(s):
    seq, place, page, off = _slots(s)
    pos = s["position"] if s["position"] is not None else s["context"][seq] + place
    k, v = s["k"][s["layer"]], s["v"][s["layer"]]
    k[page, :, off] = _rms_rotate(s["key"], s["k_weight"], pos, s).to(k.dtype)
    v[page, :, off] = s["value"].to(v.dtype)
    return _rms_rotate(s["q"], s["q_weight"], pos, s).to(s["q"].dtype), s["k"], s["v"]


def _attention(s):
    kc, vc = s["k"][s["layer"]], s["v"][s["layer"]]
    page, (rows, heads, dim) = kc.shape[2], s["q"].shape
    nseq, kvh = s["context"].numel(), kc.shape[1]
    seq, place, _, _ = _slots(s)
    t, n = s["max_rows"], s["max_context"]
    ids = s["table"][:, :-(-n // page)].long().clamp(min=0)
    # [seq, kv head, key, dim]
    k = kc[ids].permute(0, 2, 1, 3, 4).reshape(nseq, kvh, -1, dim)[:, :, :n].float()
    v = vc[ids].permute(0, 2, 1, 3, 4).reshape(nseq, kvh, -1, dim)[:, :, :n].float()
    q = torch.zeros((nseq, t, heads, dim), device="cuda")
    q[seq, place] = s["q"].float()
    q = q.view(nseq, t, kvh, heads // kvh, dim).permute(0, 2, 3, 1, 4).reshape(nseq, kvh, -1, dim)
    score = torch.matmul(q, k.transpose(2, 3)).view(nseq, kvh, heads // kvh, t, n).mul_(dim ** -0.5)
    key = torch.arange(n, device="cuda")
    back = key[None] - s["context"][:, None]  # a key's place among the sequence's new tokens
    if s["tree"] is None:
        see = back[:, None, :] <= torch.arange(t, device="cuda")[None, :, None]
    else:
        words = torch.zeros((nseq, t, s["tree"].shape[1]), dtype=torch.int32, device="cuda")
        words[seq, place] = s["tree"]
        bit = back.clamp(0, 32 * s["tree"].shape[1] - 1)
        word = words.gather(2, (bit >> 5)[:, None, :].expand(-1, t, -1))
        see = (back < 0)[:, None, :] | (((word >> (bit & 31)[:, None, :]) & 1) == 1)
    see &= (back < (s["row_start"][1:] - s["row_start"][:-1])[:, None])[:, None, :]
    score.masked_fill_(~see[:, None, None], -math.inf)
    m = score.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = score.sub_(m).exp_()
    z = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(nseq, kvh, -1, n), v).view(nseq, kvh, -1, t, dim)
    o = torch.where(z > 0, o / z, 0.0)
    lse = (m + z.log())[..., 0].reshape(nseq, heads, t).transpose(1, 2)[seq, place]
    o = o.reshape(nseq, heads, t, dim).transpose(1, 2)[seq, place]
    return o.to(s["q"].dtype), lse.contiguous()


def _fork_grow(s):
    # fork: row i of the result is row parent[i]; a page's references follow its rows
    parent, page = s["parent"].long(), s["k"].shape[3]
    table, held, lens = s["table"][parent].clone(), s["held"][parent], s["lens"][parent]
    more = torch.bincount(parent, minlength=s["held"].numel()).int() - 1
    valid = s["table"] >= 0
    refs = s["refs"].clone()
    refs.index_add_(0, s["table"][valid].long(), more[:, None].expand_as(s["table"])[valid])
    # grow: a shared last page that will be written is copied, then whole pages are added, the lowest free ids first
    want = (s["need"] + page - 1) // page
    extra = (want - held).clamp(min=0)
    last = table.long().gather(1, (lens // page).clamp(max=table.shape[1] - 1)[:, None].long())[:, 0]
    grows = (lens % page != 0) & (s["need"] > lens)
    at = last.clamp(min=0)
    sharers = torch.bincount(at[grows], minlength=refs.numel())[at]
    row = torch.arange(parent.numel(), device="cuda")
    first = torch.full((refs.numel(),), 1 << 30, device="cuda").scatter_reduce(0, at[grows], row[grows], "amin")[at]
    copy = grows & (refs[at] > 1) & ~((sharers == refs[at]) & (row == first))
    ask = extra + copy
    begin = ask.cumsum(0) - ask
    free = (refs == 0).nonzero()[:, 0]
    missing = (ask.sum() - free.numel()).clamp(min=0)
    if int(missing) == 0:
        src, dst, mine = at[copy], free[begin[copy]], row[copy]
        s["k"][:, dst] = s["k"][:, src]
        s["v"][:, dst] = s["v"][:, src]
        refs.index_add_(0, src, torch.full_like(src, -1, dtype=torch.int32))
        refs[dst] = 1
        table[mine, (lens // page).long()[copy]] = dst.int()
        j = torch.arange(table.shape[1], device="cuda")[None]
        new = (j >= held[:, None]) & (j < want[:, None])
        give = free[((begin + copy)[:, None] + j - held[:, None]).clamp(0, free.numel() - 1)]
        table = torch.where(new, give.int(), table)
        refs[give[new]] = 1
        held = torch.maximum(held, want)
    return s["k"], s["v"], refs, table, held, lens, missing.int()


def _compact(s):
    refs = s["refs"]
    live = refs > 0
    count = live.sum()
    page = torch.arange(refs.numel(), device="cuda")
    src, dst = (live & (page >= count)).nonzero()[:, 0], (~live & (page < count)).nonzero()[:, 0]
    to = page.clone()
    to[src] = dst
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    out = torch.where(page < count, refs, 0)
    out[dst] = refs[src]
    table = torch.where(s["table"] >= 0, to[s["table"].clamp(min=0).long()].int(), -1)
    return s["k"], s["v"], out.int(), table.int(), s["held"].clone(), s["lens"].clone()


def _keep(s):
    q = _norm_rope(s)[0]
    page = s["k"].shape[3]
    d = torch.arange(s["path"].shape[1], device="cuda")[None]
    take = d < s["kept"][:, None]
    seq = torch.arange(s["kept"].numel(), device="cuda")[:, None].expand_as(take)[take]
    a = (s["context"][:, None] + s["path"]).long()[take]
    b = (s["context"][:, None] + d).long()[take]
    table = s["table"].long()
    for pool in (s["k"], s["v"]):
        pool[:, table[seq, b // page], :, b % page] = pool[:, table[seq, a // page], :, a % page]
    return q, s["k"], s["v"], s["context"] + s["kept"]


# ------------------------------------------------------------------ the definition in 64 bits

def exact(c, seed):
    if c["op"] in ("fork_grow", "compact"):
        return None  # whole numbers and copies
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    rows, ctx = _sizes(c)
    start = [sum(rows[:b]) for b in range(len(rows))]
    table = s["table"].tolist()
    layer, page, kvh, dim, heads = s["layer"], c["page"], c["kv_heads"], c["dim"], c["heads"]

    def places(b, lo, hi):
        at = torch.arange(lo, hi, device="cuda")
        return torch.tensor(table[b], device="cuda")[at // page], at % page

    if c["op"] == "attention":
        out = torch.zeros((sum(rows), heads, dim), dtype=torch.float64, device="cuda")
        lse = torch.zeros((sum(rows), heads), dtype=torch.float64, device="cuda")
        trees = _trees(c) if c["tree"] else None
        for b, (r, x) in enumerate(zip(rows, ctx)):
            pg, of = places(b, 0, x + r)
            see = torch.ones((r, x + r), dtype=torch.bool, device="cuda")
            if trees:
                m = torch.zeros((r, r), dtype=torch.bool)
                for i, a in enumerate(trees[b]):
                    m[i, a] = True
                see[:, x:] = m.cuda()
            else:
                see[:, x:] = torch.ones((r, r), dtype=torch.bool, device="cuda").tril()
            for h in range(heads):
                kh = h // (heads // kvh)
                k, v = (t[layer][pg, kh, of].double() for t in (s["k"], s["v"]))
                q = s["q"][start[b]:start[b] + r, h].double()
                z = torch.where(see, q @ k.T / math.sqrt(dim), -math.inf)
                l = torch.logsumexp(z, 1)
                out[start[b]:start[b] + r, h] = torch.exp(z - l[:, None]) @ v
                lse[start[b]:start[b] + r, h] = l
        return out, lse

    def turned(x, w, pos):
        x, w = x.double(), w.double()
        y = x / torch.sqrt(torch.mean(x * x, -1, keepdim=True) + EPS) * w
        half = c["rot"] // 2
        i = torch.arange(half, device="cuda", dtype=torch.float64)
        angle = pos.double()[:, None, None] * THETA ** (-i * 2 / c["rot"])
        first = 2 * i.long() if c["pairs"] == "adjacent" else i.long()
        second = first + (1 if c["pairs"] == "adjacent" else half)
        z = torch.view_as_complex(torch.stack((y[..., first], y[..., second]), -1)) * torch.polar(torch.ones_like(angle), angle)
        y[..., first], y[..., second] = z.real, z.imag
        return y

    pos = torch.cat([torch.arange(x, x + r, device="cuda") for r, x in zip(rows, ctx)])
    if c["op"] == "keep":
        pos = torch.tensor([x + len(a) - 1 for x, t in zip(ctx, _trees(c)) for a in t], device="cuda")
    if s["k"].numel() > 1 << 29:
        return turned(s["q"], s["q_weight"], pos), None, None, None
    k, v = s["k"].double(), s["v"].double()
    nk = turned(s["key"], s["k_weight"], pos)
    for b, (r, x) in enumerate(zip(rows, ctx)):
        pg, of = places(b, x, x + r)
        k[layer, pg, :, of] = nk[start[b]:start[b] + r]
        v[layer, pg, :, of] = s["value"][start[b]:start[b] + r].double()
    if c["op"] == "keep":
        for b, n in enumerate(_kept(c)):
            path = max(_trees(c)[b], key=len)[:n]
            pg, of = places(b, ctx[b], ctx[b] + rows[b])
            for pool in (k, v):
                got = pool[:, pg[path], :, of[path]]
                pool[:, pg[:n], :, of[:n]] = got
    return (turned(s["q"], s["q_weight"], pos), k, v) + ((None,) if c["op"] == "keep" else ())
