"""What ends a decode step over a paged key/value cache and keeps the cache inside its budget, as measured work.

Three operators of :mod:`plugins_b200.attention`:

* ``draft_verify`` -- which drafted tokens of each sequence's tree stay, by the target's probabilities and given random
  numbers, and the token that follows them;
* ``attention_weight`` -- how much every cached token was attended to, accumulated over steps;
* ``cache_evict`` -- of each row, layer and kv head the heaviest tokens stay, moved together; the other pages are freed.

The plain forms are elementary torch operations: in 64 bits for the probabilities, whose cumulative sums have borders, in 32
for the attention's weights.
"""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
LOG2E = 1.4426950408889634


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one sequence, no drafts: sampling the next token, the smallest call
        dict(name="verify_token", op="verify", nseq=1, rows_lo=1, rows_hi=1, back=1, vocab=32000, dtype="f32", draft="",
             temps="warm"),
        # a small batch's chains of five drafts with the drafter's own probabilities, an odd vocabulary
        dict(name="verify_chains_8x6", op="verify", nseq=8, rows_lo=4, rows_hi=6, back=1, vocab=65537, dtype="bf16",
             draft="f16", temps="warm"),
        # 32 sequences' 16-token trees of a drafter without probabilities, a quarter of them greedy
        dict(name="verify_trees_32x16", op="verify", nseq=32, rows_lo=16, rows_hi=16, back=4, vocab=131072, dtype="bf16",
             draft="", temps="mixed"),
        # the largest: 64 sequences' ragged trees with the drafter's probabilities, 32-bit logits
        dict(name="verify_trees_64x17_q", op="verify", nseq=64, rows_lo=9, rows_hi=17, back=3, vocab=128000, dtype="f32",
             draft="bf16", temps="mixed"),
        # one sequence, one token, a short chat: latency
        dict(name="weight_token_short", op="weight", nseq=1, rows_lo=1, rows_hi=1, ctx_lo=301, ctx_hi=301, heads=32,
             kv_heads=8, dim=128, page=16, dtype="f16", tree=False, decay=1.0),
        # a batch of 32 decoding over ragged contexts: the bandwidth-bound middle
        dict(name="weight_decode_32", op="weight", nseq=32, rows_lo=1, rows_hi=1, ctx_lo=1500, ctx_hi=9001, heads=32,
             kv_heads=8, dim=128, page=64, dtype="bf16", tree=False, decay=0.99),
        # wide heads, ragged drafted trees over long contexts
        dict(name="weight_trees_d256", op="weight", nseq=9, rows_lo=5, rows_hi=17, ctx_lo=6007, ctx_hi=16301, heads=16,
             kv_heads=8, dim=256, page=128, dtype="f16", tree=True, decay=0.9),
        # a prompt's second 4096-row chunk, causal: the largest, bound by exponentials and products
        dict(name="weight_prompt_4096", op="weight", nseq=1, rows_lo=4096, rows_hi=4096, ctx_lo=4096, ctx_hi=4096, heads=32,
             kv_heads=8, dim=128, page=64, dtype="bf16", tree=False, decay=1.0),
        # one conversation cut to a quarter, two layers: the smallest call
        dict(name="evict_one", op="evict", nseq=1, nout=1, layers=2, ctx_lo=1001, ctx_hi=1001, budget_lo=250, budget_hi=250,
             sink=4, recent=32, kv_heads=8, dim=128, page=16, dtype="bf16", spare=8),
        # a serving batch over 36 layers, some rows within their budget
        dict(name="evict_ragged_36", op="evict", nseq=16, nout=16, layers=36, ctx_lo=300, ctx_hi=1300, budget_lo=400,
             budget_hi=517, sink=4, recent=64, kv_heads=8, dim=128, page=16, dtype="bf16", spare=64),
        # ten conversations forked to twenty rows: what they share is copied, not overwritten
        dict(name="evict_forked", op="evict", nseq=10, nout=20, layers=12, ctx_lo=900, ctx_hi=4001, budget_lo=511,
             budget_hi=1030, sink=1, recent=128, kv_heads=4, dim=256, page=64, dtype="f16", spare=400),
        # four long contexts cut to 4096 tokens
        dict(name="evict_long", op="evict", nseq=4, nout=4, layers=6, ctx_lo=30011, ctx_hi=40000, budget_lo=4096,
             budget_hi=4096, sink=4, recent=512, kv_heads=8, dim=128, page=64, dtype="bf16", spare=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        most, held = {"verify": (9.6e7, 6.5e8), "weight": (4.1e8, 9e8), "evict": (1.2e9, 3.5e9)}[c["op"]]
        if w["bytes"] < most and w["flops"] < 2e11 and _held_bytes(c) < held:  # at most the largest listed cases
            return c


def _held_bytes(c):
    """What a state holds on the device."""
    if c["op"] == "verify":
        return sum(_sizes(c)[0]) * c["vocab"] * (SIZE[c["dtype"]] + (SIZE[c["draft"]] if c["draft"] else 0))
    tokens = sum(_pages_of(x + r, c["page"]) for x, r in zip(_sizes(c)[1], _sizes(c)[0])) + c.get("spare", 0)
    return tokens * c["page"] * c["kv_heads"] * c["dim"] * 4 * c.get("layers", 1)


def _draw(rng):
    op = rng.choice(["verify", "weight", "evict"])
    dtype = rng.choice(["f16", "bf16"])
    page = rng.choice([16, 32, 64, 128])
    if op == "verify":
        rows = _log(rng, 1, 33)
        return dict(op=op, nseq=_log(rng, 1, 64), rows_lo=max(1, rows // 2), rows_hi=rows, back=rng.choice([1, 2, 4, 8]),
                    vocab=_log(rng, 1000, 160000), dtype=rng.choice(["f16", "bf16", "f32"]),
                    draft=rng.choice(["", "f16", "bf16", "f32"]), temps=rng.choice(["warm", "mixed"]))
    if op == "weight":
        heads, kv_heads, dim = rng.choice([(32, 8, 128), (16, 8, 256), (16, 16, 128), (24, 4, 128), (8, 1, 64),
                                           (10, 2, 128)])
        kind = rng.choice(["token", "tree", "prompt"])
        rows = 1 if kind == "token" else _log(rng, 2, 64) if kind == "tree" else _log(rng, 65, 3000)
        nseq = _log(rng, 1, 40) if kind != "prompt" else _log(rng, 1, 3)
        ctx = _log(rng, 1, 16000) if kind != "prompt" else rng.choice([0, _log(rng, 1, 4000)])
        return dict(op=op, nseq=nseq, rows_lo=max(1, rows // 2), rows_hi=rows, ctx_lo=ctx // 3, ctx_hi=ctx, heads=heads,
                    kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, tree=kind == "tree",
                    decay=rng.choice([1.0, 0.98, 0.5]))
    kv_heads, dim = rng.choice([(8, 128), (8, 256), (4, 128), (1, 64), (2, 128)])
    layers, ctx, nseq = rng.choice([1, 3, 12, 36]), _log(rng, 40, 40000), _log(rng, 1, 20)
    budget = max(1, int(ctx * rng.uniform(0.05, 1.1)))
    return dict(op=op, nseq=nseq, nout=nseq + rng.choice([0, 0, rng.randrange(0, nseq + 1)]), layers=layers,
                ctx_lo=max(1, int(ctx * rng.uniform(0.2, 1))), ctx_hi=ctx, budget_lo=max(1, budget // 2), budget_hi=budget,
                sink=rng.choice([0, 1, 4]), recent=rng.randrange(0, budget // 3 + 2), kv_heads=kv_heads, dim=dim, page=page,
                dtype=dtype, spare=rng.randrange(0, 40))


def _spread(lo, hi, n):
    """n whole numbers over [lo, hi], the ends among them, in a mixed order; the same for the same case."""
    if n == 1:
        return [hi]
    v = [lo + (hi - lo) * i // (n - 1) for i in range(n)]
    random.Random(n).shuffle(v)
    return v


def _sizes(c):
    rows = _spread(c["rows_lo"], c["rows_hi"], c["nseq"]) if "rows_lo" in c else [0] * c["nseq"]
    return rows, _spread(c["ctx_lo"], c["ctx_hi"], c["nseq"])[::-1] if "ctx_lo" in c else [0] * c["nseq"]


def _parents(c):
    """Each sequence's tree: every row's parent, one of the `back` rows before it (-1: row 0, the sequence's last token)."""
    out = []
    for b, n in enumerate(_sizes(c)[0]):
        r = random.Random(1000 * b + n)
        out.append([r.randrange(max(0, i - c.get("back", 6)), i) if i else -1 for i in range(n)])
    return out


def _depth(parents):
    deep = []
    for p in parents:
        deep.append(deep[p] + 1 if p >= 0 else 1)
    return max(deep)


def _ancestors(parents):
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if p >= 0 else []) + [i])
    return out


def _pages_of(tokens, page):
    return -(-tokens // page)


def work(c):
    rows, ctx = _sizes(c)
    if c["op"] == "verify":
        # The rows on the accepted path, read once. About six drafts in ten are accepted, so a path visits 1 / (1 - 0.6)
        # rows at most; where it ends the drafter's probabilities of that row are read too.
        visited = sum((1 - 0.6 ** _depth(p)) / 0.4 for p in _parents(c))
        ends = sum(1 for n in rows if n > 1)
        b = c["vocab"] * (visited * SIZE[c["dtype"]] + (ends * SIZE[c["draft"]] if c["draft"] else 0))
        return {"bytes": b + 16 * sum(rows), "flops": 8 * visited * c["vocab"]}
    if c["op"] == "weight":
        seen = sum(r + x for r, x in zip(rows, ctx))
        if c["tree"]:
            pairs = sum(r * x for r, x in zip(rows, ctx)) + sum(len(a) for p in _parents(c) for a in _ancestors(p))
        else:
            pairs = sum(r * x + r * (r + 1) // 2 for r, x in zip(rows, ctx))
        es = SIZE[c["dtype"]]
        return {"bytes": seen * c["kv_heads"] * (c["dim"] * es + 8) + sum(rows) * c["heads"] * (c["dim"] * es + 4),
                "flops": 2 * c["dim"] * c["heads"] * pairs}
    # the weights of rows that are cut read once; of what stays, all that leaves its slot read and written once
    p = _plan(c)
    cut = [(n, k) for n, k in zip(p["lens"], p["keep"]) if n > k]
    moved = sum(min(k, n - k) * 0.9 for n, k in cut)
    per = 2 * c["dim"] * SIZE[c["dtype"]] + 4
    return {"bytes": c["layers"] * c["kv_heads"] * (4 * sum(n for n, _ in cut) + 2 * per * moved), "flops": 0}


def _plan(c):
    """The page state of an evict case: what a server's bookkeeping holds (ids in a mixed order), rows beyond `nseq` forks of
    earlier ones."""
    ctx, page = _sizes(c)[1], c["page"]
    parent = [i if i < c["nseq"] else (7 * i) % c["nseq"] for i in range(c["nout"])]
    held = [_pages_of(x, page) for x in ctx]
    budget = _spread(c["budget_lo"], c["budget_hi"], c["nout"])
    lens = [ctx[p] for p in parent]
    keep = [min(n, max(b, c["sink"] + c["recent"])) for n, b in zip(lens, budget)]
    extra = sum(_pages_of(keep[i], page) for i in range(c["nout"]) if parent.count(parent[i]) > 1)  # may be copied
    pages = sum(held) + extra + c["spare"]
    ids = list(range(pages))
    random.Random(pages).shuffle(ids)
    table, refs, at, width = [], [0] * pages, 0, max(held) + 1
    for h in held:
        table.append(ids[at:at + h] + [-1] * (width - h))
        at += h
    for p in parent:
        for i in table[p][:held[p]]:
            refs[i] += 1
    return dict(pages=pages, refs=refs, table=[table[p] for p in parent], held=[held[p] for p in parent], lens=lens,
                budget=budget, keep=keep, width=width)


# ------------------------------------------------------------------ inputs

def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype).cuda()


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c, "op": c["op"]}
    {"verify": _prepare_verify, "weight": _prepare_weight, "evict": _prepare_evict}[c["op"]](c, s, g, seed)
    if own:
        from plugins_b200 import attention as A
        if "refs" in s:
            s["pages"] = A.PageState(s["refs"], s["table"], s["held"], s["lens"])
        else:
            s["batch"] = A.TreeBatch(s["row_start"], s["context"], s["table"], max_rows=s["max_rows"], rows=s["rows"],
                                     max_context=s["max_context"], tree=s["tree"])
        s["cache"] = A.KvCache(s["k"], s["v"])
    return s


def _batch(c, s, seed):
    rows, ctx = _sizes(c)
    page = c.get("page", 16)
    held = [_pages_of(r + x, page) for r, x in zip(rows, ctx)]
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
    s |= dict(row_start=_ints(start), context=_ints(ctx), table=_ints(table), rows=start[-1], max_rows=max(rows),
              max_context=max(r + x for r, x in zip(rows, ctx)), tree=None)
    return start, pages


def _prepare_verify(c, s, g, seed):
    """Logits with a handful of likely tokens over a broad tail, and drafts that are mostly among the likely ones."""
    start, pages = _batch(c, s, seed)
    n, vocab, dt = s["rows"], c["vocab"], DTYPES[c["dtype"]]
    s["k"], s["v"] = (torch.zeros((1, pages, 1, 16, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    x = torch.randn((n, vocab), generator=g, device="cuda").mul_(2)
    top = torch.tensor([0.9, 0.2, -0.5, -1.2], device="cuda") + math.log(vocab) + 2
    x.scatter_(1, torch.randint(vocab, (n, 4), generator=g, device="cuda"), top.expand(n, 4))
    parents, temps = _parents(c), {"warm": [0.8], "mixed": [0.7, 1.0, 0.0, 1.25]}[c["temps"]]
    flat = [start[b] + p if p >= 0 else -1 for b, t in enumerate(parents) for p in t]
    of = _ints(flat, torch.int64).clamp(min=0)
    s["logits"] = x.to(dt)
    s["draft"] = None
    if c["draft"]:  # another model's view of the same rows
        y = x.mul_(0.9).add_(torch.randn(x.shape, generator=g, device="cuda"), alpha=0.4)
        q = torch.softmax(y, 1)
        s["draft"] = q.to(DTYPES[c["draft"]])
        y = y[of]
    else:
        y = x.mul_(1.5)[of]  # its likeliest continuations
    y -= torch.empty_like(y).exponential_(generator=g).log_()
    s["tokens"] = y.argmax(1).int()
    s["parent"] = _ints([p for t in parents for p in t])
    s["uniform"] = torch.rand((n, 2), generator=g, device="cuda")
    s["temperature"] = torch.tensor([temps[b % len(temps)] for b in range(c["nseq"])], device="cuda")
    s["depth"] = max(map(_depth, parents))
    kids = [[] for _ in range(n)]
    for r, a in enumerate(flat):
        if a >= 0:
            kids[a].append(r)
    most = max(1, max(map(len, kids)))
    s["kids"] = _ints([k + [-1] * (most - len(k)) for k in kids], torch.int64)


def _prepare_weight(c, s, g, seed):
    start, pages = _batch(c, s, seed)
    dt, n, h, kh, d = DTYPES[c["dtype"]], start[-1], c["heads"], c["kv_heads"], c["dim"]
    s["layer"] = 0
    s["k"], s["v"] = (torch.randn((1, pages, kh, c["page"], d), generator=g, device="cuda", dtype=dt) for _ in range(2))
    # one projection's q|k|v rows: the queries are a view into them
    s["q"] = torch.randn((n, (h + 2 * kh) * d), generator=g, device="cuda").to(dt)[:, :h * d].unflatten(1, (h, d))
    if c["tree"]:
        words = -(-s["max_rows"] // 32)
        bits = [[sum(1 << (j - 32 * w) for j in a if j // 32 == w) for w in range(words)]
                for p in _parents(c) for a in _ancestors(p)]
        s["tree"] = _ints([[x - (1 << 32) if x >> 31 else x for x in r] for r in bits])
    s["weight"] = torch.rand((1, c["nseq"], kh, s["max_context"] + 7), generator=g, device="cuda").mul_(0.01)
    score, see, seq, place = _scores(s)  # the attention's log-sum-exp, which its call returns
    m = score.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    lse = (m + score.sub_(m).exp_().sum(-1, keepdim=True).log())[..., 0]
    s["lse"] = lse.reshape(c["nseq"], h, -1).transpose(1, 2)[seq, place].contiguous()


def _prepare_evict(c, s, g, seed):
    p, dt = _plan(c), DTYPES[c["dtype"]]
    shape = (c["layers"], p["pages"], c["kv_heads"], c["page"], c["dim"])
    s["k"], s["v"] = (torch.empty(shape, dtype=dt, device="cuda").normal_(generator=g) for _ in range(2))
    s |= dict(refs=_ints(p["refs"]), table=_ints(p["table"]), held=_ints(p["held"]), lens=_ints(p["lens"]),
              budget=_ints(p["budget"]))
    # a few tokens hold most of the weight; a tail was never attended to at all
    w = torch.randn((c["layers"], c["nout"], c["kv_heads"], max(p["lens"]) + 9), generator=g, device="cuda").mul_(2).exp_()
    s["weight"] = torch.where(w < 0.3, 0.0, w)
    s["after"] = torch.zeros_like(w)
    s["most"] = max(p["keep"])


# ------------------------------------------------------------------ one pass

def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return {"verify": _verify, "weight": _weight, "evict": _evict}[s["op"]](s)


def _run_own(s):
    from plugins_b200 import attention as A
    c = s["case"]
    if s["op"] == "verify":
        return A.draft_verify(s["cache"], s["batch"], s["logits"], s["tokens"], s["parent"], s["uniform"],
                              temperature=s["temperature"], draft=s["draft"], depth=s["depth"])
    if s["op"] == "weight":
        return A.attention_weight(s["cache"], s["layer"], s["batch"], s["q"], s["lse"], s["weight"][s["layer"]],
                                  decay=c["decay"])
    p, missing = A.cache_evict(s["cache"], s["pages"], s["weight"], s["budget"], sink=c["sink"], recent=c["recent"],
                               weight_out=s["after"])
    return s["k"], s["v"], s["after"], p.refs, p.table, p.held, p.lens, missing


def _verify(s):
    nseq, (rows, vocab) = s["context"].numel(), s["logits"].shape
    at = s["row_start"][:-1].long()
    some = s["row_start"][1:] > s["row_start"][:-1]
    alive, every = some, torch.arange(nseq, device="cuda")
    temp = s["temperature"].double()[:, None]
    greedy = temp[:, 0] == 0
    path = torch.full((nseq, s["depth"]), -1, dtype=torch.int32, device="cuda")
    kept, end = torch.zeros_like(at), torch.zeros((nseq, vocab), dtype=torch.float64, device="cuda")
    last = at.clone()
    for d in range(s["depth"]):
        node = at.clamp(max=rows - 1)
        path[:, d] = torch.where(alive, at - s["row_start"][:-1], -1).int()
        kept = kept + alive
        last = torch.where(alive, node, last)
        x = s["logits"][node].double()
        x = x - x.amax(1, keepdim=True)
        z = torch.where(greedy[:, None], 0.0, x / temp * LOG2E)
        p = torch.where(z >= -100, torch.exp2(z), 0.0)
        one = torch.zeros_like(p).scatter_(1, x.argmax(1, keepdim=True), 1.0)
        p = torch.where(greedy[:, None], one, p / p.sum(1, keepdim=True))
        r, z = p, torch.ones(nseq, dtype=torch.float64, device="cuda")
        on = torch.zeros_like(alive)
        for j in range(s["kids"].shape[1] if d + 1 < s["depth"] else 0):
            kid = s["kids"][node, j]
            asks = alive & (kid >= 0) & ~on
            tok = s["tokens"][kid.clamp(min=0)].long()
            q = torch.zeros_like(p).scatter_(1, tok[:, None], 1.0)
            if s["draft"] is not None:
                q = torch.where(greedy[:, None], q, s["draft"][node].double())
            yes = asks & (s["uniform"][kid.clamp(min=0), 0].double() * q[every, tok] * z < r[every, tok])
            less = (r - z[:, None] * q).clamp(min=0)
            less = torch.where(less.sum(1, keepdim=True) > 0, less, p)
            r = torch.where((asks & ~yes)[:, None], less, r)
            z = r.sum(1)
            on = on | yes
            at = torch.where(yes, kid, at)
        end = torch.where((alive & ~on)[:, None], r, end)
        alive = alive & on
    total = end.sum(1, keepdim=True)
    over = end.cumsum(1) > s["uniform"][last.clamp(max=rows - 1), 1].double()[:, None] * total
    final = (end > 0).int().mul_(torch.arange(1, vocab + 1, device="cuda")[None]).amax(1) - 1  # the last possible token
    token = torch.where(over.any(1), over.int().argmax(1), final)
    return path, kept.int(), torch.where(some, token, -1).int()


def _scores(s):
    """Every row's scaled scores over its sequence's slots, -inf where it does not see them, and where its row lies."""
    c = s["case"]
    kc = s["k"][s["layer"]]
    page, (rows, heads, dim) = kc.shape[2], s["q"].shape
    nseq, kvh, start = s["context"].numel(), kc.shape[1], s["row_start"].long()
    row = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(start, row, right=True) - 1
    place = row - start[seq]
    t, n = s["max_rows"], s["max_context"]
    ids = s["table"][:, :-(-n // page)].long().clamp(min=0)
    k = kc[ids].permute(0, 2, 1, 3, 4).reshape(nseq, kvh, -1, dim)[:, :, :n].float()
    q = torch.zeros((nseq, t, heads, dim), device="cuda")
    q[seq, place] = s["q"].float()
    q = q.view(nseq, t, kvh, heads // kvh, dim).permute(0, 2, 3, 1, 4).reshape(nseq, kvh, -1, dim)
    score = torch.matmul(q, k.transpose(2, 3)).view(nseq, kvh, heads // kvh, t, n).mul_(dim ** -0.5)
    back = torch.arange(n, device="cuda")[None] - s["context"][:, None]  # a slot's place among the new tokens
    if s["tree"] is None:
        see = back[:, None, :] <= torch.arange(t, device="cuda")[None, :, None]
    else:
        words = torch.zeros((nseq, t, s["tree"].shape[1]), dtype=torch.int32, device="cuda")
        words[seq, place] = s["tree"]
        bit = back.clamp(0, 32 * s["tree"].shape[1] - 1)
        word = words.gather(2, (bit >> 5)[:, None, :].expand(-1, t, -1))
        see = (back < 0)[:, None, :] | (((word >> (bit & 31)[:, None, :]) & 1) == 1)
    see &= (back < (s["row_start"][1:] - s["row_start"][:-1])[:, None])[:, None, :]
    return score.masked_fill_(~see[:, None, None], -math.inf), back, seq, place


def _weight(s):
    score, back, seq, place = _scores(s)
    nseq, kvh, group, t, n = score.shape
    lse = torch.full((nseq, t, kvh * group), math.inf, device="cuda")  # (a row that is not there, or sees nothing, adds nothing)
    lse[seq, place] = torch.where(s["lse"] == -math.inf, math.inf, s["lse"])
    score.sub_(lse.transpose(1, 2).reshape(nseq, kvh, group, t, 1)).exp_()
    got = score.sum((2, 3))
    w = s["weight"][s["layer"]]
    old = torch.where(back < 0, s["case"]["decay"], 0.0)[:, None] * w[..., :n]
    rows = (s["row_start"][1:] - s["row_start"][:-1])[:, None]
    inside = ((back < rows) & (rows > 0))[:, None]
    w[..., :n] = torch.where(inside, old + got, w[..., :n])
    return w


def _evict(s):
    c, page, pages = s["case"], s["case"]["page"], s["refs"].numel()
    lens, table = s["lens"], s["table"].long()
    keep = torch.minimum(lens, s["budget"].clamp(min=c["sink"] + c["recent"]))
    cut = lens > keep
    held = torch.where(cut, (keep + page - 1) // page, s["held"])
    # pages: those a cut row shares are replaced by free ones, those past its tokens given back
    j = torch.arange(table.shape[1], device="cuda")[None]
    mine = table.clamp(min=0)
    used = j < s["held"][:, None]
    stays = cut[:, None] & (j < held[:, None])
    copied = stays & (s["refs"][mine] > 1)
    free = (s["refs"] == 0).nonzero()[:, 0]
    missing = (copied.sum() - free.numel()).clamp(min=0)
    refs = s["refs"].clone()
    leaves = copied | (cut[:, None] & used & ~stays)
    refs.index_add_(0, mine[leaves], torch.full_like(mine[leaves], -1, dtype=torch.int32))
    new = mine.clone()
    new[copied] = free[:copied.sum()]
    refs[new[copied]] = 1
    new = torch.where(j < held[:, None], new, -1)
    # tokens: of the slots, the first, the last, then the heaviest of the others, as they stood in order
    w, n = s["weight"], s["weight"].shape[3]
    slot = torch.arange(n, device="cuda")
    always = (slot < c["sink"]) | (slot >= (lens - c["recent"])[:, None])
    past = slot >= lens[:, None]
    level = torch.where(always[:, None], 2.0, 1.0).masked_fill_(past[:, None], 0.0).expand(w.shape)
    order = torch.where(past[:, None], 0.0, w).sort(dim=-1, descending=True, stable=True)[1]
    order = order.gather(-1, level.gather(-1, order).sort(dim=-1, descending=True, stable=True)[1])[..., :s["most"]]
    src = torch.where(slot[:s["most"]] < keep[:, None, None], order, n).sort(-1)[0]
    at = (src < n) & cut[:, None, None]
    la, row, head, dst = at.nonzero(as_tuple=True)
    src = src[at]
    for pool in (s["k"], s["v"]):
        pool[la, new[row, dst // page], head, dst % page] = pool[la, mine[row, src // page], head, src % page]
    after = s["after"]
    after[la, row, head, dst] = w[la, row, head, src]
    whole = (slot < lens[:, None]) & ~cut[:, None]
    after[:] = torch.where(whole[:, None], w, after)
    return s["k"], s["v"], after, refs, new.int(), held, keep, missing.int()


# ------------------------------------------------------------------ the definition in 64 bits

def exact(c, seed):
    if c["op"] != "weight":
        return None  # whole numbers and copies
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    (rows, ctx), page, heads, kvh, dim = _sizes(c), c["page"], c["heads"], c["kv_heads"], c["dim"]
    start = [sum(rows[:b]) for b in range(len(rows))]
    out = s["weight"][0].double()
    for b, (r, x) in enumerate(zip(rows, ctx)):
        at = torch.arange(x + r, device="cuda")
        pg = s["table"][b].long()[at // page]
        see = torch.ones((r, x + r), dtype=torch.bool, device="cuda")
        see[:, x:] = see[:, x:].tril()
        if c["tree"]:
            m = torch.zeros((r, r), dtype=torch.bool)
            for i, a in enumerate(_ancestors(_parents(c)[b])):
                m[i, a] = True
            see[:, x:] = m.cuda()
        for kh in range(kvh):
            k = s["k"][0][pg, kh, at % page].double()
            w = torch.cat((out[b, kh, :x] * c["decay"], torch.zeros(r, dtype=torch.float64, device="cuda")))
            for h in range(kh * (heads // kvh), (kh + 1) * (heads // kvh)):
                q = s["q"][start[b]:start[b] + r, h].double()
                e = torch.exp(q @ k.T / math.sqrt(dim) - s["lse"][start[b]:start[b] + r, h].double()[:, None])
                w += torch.where(see, e, 0.0).sum(0)
            out[b, kh, :x + r] = w
    return out
