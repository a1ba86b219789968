"""Pages and lengths that several rows, or several arguments, share (plugins_b200/attention.py)."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture()
def A():
    from plugins_b200 import attention
    from plugins_b200 import quant as Q
    Q.device_error(0, clear=True)
    yield attention
    assert Q.device_error(0, clear=True) == 0


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def scattered(held, seed):
    """A table of pages in a mixed order, and how many pages there are."""
    ids = list(range(sum(held) + 3))
    random.Random(seed).shuffle(ids)
    width, table, at = max(held) + 1, [], 0
    for h in held:
        table.append(ids[at:at + h] + [-1] * (width - h))
        at += h
    return table, len(ids)


@pytest.mark.parametrize("alias", ["context", "kept"])
@pytest.mark.parametrize("layers,kv_heads,dim,nseq", [(36, 8, 128, 48), (36, 8, 128, 200), (1, 1, 64, 9000)])
def test_keep_into_the_batchs_own_lengths(A, layers, kv_heads, dim, nseq, alias):
    """Many blocks per sequence, more than the GPU holds at once, and more sequences than one launch counts."""
    page, r = 16, random.Random(nseq)
    lens = [r.randrange(0, 40) for _ in range(nseq)]
    rows = [r.randrange(1, 9) for _ in range(nseq)]
    table, pages = scattered([-(-(a + b) // page) for a, b in zip(lens, rows)], nseq)
    g = torch.Generator(device="cuda").manual_seed(1)
    shape = (layers, pages, kv_heads, page, dim)
    k, v = (torch.randn(shape, generator=g, device="cuda", dtype=torch.float16) for _ in range(2))
    path = [sorted(r.sample(range(n), r.randrange(1, n + 1))) for n in rows]
    kept = [r.randrange(len(p) + 1) for p in path]
    path = i32([p + [-1] * (8 - len(p)) for p in path])
    start = [0]
    for n in rows:
        start.append(start[-1] + n)

    def keep(into):
        cache = A.KvCache(k.clone(), v.clone())
        context, count = i32(lens), i32(kept)
        batch = A.TreeBatch(i32(start), context, i32(table), max_rows=8, rows=start[-1])
        out = {"own": None, "context": context, "kept": count}[into]
        got = A.cache_keep(cache, batch, path, count, out=out)
        assert out is None or got is out
        assert got.tolist() == [a + b for a, b in zip(lens, kept)]
        return cache

    want = keep("own")
    for _ in range(3):
        got = keep(alias)
        assert torch.equal(got.k, want.k) and torch.equal(got.v, want.v)
    # and the separate output against the definition
    k2, v2 = k.clone(), v.clone()
    for s in random.Random(2).sample(range(nseq), 20):
        for d in range(kept[s]):
            a, b = lens[s] + int(path[s, d]), lens[s] + d
            for t, src in ((k2, k), (v2, v)):
                t[:, table[s][b // page], :, b % page] = src[:, table[s][a // page], :, a % page]
        for pg in table[s]:
            if pg >= 0:
                assert torch.equal(want.k[:, pg], k2[:, pg]) and torch.equal(want.v[:, pg], v2[:, pg])


# ------------------------------------------------------------------ grow

def grown(refs, table, lens, width, need, page):
    """The rule of exl3_cache_grow in plain Python -> (refs, table, copies, missing)."""
    writes = [range(n // page, min(-(-want // page), len(row))) if want > n else range(0)
              for row, n, want in zip(table, lens, need)]
    writers = {}
    for i, (row, places) in enumerate(zip(table, writes)):
        for j in places:
            writers.setdefault(row[j], []).append(i)
    free = [i for i, c in enumerate(refs) if c == 0]
    out, new, copies, asked = list(refs), [list(row) for row in table], [], 0

    def give():
        nonlocal asked
        asked += 1
        return free[asked - 1] if asked <= len(free) else 0
    for i, row in enumerate(table):
        for j in writes[i]:
            p = row[j]
            if refs[p] > 1 and not (len(writers[p]) == refs[p] and writers[p][0] == i):
                new[i][j] = give()
                out[p] -= 1
                out[new[i][j]] = 1
                if j * page < lens[i]:
                    copies.append((p, new[i][j]))
        for _ in range(len(row), min(-(-need[i] // page), width)):
            new[i].append(give())
            out[new[i][-1]] = 1
    missing = max(0, asked - len(free)) + sum(max(0, -(-n // page) - width) for n in need)
    return (refs, table, [], missing) if missing else (out, new, copies, 0)


def apart(table, refs, lens, need, page):
    """No slot a row is about to write lies in a page that anyone else holds."""
    holders = {}
    for row in table:
        for p in row:
            holders[p] = holders.get(p, 0) + 1
    for row, n, want in zip(table, lens, need):
        for at in range(n, want):
            assert holders[row[at // page]] == 1 == refs[row[at // page]]


def shared_state(nseq, page, width, seed, cut):
    """Rows forked from others that hold more pages than their tokens need, as after rejected drafts; some of them cut
    back further into what they share."""
    r = random.Random(seed)
    first = [r.randrange(0, (width - 4) * page) for _ in range(nseq)]
    first = [n // page * page if r.random() < 0.4 else n for n in first]
    held = [-(-n // page) + r.choice([0, 0, 1, 2, 3]) for n in first]
    pages = sum(held) + nseq * (width + 1)
    ids = list(range(pages))
    r.shuffle(ids)
    rows = []
    for h in held:
        rows.append(ids[:h])
        ids = ids[h:]
    parent = [r.randrange(nseq) for _ in range(nseq)]
    table = [list(rows[p]) for p in parent]
    lens = [first[p] for p in parent]
    if cut:
        lens = [r.randrange(n + 1) if r.random() < 0.3 else n for n in lens]
    refs = [0] * pages
    for row in table:
        for p in row:
            refs[p] += 1
    return refs, table, lens


def on_gpu(A, refs, table, lens, width):
    n = len(table)
    return A.PageState(i32(refs), i32([row + [-1] * (width - len(row)) for row in table]).view(n, width),
                       i32([len(row) for row in table]).view(n), i32(lens).view(n))


@pytest.mark.parametrize("nseq,page,width,add", [(2, 16, 6, 6), (2, 16, 8, 40), (9, 16, 9, 33), (40, 32, 8, 70),
                                                 (33, 64, 7, 1), (1500, 16, 8, 20), (7, 16, 200, 700)])
@pytest.mark.parametrize("cut", [False, True])
def test_a_row_grows_into_pages_of_its_own(A, nseq, page, width, add, cut):
    r = random.Random(nseq + add)
    refs, table, lens = shared_state(nseq, page, width, nseq, cut)
    need = [min(n + r.randrange(add + 1), width * page) for n in lens]
    want_refs, want, copies, missing = grown(refs, table, lens, width, need, page)
    assert missing == 0
    apart(want, want_refs, lens, need, page)
    g = torch.Generator().manual_seed(nseq)
    k, v = (torch.randn((2, len(refs), 1, page, 64), generator=g).half() for _ in range(2))
    cache = A.KvCache(k.cuda(), v.cuda())
    state = on_gpu(A, refs, table, lens, width)
    out, lacking = A.cache_grow(cache, state, i32(need))
    assert int(lacking) == 0
    got = [row[:h] for row, h in zip(out.table.tolist(), out.held.tolist())]
    got_refs = out.refs.tolist()
    apart(got, got_refs, lens, need, page)
    count = [0] * len(refs)
    for row in got:
        for p in row:
            count[p] += 1
    assert count == got_refs  # every reference is a row's
    assert got == want and got_refs == want_refs and out.lens.tolist() == lens
    for a, b in copies:
        k[:, b], v[:, b] = k[:, a], v[:, a]
    assert torch.equal(cache.k.cpu(), k) and torch.equal(cache.v.cpu(), v)
    for i, n in enumerate(lens):  # a row's tokens are where its table says, as before
        for at in range(0, n, max(1, n // 7)):
            assert torch.equal(k[:, got[i][at // page], :, at % page], k[:, table[i][at // page], :, at % page])


@pytest.mark.parametrize("tokens,tables", [(15, [[0, 1, 2], [3, 4, 2]]), (16, [[0, 1, 2], [0, 3, 2]]),
                                           (14, [[0, 1, 2], [3, 4, 2]])])
def test_pages_past_the_tokens_of_forked_rows(A, tokens, tables):
    """One row of three pages forked twice, both about to write six tokens: over a page's end and from one on."""
    cache = A.KvCache(*(torch.zeros((1, 8, 1, 16, 64), dtype=torch.float16, device="cuda") for _ in range(2)))
    state = A.cache_fork(cache, on_gpu(A, [1, 1, 1] + [0] * 5, [[0, 1, 2]], [tokens], 3), i32([0, 0]))
    out, missing = A.cache_grow(cache, state, i32([tokens + 6] * 2))
    assert int(missing) == 0 and out.table.tolist() == tables
    apart(out.table.tolist(), out.refs.tolist(), [tokens] * 2, [tokens + 6] * 2, 16)
    # one that grows alone leaves the other's pages to it
    out, missing = A.cache_grow(cache, state, i32([tokens, tokens + 6]))
    assert int(missing) == 0 and out.table[0].tolist() == [0, 1, 2]
    apart([out.table[1].tolist(), [0, 1, 2]], out.refs.tolist(), [tokens], [tokens + 6], 16)


def test_grow_that_lacks_pages_for_what_is_shared_changes_nothing(A):
    refs, table, lens, need = [2, 2, 2, 0], [[0, 1, 2], [0, 1, 2]], [15, 15], [21, 21]
    assert grown(refs, table, lens, 3, need, 16)[3] == 1
    cache = A.KvCache(*(torch.randn((1, 4, 1, 16, 64), device="cuda").half() for _ in range(2)))
    k = cache.k.clone()
    out, missing = A.cache_grow(cache, on_gpu(A, refs, table, lens, 3), i32(need))
    assert int(missing) == 1 and out.refs.tolist() == refs and out.table.tolist() == table
    assert out.held.tolist() == [3, 3] and out.lens.tolist() == lens and torch.equal(cache.k, k)


@pytest.mark.parametrize("prompt,page", [(14, 16), (15, 16), (31, 16), (29, 16), (7, 16)])
def test_a_forked_pair_that_diverges_decodes_as_unshared_rows_do(prompt, page):
    """Drafts rejected over a page's end, a fork, then two different continuations: tokens, keys and values as of two rows
    that never shared a page (the second row's copied from the first's)."""
    from plugins_b200 import quant as Q
    from plugins_b200 import tree_decode as T
    heads, kv, dim, hidden, vocab = 8, 2, 128, 512, 512
    layers = T.random_layers(2, hidden, heads, kv, dim, 1024, seed=3)
    embed = torch.randn((vocab, hidden), generator=torch.Generator("cuda").manual_seed(1), device="cuda").bfloat16()
    text = [(11 * i + 5) % vocab for i in range(prompt)]

    def run(fork):
        dec = T.TreeDecoder(layers, embed, heads, kv, dim, pages=64, page_size=page, nseq=2, max_pages=16)
        last = dec.prompt([text, text])[0]
        wrong = [(i - 1, (last + 1 + i) % vocab) for i in range(40)]  # a chain of drafts, none of them right
        got = dec.step([wrong, wrong])
        if fork:
            dec.reorder([0, 0])
        else:
            at = torch.arange(dec.lens[0], device="cuda")
            a, b = (dec.state.table[s].long()[at // page] for s in range(2))
            for t in (dec.cache.k, dec.cache.v):
                t[:, b, :, at % page] = t[:, a, :, at % page]
            assert dec.lens[0] == dec.lens[1]
        dec.last = [3, 400]
        tokens = []
        for i in range(3 * page):
            tokens.append(dec.step([[(-1, 1), (0, 2)] if i % 5 == 0 else []] * 2))
        keep = []
        for s in range(2):
            at = torch.arange(dec.lens[s], device="cuda")
            pg = dec.state.table[s].long()[at // page]
            keep.append((dec.cache.k[:, pg, :, at % page], dec.cache.v[:, pg, :, at % page]))
        table = [row[:h] for row, h in zip(dec.state.table.tolist(), dec.state.held.tolist())]
        return got[0], tokens, keep, set(table[0][prompt // page + 1:]) & set(table[1][prompt // page + 1:])

    got, tokens, keep, _ = run(False)
    got2, tokens2, keep2, both = run(True)
    assert got == got2 and tokens == tokens2 and not both
    for a, b in zip(keep, keep2):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert Q.device_error(0, clear=True) == 0


@pytest.mark.parametrize("nseq", [0, 1, 40, 4096])
def test_grow_asked_for_more_than_can_be_counted(A, nseq):
    """No rows; and rows that together lack more pages than 32 bits hold: all of them said, nothing changed."""
    cache = A.KvCache(*(torch.zeros((1, 8, 1, 16, 64), dtype=torch.float16, device="cuda") for _ in range(2)))
    refs, table = [1] + [0] * 7, [[0]] + [[]] * (nseq - 1) if nseq else []
    state = on_gpu(A, refs if nseq else [0] * 8, table, [3] + [0] * (nseq - 1) if nseq else [], 4)
    out, missing = A.cache_grow(cache, state, i32([2 ** 31 - 1] * nseq).view(nseq))
    asked = nseq * (2 ** 27 - 4) + max(0, 4 * nseq - (1 if nseq else 0) - (7 if nseq else 8))
    assert int(missing) == min(asked, 2 ** 31 - 1)
    assert out.refs.tolist() == state.refs.tolist() and out.table.tolist() == state.table.tolist()
    assert out.held.tolist() == state.held.tolist() and out.lens.tolist() == state.lens.tolist()


def test_grow_of_too_many_rows_is_refused(A):
    cache = A.KvCache(*(torch.zeros((1, 8, 1, 16, 64), dtype=torch.float16, device="cuda") for _ in range(2)))
    with pytest.raises(A.Exl3Error, match="4096"):
        A.cache_grow(cache, A.PageState.empty(cache, 4097, 2), i32([0] * 4097))


def test_a_page_without_references_is_free_to_every_call(A):
    """Counts that a host kept too low fall below zero when its rows end (the page of row 0 here): grow and compact both
    take such a page as free."""
    cache = A.KvCache(*(torch.randn((1, 6, 1, 16, 64), device="cuda").half() for _ in range(2)))
    state = A.cache_fork(cache, on_gpu(A, [0, 1, 0, 0, 1, 0], [[0], [1], [4]], [9, 9, 9], 3), i32([1, 2]))
    assert state.refs.tolist() == [-1, 1, 0, 0, 1, 0]
    grown, missing = A.cache_grow(cache, state, i32([33, 17]))
    assert int(missing) == 0 and grown.table.tolist() == [[1, 0, 2], [4, 3, -1]] and grown.refs.tolist() == [1, 1, 1, 1, 1, 0]
    k = cache.k.clone()
    packed = A.cache_compact(cache, state)
    assert packed.table.tolist() == [[1, -1, -1], [0, -1, -1]] and packed.refs.tolist() == [1, 1, 0, 0, 0, 0]
    assert torch.equal(cache.k[:, 0], k[:, 4])


@pytest.mark.parametrize("seed", range(6))
def test_chains_of_page_calls_keep_every_rows_tokens(A, seed):
    """Grow (also for more than is kept), append, keep in place, fork, compact and lengths cut back, in a random order: every
    row's tokens, in every layer, are those it was given, and no page a row grew into is another's."""
    r = random.Random(seed)
    page, layers, kv_heads, pages, width = r.choice([16, 32]), 3, 2, 200, 8
    cache = A.KvCache(*(torch.zeros((layers, pages, kv_heads, page, 64), dtype=torch.float16, device="cuda") for _ in range(2)))
    tokens, state, copy, last = [[] for _ in range(5)], A.PageState.empty(cache, 5, width), A.NormRope(None), 0
    for _ in range(60):
        what, n = r.choice(["grow", "grow", "grow", "fork", "compact", "cut"]), len(tokens)
        if what == "grow":
            rows = [min(r.choice([0, 1, r.randrange(1, 40)]), width * page - len(t)) for t in tokens]
            need = [min(len(t) + c + r.choice([0, 0, page, 50]), width * page) for t, c in zip(tokens, rows)]
            grown, missing = A.cache_grow(cache, state, i32(need))
            if int(missing) or not sum(rows):
                continue
            state = grown
            held = [row[:h] for row, h in zip(state.table.tolist(), state.held.tolist())]
            apart(held, state.refs.tolist(), [len(t) for t in tokens], need, page)
            start = [0]
            for c in rows:
                start.append(start[-1] + c)
            new = [(last + i) % 2000 for i in range(start[-1])]
            last += start[-1]
            batch = A.TreeBatch(i32(start), state.lens, state.table, max_rows=max(rows), rows=start[-1])
            x = torch.tensor(new, device="cuda").half()[:, None, None].expand(-1, kv_heads, 64).contiguous()
            for layer in range(layers):
                A.qk_norm_rope(cache, layer, batch, x, x, x + layer + 1, copy)
            path = [sorted(r.sample(range(c), r.randrange(c + 1))) for c in rows]
            deep = max(1, *map(len, path))
            A.cache_keep(cache, batch, i32([p + [-1] * (deep - len(p)) for p in path]), i32([len(p) for p in path]),
                         out=state.lens)
            for t, p, a in zip(tokens, path, start):
                t += [new[a + j] for j in p]
        elif what == "fork":
            parent = [r.randrange(-1, n) for _ in range(r.randrange(1, 9))]
            state = A.cache_fork(cache, state, i32(parent))
            tokens = [list(tokens[p]) if p >= 0 else [] for p in parent]
        elif what == "compact":
            state = A.cache_compact(cache, state)
        else:
            tokens = [t[:r.randrange(len(t) + 1)] if r.random() < 0.3 else t for t in tokens]
            state.lens.copy_(i32([len(t) for t in tokens]))
        assert state.lens.tolist() == [len(t) for t in tokens]
        for row, t in zip(state.table.cpu().long(), tokens):
            at = torch.arange(len(t))
            want = torch.tensor(t, dtype=torch.float16)[:, None, None]
            k, v = (p.cpu()[:, row[at // page], :, at % page] for p in (cache.k, cache.v))
            assert bool((k == want[..., None]).all())
            assert bool((v == (want + torch.arange(1, layers + 1).half()[:, None])[..., None]).all())
