"""The cache's page bookkeeping on the GPU (plugins_b200/attention.py) against plain Python."""
import random

import pytest
import torch

from plugins_b200 import _lib as L

pytestmark = pytest.mark.gpu


@pytest.fixture()
def A():
    from plugins_b200 import attention
    from plugins_b200 import quant as Q
    Q.device_error(0, clear=True)
    yield attention
    assert Q.device_error(0, clear=True) == 0


class Plain:
    """The page state as lists; the pool's contents as a tensor on the CPU."""

    def __init__(self, refs, table, lens, width):
        self.refs, self.table, self.lens, self.width = refs, table, lens, width

    def on(self, A):
        t = [row + [-1] * (self.width - len(row)) for row in self.table]
        i = (lambda v: torch.tensor(v, dtype=torch.int32).cuda())
        n = len(t)
        return A.PageState(i(self.refs), i(t).view(n, self.width), i([len(r) for r in self.table]).view(n), i(self.lens).view(n))

    def same(self, st):
        assert st.refs.tolist() == self.refs
        assert [r[:h] for r, h in zip(st.table.tolist(), st.held.tolist())] == self.table
        assert all(x == -1 for r, h in zip(st.table.tolist(), st.held.tolist()) for x in r[h:])
        assert st.lens.tolist() == self.lens


def state(nseq, pages, page, width, seed, longest=5):
    r = random.Random(seed)
    ids = list(range(pages))
    r.shuffle(ids)
    refs, table, lens = [0] * pages, [], []
    for _ in range(nseq):
        n = r.randrange(0, longest * page)
        held = -(-n // page) + r.randrange(2)
        row, ids = ids[:held], ids[held:]
        for p in row:
            refs[p] += 1
        table.append(row)
        lens.append(n)
    return Plain(refs, table, lens, width)


def pool(A, pages, page, seed, layers=3, kv_heads=2, dim=64, layout="hpd"):
    g = torch.Generator().manual_seed(seed)
    if layout == "hpd":
        k, v = (torch.randn((layers, pages, kv_heads, page, dim), generator=g).half() for _ in range(2))
        return A.KvCache(k.cuda(), v.cuda())
    k, v = (torch.randn((pages, layers, page, kv_heads, dim), generator=g).half() for _ in range(2))
    return A.KvCache(*(t.cuda().permute(1, 0, 3, 2, 4) for t in (k, v)))


def fork(p, parent):
    table = [list(p.table[i]) if i >= 0 else [] for i in parent]
    refs = list(p.refs)
    for i, row in enumerate(p.table):
        for x in row:
            refs[x] += parent.count(i) - 1
    return Plain(refs, table, [p.lens[i] if i >= 0 else 0 for i in parent], p.width)


def grow(p, need, page):
    """(the grown state or None, moves, missing)"""
    last = [row[n // page] if need[i] > n and n % page and n // page < len(row) else None
            for i, (row, n) in enumerate(zip(p.table, p.lens))]
    free = [i for i, c in enumerate(p.refs) if c == 0]
    refs, table, moves, asks = list(p.refs), [list(r) for r in p.table], [], 0
    for i, row in enumerate(p.table):
        want = -(-need[i] // page)
        x = last[i]
        if x is not None and p.refs[x] > 1:
            sharers = [j for j in range(len(last)) if last[j] == x]
            if not (len(sharers) == p.refs[x] and sharers[0] == i):
                if asks < len(free):
                    moves.append((x, free[asks]))
                    refs[x] -= 1
                    refs[free[asks]] = 1
                    table[i][p.lens[i] // page] = free[asks]
                asks += 1
        for _ in range(max(0, min(want, p.width) - len(row))):
            if asks < len(free):
                table[i].append(free[asks])
                refs[free[asks]] = 1
            asks += 1
    over = sum(max(0, -(-n // page) - p.width) for n in need)
    missing = max(0, asks - len(free)) + over
    return (None if missing else Plain(refs, table, p.lens, p.width)), moves, missing


@pytest.mark.parametrize("nseq,pages,parent", [
    (1, 8, [0]), (1, 8, [-1]), (1, 8, []), (3, 64, [2, 2, 0, 2, -1, 1]), (7, 300, [0, 1, 3, 3, 6]),
    (40, 1000, [(7 * i) % 41 - 1 for i in range(90)]), (2000, 20000, [(7 * i) % 2000 for i in range(1500)])])
def test_fork(A, nseq, pages, parent):
    p = state(nseq, pages, 16, 9, seed=nseq)
    cache = pool(A, pages, 16, 1, layers=1, kv_heads=1)
    k = cache.k.clone()
    out = A.cache_fork(cache, p.on(A), torch.tensor(parent, dtype=torch.int32).cuda())
    fork(p, parent).same(out)
    assert torch.equal(cache.k, k)


@pytest.mark.parametrize("layout", ["hpd", "phd"])
@pytest.mark.parametrize("nseq,pages,page,add", [(1, 8, 16, 1), (1, 8, 16, 0), (5, 90, 16, 20), (12, 300, 64, 70),
                                                 (33, 700, 32, 1), (1100, 20000, 16, 9)])
def test_grow_copies_what_is_shared(A, nseq, pages, page, add, layout):
    r = random.Random(pages)
    first = state(nseq, pages, page, 12, seed=pages)
    p = fork(first, [r.randrange(nseq) for _ in range(nseq)] if nseq > 1 else [0])
    need = [n + r.randrange(add + 1) for n in p.lens]
    cache = pool(A, pages, page, 2, layout=layout, layers=1 if nseq > 1000 else 3)
    k, v = cache.k.clone(), cache.v.clone()
    want, moves, missing = grow(p, need, page)
    assert missing == 0
    out, lacking = A.cache_grow(cache, p.on(A), torch.tensor(need, dtype=torch.int32).cuda())
    assert int(lacking) == 0
    want.same(out)
    for a, b in moves:
        k[:, b], v[:, b] = k[:, a], v[:, a]
    assert torch.equal(cache.k, k) and torch.equal(cache.v, v)


def test_all_sharers_grow_and_the_first_keeps_the_page(A):
    p = Plain([3, 2, 0, 0, 0, 1], [[0, 1], [0, 1], [0], [5]], [20, 20, 16, 3], 4)
    need = [21, 25, 17, 3]
    want, moves, missing = grow(p, need, 16)
    assert moves == [(1, 2)] and missing == 0 and want.table == [[0, 1], [0, 2], [0, 3], [5]]
    cache = pool(A, 6, 16, 3)
    k = cache.k.clone()
    out, lacking = A.cache_grow(cache, p.on(A), torch.tensor(need, dtype=torch.int32).cuda())
    want.same(out)
    assert int(lacking) == 0 and torch.equal(cache.k[:, 2], k[:, 1])


@pytest.mark.parametrize("need,what", [([100, 17], "pages"), ([16 * 5, 2], "width")])
def test_grow_that_lacks_pages_changes_nothing(A, need, what):
    p = Plain([2, 0, 0], [[0], [0]], [10, 10], 10 if what == "pages" else 2)
    cache = pool(A, 3 if what == "pages" else 3, 16, 4)
    k = cache.k.clone()
    want, _, missing = grow(p, need, 16)
    assert want is None and missing > 0
    out, lacking = A.cache_grow(cache, p.on(A), torch.tensor(need, dtype=torch.int32).cuda())
    assert int(lacking) == missing
    p.same(out)
    assert torch.equal(cache.k, k)


@pytest.mark.parametrize("layout", ["hpd", "phd"])
@pytest.mark.parametrize("nseq,pages,drop", [(1, 4, 0), (2, 16, 1), (9, 130, 4), (40, 1000, 20), (40, 300, 0),
                                             (1500, 30000, 700), (3, 9000, 3)])
def test_compact(A, nseq, pages, drop, layout):
    first = state(nseq, pages, 16, 8, seed=nseq + drop)
    p = fork(first, list(range(drop, nseq)) + ([nseq - 1] if drop < nseq else []))
    live = [i for i, c in enumerate(p.refs) if c]
    n = len(live)
    movers, holes = [i for i in live if i >= n], [i for i in range(n) if not p.refs[i]]
    to = {i: i for i in live} | dict(zip(movers, holes))
    refs = [0] * pages
    for i in live:
        refs[to[i]] = p.refs[i]
    want = Plain(refs, [[to[x] for x in row] for row in p.table], p.lens, p.width)
    cache = pool(A, pages, 16, 5, layout=layout, layers=2, kv_heads=1 if pages > 5000 else 2)
    k, v = cache.k.clone(), cache.v.clone()
    want.same(A.cache_compact(cache, p.on(A)))
    if movers:
        k[:, holes], v[:, holes] = k[:, movers], v[:, movers]
    assert torch.equal(cache.k, k) and torch.equal(cache.v, v)


@pytest.mark.parametrize("layout", ["hpd", "phd"])
@pytest.mark.parametrize("rows,lens,page,dim", [([1], [0], 16, 64), ([5, 0, 9], [3, 20, 15], 16, 64),
                                                ([40, 33, 2], [100, 1, 63], 32, 128), ([70], [9], 16, 256)])
def test_keep(A, rows, lens, page, dim, layout):
    r = random.Random(len(rows) + dim)
    held = [-(-(a + b) // page) for a, b in zip(rows, lens)]
    width = max(held) + 1
    ids = list(range(sum(held) + 2))
    r.shuffle(ids)
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-1] * (width - h))
        at += h
    cache = pool(A, len(ids), page, 6, layers=2, kv_heads=3, dim=dim, layout=layout)
    start = [sum(rows[:i]) for i in range(len(rows) + 1)]
    i32 = (lambda x: torch.tensor(x, dtype=torch.int32).cuda())
    batch = A.TreeBatch(i32(start), i32(lens), i32(table), max_rows=max(rows), rows=start[-1])
    depth = max(max(rows), 1)
    path = [sorted(r.sample(range(n), r.randrange(1, n + 1))) if n else [] for n in rows]
    kept = [r.randrange(len(p) + 1) for p in path]
    kept[0] = len(path[0])
    k, v = cache.k.clone(), cache.v.clone()
    for s, (p, c) in enumerate(zip(path, kept)):
        old = [(table[s][(lens[s] + x) // page], (lens[s] + x) % page) for x in range(rows[s])]
        for t, src in ((k, cache.k), (v, cache.v)):
            moved = [src[:, old[x][0], :, old[x][1]].clone() for x in p[:c]]
            for d, m in enumerate(moved):
                t[:, old[d][0], :, old[d][1]] = m
    out = A.cache_keep(cache, batch, i32([p + [-1] * (depth - len(p)) for p in path]).view(len(rows), depth), i32(kept))
    assert out.tolist() == [a + b for a, b in zip(lens, kept)]
    assert torch.equal(cache.k, k) and torch.equal(cache.v, v)
    out = A.cache_keep(cache, batch, None, i32(kept))
    assert out.tolist() == [a + b for a, b in zip(lens, kept)]
    assert torch.equal(cache.k, k)


def test_bad_paths_and_ids_are_recorded_not_followed(A):
    from plugins_b200 import quant as Q
    cache = pool(A, 4, 16, 7)
    k = cache.k.clone()
    i32 = (lambda x: torch.tensor(x, dtype=torch.int32).cuda())
    batch = A.TreeBatch(i32([0, 4]), i32([3]), i32([[1, 2]]), max_rows=4, rows=4)
    for path, kept in (([[2, 1]], [2]), ([[1, 4]], [2]), ([[0, 1]], [3]), ([[0, 1]], [-1])):
        assert A.cache_keep(cache, batch, i32(path), i32(kept)).tolist() == [3]
        assert Q.device_error(0, clear=True) & L.ERR_BAD_SHAPE
    assert torch.equal(cache.k, k)
    st = A.PageState(i32([0, 1, 0, 0]), i32([[1, -1], [9, -1]]), i32([1, 1]), i32([5, 5]))
    A.cache_fork(cache, st, i32([0, 7]))
    assert Q.device_error(0, clear=True) & L.ERR_BAD_SHAPE
    A.cache_compact(cache, st)
    assert Q.device_error(0, clear=True) & L.ERR_BAD_SHAPE
    A.cache_grow(cache, st, i32([6, 6]))
    assert Q.device_error(0, clear=True) & L.ERR_BAD_SHAPE
