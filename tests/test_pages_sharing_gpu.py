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
