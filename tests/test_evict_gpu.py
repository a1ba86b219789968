"""exl3_cache_evict on the GPU against slot-by-slot eviction in plain Python (tests/evict_ref.py): whole numbers and copies,
so everything has to be the same."""
import math
import random

import pytest
import torch

import evict_ref as E
from test_pages_gpu import A  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


class Case:
    """Rows of `lens` tokens; rows past the first len(lens) are forks of `parents`."""

    def __init__(self, lens, budget, sink=0, recent=0, layers=2, kv_heads=2, dim=64, page=16, dtype=torch.float16, parents=(),
                 spare=40, layout="hpd", seed=0, extra=0, slots=None, weight=None):
        r = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        held = [-(-n // page) + extra for n in lens]
        self.pages = sum(held) + spare
        ids = list(range(self.pages))
        r.shuffle(ids)
        rows, at = [], 0
        for h in held:
            rows.append(ids[at:at + h])
            at += h
        order = list(range(len(lens))) + list(parents)
        self.table = [list(rows[i]) for i in order]
        self.held = [held[i] for i in order]
        self.lens = [lens[i] for i in order]
        self.refs = [0] * self.pages
        for t in self.table:
            for p in t:
                self.refs[p] += 1
        self.width = max(self.held + [1]) + 1
        self.budget = budget if isinstance(budget, list) else [budget] * len(order)
        self.sink, self.recent, self.layout = sink, recent, layout
        shape = (layers, self.pages, kv_heads, page, dim)
        self.k, self.v = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
        n = max(self.lens + [1]) + 3 if slots is None else slots
        w = torch.randn((layers, len(order), kv_heads, n), generator=g).mul(2).exp()
        self.w = torch.where(w < 0.3, 0.0, w) if weight is None else weight(w)

    def state(self, A):
        i = (lambda v: torch.tensor(v, dtype=torch.int32).cuda())
        n = len(self.lens)
        t = [row + [-1] * (self.width - len(row)) for row in self.table]
        return A.PageState(i(self.refs), i(t).view(n, self.width), i(self.held).view(n), i(self.lens).view(n))

    def cache(self, A):
        if self.layout == "hpd":
            return A.KvCache(self.k.cuda(), self.v.cuda())
        return A.KvCache(*(t.permute(1, 0, 3, 2, 4).contiguous().cuda().permute(1, 0, 3, 2, 4) for t in (self.k, self.v)))

    def want(self, after=None):
        return E.evict(self.k, self.v, self.w, self.refs, self.table, self.held, self.lens, self.budget, self.sink, self.recent,
                       after)

    def check(self, A, in_place=True):
        cache, st, w = self.cache(A), self.state(A), self.w.cuda()
        budget = torch.tensor(self.budget, dtype=torch.int32).cuda()
        out = None if in_place else torch.full_like(w, -7.0)
        new, missing = A.cache_evict(cache, st, w, budget, sink=self.sink, recent=self.recent, weight_out=out)
        k, v, w2, refs, table, held, lens, lacking = self.want(None if in_place else torch.full_like(self.w, -7.0))
        assert int(missing) == lacking
        assert new.lens.tolist() == lens and new.held.tolist() == held and new.refs.tolist() == refs
        for got, row in zip(new.table.tolist(), table):
            assert got == [p for p in row if p >= 0] + [-1] * (self.width - sum(p >= 0 for p in row))
        bits = (lambda t: t.cpu().contiguous().view({2: torch.int16, 4: torch.int32}[t.element_size()]))  # (NaN compares too)
        if not in_place:
            assert torch.equal(bits(w), bits(self.w))
        assert torch.equal(bits(w if in_place else out), bits(w2))
        assert torch.equal(bits(cache.k), bits(k)) and torch.equal(bits(cache.v), bits(v))
        # what was read stays as it was
        assert st.refs.tolist() == self.refs and st.lens.tolist() == self.lens and st.held.tolist() == self.held
        return new


@pytest.mark.parametrize("lens", [[1], [2], [16], [17], [100, 1, 0, 33], [511, 512, 513], [2047, 2048, 2049], [4500, 3, 2100]])
@pytest.mark.parametrize("budget", [0, 1, 7, 64, 500])
@pytest.mark.parametrize("in_place", [True, False])
def test_lengths_and_budgets(A, lens, budget, in_place):
    Case(lens, budget, sink=1, recent=3, seed=len(lens) + budget).check(A, in_place)


@pytest.mark.parametrize("sink,recent", [(0, 0), (0, 1), (1, 0), (4, 60), (100, 100), (0, 1000), (1000, 0), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_what_always_stays(A, sink, recent):
    Case([300, 90, 250], [80, 20, 200], sink=sink, recent=recent, seed=5).check(A)


@pytest.mark.parametrize("dim,page,dtype,layout", [(64, 16, torch.float16, "hpd"), (128, 32, torch.bfloat16, "phd"),
                                                   (256, 128, torch.float16, "hpd"), (128, 256, torch.bfloat16, "hpd"),
                                                   (64, 64, torch.bfloat16, "phd")])
def test_layouts(A, dim, page, dtype, layout):
    Case([700, 130, 55], [300, 129, 60], sink=2, recent=16, dim=dim, page=page, dtype=dtype, layout=layout, layers=3,
         kv_heads=3, seed=dim + page).check(A)


def test_equal_weights_keep_the_lowest_slots(A):
    for value in (0.0, 1.0, -1.0, math.inf, math.nan):
        Case([500, 2500], 100, sink=1, recent=5, weight=lambda w: torch.full_like(w, value)).check(A)
    few = (lambda w: (w * 2).floor().clamp(0, 3))
    Case([900, 5000], [333, 1500], weight=few, seed=2).check(A)


def test_infinities_nan_negative_and_tiny_weights(A):
    def odd(w):
        g = torch.Generator().manual_seed(9)
        pick = torch.randint(0, 10, w.shape, generator=g)
        for i, x in enumerate((math.nan, math.inf, -math.inf, -0.0, 0.0, 1e-45, -1e-45)):
            w = torch.where(pick == i, x, w)
        return torch.where(pick == 8, -w, w)
    Case([800, 3000, 77], [200, 1600, 30], sink=3, recent=9, weight=odd, seed=4).check(A)
    neg = (lambda w: torch.where(w > 1, w, torch.tensor(float("nan")).neg() * torch.ones_like(w)))  # NaN of either sign
    Case([400], [150], weight=neg, seed=4).check(A)


def test_all_but_one_and_one_of_all(A):
    Case([1000, 257, 2049], [999, 256, 2048], seed=1).check(A)
    Case([1000, 257, 2049], [1, 1, 1], seed=1).check(A)


@pytest.mark.parametrize("parents", [[0], [0, 0, 1, 2, 2], [1, 1]])
@pytest.mark.parametrize("extra", [0, 2])
def test_shared_pages_are_left_to_the_others(A, parents, extra):
    """Forks: all cut, some cut, cut to different lengths; pages held beyond the tokens."""
    n = 3 + len(parents)
    for budget in ([50] * n, [1000] * 3 + [40] * len(parents), [20 * (i + 1) for i in range(n)], [33, 1000] * n):
        Case([200, 333, 90], budget[:n], sink=2, recent=10, parents=parents, spare=120, extra=extra, seed=n).check(A)


def test_too_few_free_pages_change_nothing(A):
    for spare, budget in ((0, [64, 64, 64]), (3, [64, 64, 64]), (7, [64, 64, 64]), (8, [64, 64, 64]), (0, [500, 500, 64])):
        c = Case([200], budget, parents=[0, 0], spare=spare, seed=3)
        c.check(A)
        c.check(A, in_place=False)


def test_page_bookkeeping_of_many_rows(A):
    r = random.Random(1)
    lens = [r.randrange(0, 60) for _ in range(1500)]
    Case(lens, [r.randrange(0, 50) for _ in lens], sink=1, recent=2, layers=1, kv_heads=1, seed=1).check(A)


@pytest.mark.parametrize("dim,in_place", [(64, True), (128, False), (256, True)])
def test_many_rows_of_layers_and_heads(A, dim, in_place):
    """2560 of them, which take smaller blocks: two rows of several runs among many short ones."""
    r = random.Random(dim)
    lens = [1500, 1030, 1024, 1025] + [r.randrange(0, 60) for _ in range(36)]
    odd = (lambda w: torch.where(w > 20, torch.nan, (w * 4).floor() / 4))  # many equals
    c = Case(lens, [700, 40, 500, 1024] + [r.randrange(0, 50) for _ in range(36)], sink=2, recent=3, layers=8, kv_heads=8, dim=dim,
             weight=odd if dim == 128 else None, seed=dim)
    assert 8 * 8 * len(c.lens) >= 16 * torch.cuda.get_device_properties(0).multi_processor_count
    c.check(A, in_place)


def test_tokens_can_be_evicted_again_and_grown(A):
    """Evict, grow, evict: the states chain, and no live page has two owners."""
    c = Case([300, 450, 120], [100, 150, 100], sink=4, recent=20, parents=[1], spare=60, seed=8, slots=600)
    c.budget = [100, 150, 100, 140]
    cache, st, w = c.cache(A), c.state(A), c.w.cuda()
    budget = torch.tensor(c.budget, dtype=torch.int32).cuda()
    for _ in range(3):
        st, missing = A.cache_evict(cache, st, w, budget, sink=4, recent=20)
        assert int(missing) == 0
        rows = [t[:h] for t, h in zip(st.table.tolist(), st.held.tolist())]
        count = [0] * c.pages
        for row in rows:
            for p in row:
                count[p] += 1
        assert st.refs.tolist() == count
        need = st.lens + 30
        st, missing = A.cache_grow(cache, st, need)
        assert int(missing) == 0
        st.lens.copy_(need)  # thirty tokens written


def test_captures_streams_and_given_results(A):
    c = Case([700, 2500], [300, 1000], sink=4, recent=64, layers=3, seed=6)
    budget = torch.tensor(c.budget, dtype=torch.int32).cuda()
    cache, st, w = c.cache(A), c.state(A), c.w.cuda()
    k0, v0 = cache.k.clone(), cache.v.clone()
    out = A.PageState(*(torch.zeros_like(t) for t in st._tensors()))
    kept = torch.zeros_like(w)
    missing = torch.full((), 9, dtype=torch.int32, device="cuda")
    A.cache_evict(cache, st, w, budget, 4, 64, out=out, weight_out=kept, missing=missing)
    want = [cache.k.clone(), cache.v.clone(), kept.clone(), *(t.clone() for t in out._tensors())]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.cache_evict(cache, st, w, budget, 4, 64, out=out, weight_out=kept, missing=missing)
    cache.k.copy_(k0), cache.v.copy_(v0), kept.zero_()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip([cache.k, cache.v, kept, *out._tensors()], want)) and int(missing) == 0
    cache.k.copy_(k0), cache.v.copy_(v0), kept.zero_()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    new, miss = A.cache_evict(cache, st, w, budget, 4, 64, weight_out=kept, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip([cache.k, cache.v, kept, *new._tensors()], want)) and int(miss) == 0


def test_strided_weights(A):
    c = Case([300, 90], [100, 40], sink=1, recent=8, layers=2, kv_heads=2, seed=7)
    cache, st = c.cache(A), c.state(A)
    n = c.w.shape[3]
    pool = torch.full((2, 2, 2, n + 11), -3.0, device="cuda")  # [row][head][layer][slot]
    view = pool.permute(2, 0, 1, 3)[..., 5:5 + n]
    view.copy_(c.w)
    A.cache_evict(cache, st, view, torch.tensor(c.budget, dtype=torch.int32).cuda(), 1, 8)
    k, v, w2, *_ = c.want()
    assert torch.equal(view.cpu(), w2) and torch.equal(cache.k.cpu(), k) and torch.equal(cache.v.cpu(), v)
    view.fill_(-3.0)
    assert bool((pool == -3.0).all())


def test_no_rows(A):
    cache = A.KvCache.empty(2, 8, 16, 2, 64, torch.float16)
    st = A.PageState.empty(cache, 0, 4)
    w = torch.zeros((2, 0, 2, 5), device="cuda")
    new, missing = A.cache_evict(cache, st, w, torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert int(missing) == 0 and new.refs.tolist() == [0] * 8


def test_rows_that_make_no_sense_are_recorded_and_left():
    from plugins_b200 import attention as A
    from plugins_b200 import quant as Q
    c = Case([300, 90, 250, 60], [100, -1, 100, 20], seed=7, slots=260)
    cache, st, w = c.cache(A), c.state(A), c.w.cuda()
    st.lens[3] = 70  # beyond its pages
    Q.device_error(0, clear=True)
    # row 0 has more tokens than the weights have slots
    k0, w0 = cache.k.clone(), w.clone()
    new, missing = A.cache_evict(cache, st, w, torch.tensor(c.budget, dtype=torch.int32).cuda())
    assert Q.device_error(0, clear=True) != 0
    assert int(missing) == 0 and new.lens.tolist() == [300, 90, 100, 70]
    assert new.held.tolist()[:2] == st.held.tolist()[:2] and new.table[3].tolist() == st.table[3].tolist()
    assert torch.equal(w[:, [0, 1, 3]], w0[:, [0, 1, 3]])
    used = [p for i in (0, 1, 3) for p in c.table[i]]
    assert torch.equal(cache.k[:, used], k0[:, used])


def test_a_length_past_the_weights_slots_copies_what_there_is(A):
    from plugins_b200 import quant as Q
    c = Case([300, 90, 250], [100, 50, 100], seed=8, slots=260)
    for far in (300, 2 ** 31 - 1, -5):
        cache, st, w = c.cache(A), c.state(A), c.w.cuda()
        st.lens[0] = far
        whole = torch.full((2, 4, 2, 262), -7.0, device="cuda")  # the result lies inside
        out = whole[:, :3, :, 1:261]
        Q.device_error(0, clear=True)
        new, missing = A.cache_evict(cache, st, w, torch.tensor(c.budget, dtype=torch.int32).cuda(), weight_out=out)
        assert Q.device_error(0, clear=True) != 0
        assert int(missing) == 0 and new.lens.tolist() == [far, 50, 100]
        want = w[:, 0] if far > 0 else torch.full_like(w[:, 0], -7.0)
        assert torch.equal(out[:, 0], want)
        assert (whole[:, 3] == -7).all() and (whole[..., [0, 261]] == -7).all()


def test_slots_past_two_to_the_31_elements(A):
    """A pool whose last pages lie beyond 2^31 elements; only what is used is looked at."""
    page, dim = 256, 256
    pages = 2 ** 31 // (page * dim) + 8
    k = torch.empty((1, pages, 1, page, dim), dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    cache = A.KvCache(k, v)
    ids = [pages - 1, 0, pages - 2, pages - 5]
    g = torch.Generator(device="cuda").manual_seed(1)
    for p in ids:
        k[0, p].normal_(generator=g), v[0, p].normal_(generator=g)
    n = 1000
    at = torch.arange(n, device="cuda")
    tab = torch.tensor(ids, device="cuda")
    was = [t[0, tab[at // page], 0, at % page].clone() for t in (k, v)]
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[tab] = 1
    i = (lambda x: torch.tensor(x, dtype=torch.int32, device="cuda"))
    st = A.PageState(refs, i([ids]), i([4]), i([n]))
    w = torch.rand((1, 1, 1, n), generator=g, device="cuda")
    new, missing = A.cache_evict(cache, st, w.clone(), i([300]), 2, 30)
    keep = torch.tensor(E.kept_slots(w.flatten().tolist(), n, 300, 2, 30), device="cuda")
    at = torch.arange(300, device="cuda")
    for t, old in zip((k, v), was):
        assert torch.equal(t[0, new.table[0].long()[at // page], 0, at % page], old[keep])
    assert new.held.tolist() == [2] and int(missing) == 0


def test_arguments_the_wrappers_refuse(A):
    c = Case([100, 40], [50, 20])
    cache, st, w = c.cache(A), c.state(A), c.w.cuda()
    budget = torch.tensor(c.budget, dtype=torch.int32).cuda()
    k0 = cache.k.clone()
    for change in (dict(weight=w[:1]), dict(weight=w[:, :1]), dict(weight=w.double()), dict(weight=w.cpu()), dict(weight=w[0]),
                   dict(weight=w[..., ::2]), dict(weight_out=w[..., :50]), dict(budget=budget.long()), dict(budget=budget[:1]),
                   dict(sink=-1), dict(recent=-5), dict(recent=2 ** 32 + 5), dict(sink=2 ** 31),
                   dict(weight_out=w.flatten()[:w[..., 1:].numel()].view_as(w[..., 1:])), dict(out=st)):
        call = dict(weight=w, budget=budget) | change
        with pytest.raises(A.Exl3Error):
            A.cache_evict(cache, st, **call)
    lse, q = torch.zeros((2, 4), device="cuda"), torch.zeros((2, 4, 64), dtype=torch.float16, device="cuda")
    batch = A.TreeBatch(*(torch.tensor(x, dtype=torch.int32).cuda() for x in ([0, 1, 2], [100, 40], c.state(A).table.tolist())), max_rows=1, rows=2)
    for change in (dict(weight=w), dict(weight=w[0, :1]), dict(weight=w[0].half()), dict(lse=lse[:1]), dict(lse=lse.double()),
                   dict(lse=lse.t().contiguous().t()), dict(decay=1.5), dict(decay=-0.5), dict(scale=-1.0), dict(q=q.float()), dict(layer=2)):
        call = dict(layer=0, q=q, lse=lse, weight=w[0]) | change
        with pytest.raises(A.Exl3Error):
            A.attention_weight(cache, batch=batch, **call)
    assert torch.equal(cache.k, k0)
