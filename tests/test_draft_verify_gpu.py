"""exl3_draft_verify against its definition in 64 bits (tests/draft_ref.py), at the sizes and values where it can go wrong.

The results are whole numbers and have to be the reference's.  A decision that lies within the f32 exponentials' error of its
border (the reference says how near each comes) may go either way: such a sequence's random numbers are drawn again, by the
reference alone, before the kernel runs."""
import math

import pytest
import torch

import draft_ref as R

pytestmark = pytest.mark.gpu

F = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def setup(rows, back, vocab, dtype, draft, temps, seed, pad=0, peak=9.0):
    """Inputs on the CPU: peaked logits (as a strided view where pad), drafts that are often right, trees."""
    g = torch.Generator().manual_seed(seed)
    start = [0]
    for n in rows:
        start.append(start[-1] + n)
    total = start[-1]
    wide = torch.randn((max(total, 1), vocab + pad), generator=g) * 2
    wide.scatter_(1, torch.randint(vocab, (max(total, 1), min(3, vocab)), generator=g), peak + math.log(vocab) / 2)
    logits = wide.to(F[dtype])[:total, :vocab]
    parent, of = [], []
    for s, n in enumerate(rows):
        for i in range(n):
            p = int(torch.randint(max(0, i - back), i, (1,), generator=g)) if i else -1
            parent.append(p)
            of.append(start[s] + max(p, 0))
    x = logits.float() * 0.9 + 0.3 * torch.randn((total, vocab), generator=g)
    q = torch.softmax(x, 1).to(F[draft]) if draft else None
    x = x[of] if total else x
    noise = -torch.log(-torch.log(torch.rand((total, vocab), generator=g).clamp(1e-9, 1 - 1e-7)))
    tokens = (x + noise).argmax(1).int() if total else torch.zeros(0, dtype=torch.int32)
    uniform = torch.rand((total, 2), generator=g)
    temperature = None if temps is None else torch.tensor([temps[s % len(temps)] for s in range(len(rows))])
    return dict(start=start, rows=rows, logits=logits, wide=wide.to(F[dtype]), tokens=tokens,
                parent=torch.tensor(parent, dtype=torch.int32), uniform=uniform, temperature=temperature, draft=q)


def make(i, spare=0):
    """The same on the GPU: (cache, batch, arguments)."""
    from plugins_b200 import attention as A
    cache = A.KvCache.empty(1, 2, 16, 1, 64)
    n = len(i["rows"])
    ints = (lambda v: torch.tensor(v, dtype=torch.int32, device="cuda"))
    total = i["start"][-1]
    batch = A.TreeBatch(ints(i["start"]), ints([0] * n), ints([[0]] * n) if n else ints([]).view(0, 1),
                        max_rows=max(list(i["rows"]) + [0]), rows=total + spare)
    vocab = i["logits"].shape[1]
    cuda = (lambda t: None if t is None else t.cuda())
    logits = i["wide"].cuda()[:total, :vocab] if i["wide"].shape[0] >= total else i["logits"].cuda()
    return cache, batch, [logits, cuda(i["tokens"]), cuda(i["parent"]), cuda(i["uniform"])], dict(
        temperature=cuda(i["temperature"]), draft=cuda(i["draft"]))


def check(i, depth=None, chain=False):
    from plugins_b200 import attention as A
    from plugins_b200 import quant as Q
    deep = max(1, max(i["rows"], default=1)) if depth is None else depth
    again = torch.Generator().manual_seed(7)
    for _ in range(200):
        paths, tokens, near = R.verify(i["start"], i["logits"], i["tokens"], None if chain else i["parent"], i["uniform"],
                                       i["temperature"], i["draft"], deep)
        close = [s for s, d in enumerate(near) if d <= 1]
        for s in close:
            a, b = i["start"][s], i["start"][s + 1]
            i["uniform"][a:b] = torch.rand((b - a, 2), generator=again)
        if not close:
            break
    assert not close
    cache, batch, args, kw = make(i)
    if chain:
        args[2] = None
    path, kept, token = A.draft_verify(cache, batch, *args, **kw, depth=depth)
    assert path.shape == (len(i["rows"]), deep)
    assert kept.tolist() == [len(p) for p in paths]
    assert path.tolist() == [p + [-1] * (deep - len(p)) for p in paths]
    assert token.tolist() == tokens
    assert Q.device_error(0) == 0
    return paths, tokens


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("draft", ["", "f32", "bf16", "f16"])
def test_trees_of_every_type(dtype, draft):
    i = setup([6, 1, 9, 0, 12, 5, 7, 3], 3, 4097, dtype, draft, [0.8, 1.0, 0.0, 1.3], seed=1)
    paths, _ = check(i)
    assert any(len(p) > 1 for p in paths)


@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 8, 9, 31, 63, 64, 65, 257, 1000, 4096, 32001, 65537])
@pytest.mark.parametrize("draft", ["", "bf16"])
def test_vocabularies(vocab, draft):
    check(setup([5, 4], 2, vocab, "bf16", draft, [1.0], seed=vocab))


@pytest.mark.parametrize("draft", ["", "f16"])
def test_the_largest_vocabulary(draft):
    check(setup([4, 1], 2, 393216, "f32", draft, [0.9], seed=5))


@pytest.mark.parametrize("pad", [1, 2, 3, 5, 8, 13])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_of_any_stride(pad, dtype):
    check(setup([7, 5, 6], 2, 3001, dtype, "f32", [0.9, 0.0], seed=pad, pad=pad))


@pytest.mark.parametrize("draft", ["", "f32"])
def test_one_row_each_is_sampling(draft):
    check(setup([1] * 70, 1, 2048, "f16", draft, [0.7, 1.0, 0.0], seed=11, peak=3.0))


@pytest.mark.parametrize("rows,depth", [(9, 1), (9, 3), (9, 20), (33, 33), (40, None)])
@pytest.mark.parametrize("draft", ["", "f32"])
def test_chains_of_any_depth(rows, depth, draft):
    i = setup([rows, 1, rows // 2], 1, 300, "f32", draft, [0.5, 1.0], seed=rows, peak=14.0)
    i["uniform"][:, 0] *= 0.2  # long paths
    check(i, depth, chain=True)


@pytest.mark.parametrize("draft", ["", "f32"])
def test_many_siblings_and_the_same_token_twice(draft):
    """A root with 70 children over few tokens: rejections, repeated tokens, the rest of p after them."""
    i = setup([71, 71], 70, 40, "f32", draft, [1.0, 0.0], seed=3, peak=0.0)
    i["parent"] = torch.tensor(([-1] + [0] * 70) * 2, dtype=torch.int32)
    i["uniform"][:, 0] = 0.97 + 0.03 * i["uniform"][:, 0]
    paths, _ = check(i)


def test_tokens_and_parents_that_do_not_exist():
    i = setup([6, 6], 2, 500, "f32", "f32", [1.0, 0.0], seed=4)
    i["tokens"][1], i["tokens"][2], i["tokens"][7], i["tokens"][8] = -1, 500, 2 ** 31 - 1, -2 ** 31
    i["parent"][3], i["parent"][4], i["parent"][9] = 5, 4, -7  # later than itself, itself, none
    check(i)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_infinities_and_nan(dtype):
    i = setup([3, 3, 3, 3, 3], 1, 777, dtype, "f32", [1.0, 0.0], seed=6)
    x = i["wide"]
    x[0, 5:700] = -math.inf
    x[1, ::3] = math.nan
    x[3, 100] = math.inf
    x[3, 650] = math.inf
    x[6], x[9] = -math.inf, -math.inf  # nothing can follow these rows
    x[12, 3] = math.nan
    i["logits"] = x[:15, :777]
    i["draft"][0, 10], i["draft"][1, 11], i["draft"][2, 12] = math.nan, -1.0, 0.0
    _, tokens = check(i)
    assert tokens[2] == tokens[3] == -1


def test_a_greedy_tie_takes_the_lowest():
    for at in ([70, 5, 900], [900, 901], [0, 999], [513, 512]):
        i = setup([2, 1], 1, 1000, "f32", "", [0.0], seed=9)
        i["wide"].clamp_(max=3)
        i["wide"][:, at] = 7.0
        i["logits"] = i["wide"]
        i["tokens"][1] = min(at)
        paths, tokens = check(i)
        assert tokens == [min(at)] * 2 and len(paths[0]) == 2


def test_the_ends_of_the_random_numbers():
    """u = 0 takes the first token with any probability, u just below one the last that the sums reach."""
    i = setup([1, 1, 1, 1], 1, 100, "f32", "", [1.0], seed=2)
    x = torch.full((4, 100), -400.0)
    x[0, 40], x[0, 41] = 0.0, -30.0
    x[1, 7], x[1, 93] = -69.0, 0.0       # 2^-99.5 and one: counts
    x[2, 7], x[2, 93] = -69.5, 0.0       # 2^-100.3: does not
    x[3, 10:20] = 0.0
    i["wide"] = i["logits"] = x
    i["uniform"][:, 1] = torch.tensor([0.0, 0.0, 0.0, 1 - 2.0 ** -24])
    from plugins_b200 import attention as A
    cache, batch, args, kw = make(i)
    _, kept, token = A.draft_verify(cache, batch, *args, **kw)
    assert kept.tolist() == [1] * 4 and token.tolist() == [40, 7, 93, 19]


@pytest.mark.parametrize("temp", [1e-30, 1e-4, 0.01, 50.0, 1e6, 1e30])
def test_temperatures(temp):
    i = setup([5, 4, 3], 2, 1500, "bf16", "f32", [temp], seed=8)
    check(i)


def test_no_temperature_is_one():
    i = setup([5, 4, 3], 2, 1500, "f32", "f32", None, seed=8)
    check(i)


def test_the_law_of_the_next_tokens():
    """Whatever the drafter, the first new token (the first accepted draft, else the token) is distributed as p: 40000
    sequences of two different drafts each; a frequency's deviation is sqrt(p (1 - p) / n), five of which one of 8 tokens
    passes once in 200000 sets."""
    from plugins_b200 import attention as A
    n, vocab = 40000, 8
    g = torch.Generator().manual_seed(3)
    x = torch.tensor([1.0, 0.5, 0.0, 2.0, -1.0, -3.0, 0.3, 1.2])
    q = torch.softmax(torch.tensor([0.0, 1.5, 0.2, 0.0, -1.0, 1.0, 0.3, -2.0]), 0)
    p = torch.softmax(x.double() / 0.9, 0)
    for with_q in (True, False):
        if with_q:
            drafts = torch.multinomial(q.expand(n, vocab), 2, replacement=True, generator=g)
        else:
            drafts = torch.randint(vocab, (n, 2), generator=g)
        tokens = torch.cat([torch.zeros((n, 1), dtype=torch.int64), drafts], 1).reshape(-1).int().cuda()
        parent = torch.tensor([-1, 0, 0], dtype=torch.int32).repeat(n).cuda()
        cache = A.KvCache.empty(1, 2, 16, 1, 64)
        ints = (lambda v: torch.as_tensor(v, dtype=torch.int32, device="cuda"))
        batch = A.TreeBatch(ints(torch.arange(n + 1) * 3), ints(torch.zeros(n)), ints(torch.zeros((n, 1))), max_rows=3,
                            rows=3 * n)
        path, kept, token = A.draft_verify(
            cache, batch, x.cuda().expand(3 * n, vocab), tokens, parent, torch.rand((3 * n, 2), generator=g).cuda(),
            temperature=torch.full((n,), 0.9, device="cuda"), draft=q.cuda().expand(3 * n, vocab) if with_q else None)
        first = torch.where(kept == 2, tokens.view(n, 3).gather(1, path[:, 1:2].clamp(min=0).long())[:, 0], token)
        seen = torch.bincount(first.cpu(), minlength=vocab).double() / n
        assert float(((seen - p).abs() / (p * (1 - p) / n).sqrt()).max()) < 5
        assert int((kept == 2).sum()) > n // 10


def test_the_same_call_gives_the_same_bits_and_captures():
    from plugins_b200 import attention as A
    i = setup([9, 17, 4], 3, 20000, "bf16", "f16", [0.8, 1.1], seed=12)
    cache, batch, args, kw = make(i)
    outs = [torch.empty((3, 17), dtype=torch.int32, device="cuda"), *(torch.empty(3, dtype=torch.int32, device="cuda") for _ in range(2))]
    A.draft_verify(cache, batch, *args, **kw, path=outs[0], kept=outs[1], token=outs[2])
    want = [o.clone() for o in outs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.draft_verify(cache, batch, *args, **kw, path=outs[0], kept=outs[1], token=outs[2])
    for o in outs:
        o.fill_(77)
    graph.replay()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    j = setup([9, 17, 4], 3, 20000, "bf16", "f16", [0.8, 1.1], seed=13)  # new values in the captured tensors
    for a, b in zip(args, (j["logits"], j["tokens"], j["parent"], j["uniform"])):
        a.copy_(b)
    kw["draft"].copy_(j["draft"])
    graph.replay()
    fresh = A.draft_verify(cache, batch, *args, **kw)
    assert all(torch.equal(o, w) for o, w in zip(outs, fresh))


def test_another_stream_and_padding_rows():
    from plugins_b200 import attention as A
    i = setup([5, 6], 2, 3000, "f32", "", [0.9], seed=14)
    cache, batch, args, kw = make(i)
    want = A.draft_verify(cache, batch, *args, **kw)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    got = A.draft_verify(cache, batch, *args, **kw, stream=st)
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # rows past the last sequence take no part
    cache, batch, args, kw = make(i, spare=3)
    more = [torch.cat([a, a[:3]]) for a in args]
    got = A.draft_verify(cache, batch, *more, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_values_out_of_range_are_recorded_and_not_followed():
    from plugins_b200 import attention as A
    from plugins_b200 import quant as Q
    i = setup([5, 6], 2, 300, "f32", "", [0.9], seed=14)
    cache, batch, args, kw = make(i)
    Q.device_error(0, clear=True)
    kw["temperature"] = torch.tensor([-1.0, math.nan], device="cuda")  # taken as greedy
    got = A.draft_verify(cache, batch, *args, **kw)
    assert Q.device_error(0, clear=True) != 0
    kw["temperature"] = torch.zeros(2, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(got, A.draft_verify(cache, batch, *args, **kw)))
    assert Q.device_error(0, clear=True) == 0
    batch._keep[0].copy_(torch.tensor([-3, 5, 400], dtype=torch.int32))
    A.draft_verify(cache, batch, *args, **kw)
    assert Q.device_error(0, clear=True) != 0


def test_arguments_the_wrappers_refuse():
    from plugins_b200 import attention as A
    i = setup([3, 2], 2, 300, "f32", "f16", [0.9], seed=14)
    cache, batch, args, kw = make(i)
    logits, tokens, parent, uniform = args
    bad = [dict(logits=logits[:, ::2]), dict(logits=logits.cpu()), dict(logits=logits[:3]), dict(logits=logits.double()),
           dict(logits=logits.int()), dict(tokens=tokens.long()), dict(tokens=tokens[:2]), dict(parent=parent.float()),
           dict(uniform=uniform[:, :1]), dict(uniform=uniform.double()), dict(uniform=uniform.t().contiguous().t()),
           dict(temperature=kw["temperature"][:1]), dict(temperature=kw["temperature"].half()),
           dict(draft=kw["draft"][:, :200]), dict(draft=kw["draft"].long()), dict(depth=0), dict(depth=-3),
           dict(path=torch.zeros((2, 4), dtype=torch.int32, device="cuda"), depth=3), dict(kept=torch.zeros(2, device="cuda"))]
    for change in bad:
        call = dict(logits=logits, tokens=tokens, parent=parent, uniform=uniform) | kw | change
        with pytest.raises(A.Exl3Error):
            A.draft_verify(cache, batch, **call)
