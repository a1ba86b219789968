"""exl3_attention_weight against its formula in 64 bits (tests/evict_ref.py, which derives the tolerance), at the sizes,
masks and values where it can go wrong."""
import math

import pytest
import torch

import evict_ref as E
from test_attention_gpu import A, DT, Step, chain, cuda, random_tree  # noqa: F401  (A: a fixture)

pytestmark = pytest.mark.gpu


def queries(step, heads, dim, seed=1, pad=0):
    g = torch.Generator().manual_seed(seed)
    n = step.row_start[-1]
    return (1.5 * torch.randn((n, heads * dim + pad), generator=g)).to(step.dtype).cuda()[:, :heads * dim].unflatten(1, (heads, dim))


def old_weights(step, kv_heads, slots, seed=2):
    g = torch.Generator().manual_seed(seed)
    return 0.01 * torch.rand((len(step.rows), kv_heads, slots), generator=g)


def check(A, step, heads, kv_heads, dim, decay=1.0, slots=None, max_context=0, q=None, scale=None):
    cache, batch = step.device(A, max_context=max_context, rows=step.row_start[-1])
    q = queries(step, heads, dim) if q is None else q
    most = max(r + n for r, n in zip(step.rows, step.lens))
    old = old_weights(step, kv_heads, most + 3 if slots is None else slots)
    _, lse = A.tree_attention(cache, step.layer, batch, q, scale=scale, lse=True)
    w = old.cuda()
    assert A.attention_weight(cache, step.layer, batch, q, lse, w, scale=scale, decay=decay) is w
    want, off = E.weights(step.k[step.layer], q.cpu(), lse.cpu(), step.row_start, step.lens, step.table,
                          dim ** -0.5 if scale is None else scale, decay, old, step.tree)
    err = (w.cpu().double() - want).abs()
    assert bool((err <= off).all()), f"worst {float((err / off.clamp(min=1e-30)).max()):.2f} x the tolerance"
    return cache, batch, q, lse, old, w


CASES = [
    # rows, context, heads, kv heads, dim, page, dtype
    ([1], [0], 8, 8, 64, 16, "f16"), ([1], [1], 8, 2, 128, 16, "bf16"), ([1], [126], 4, 4, 128, 32, "f16"),
    ([1, 1, 1], [127, 128, 129], 8, 2, 128, 64, "bf16"), ([1, 1, 1], [254, 255, 256], 32, 4, 64, 128, "f16"),
    ([1, 0, 2, 1], [300, 50, 0, 1111], 10, 2, 128, 16, "bf16"), ([3, 17, 1], [600, 31, 5], 24, 4, 128, 64, "f16"),
    ([5], [2000], 16, 8, 256, 128, "f16"), ([9, 4], [130, 777], 6, 1, 256, 32, "bf16"), ([2], [90], 48, 1, 64, 256, "bf16"),
    ([130], [0], 4, 1, 128, 16, "bf16"), ([300, 70], [77, 513], 8, 2, 128, 64, "f16"), ([65], [200], 7, 1, 64, 16, "bf16"),
    ([700], [0], 2, 2, 256, 64, "bf16"), ([257, 255, 256], [0, 1, 255], 4, 2, 64, 32, "f16"), ([33], [3], 130, 1, 128, 16, "bf16"),
    ([1] * 40, list(range(0, 1200, 30)), 8, 2, 128, 16, "bf16"), ([1000], [1500], 16, 2, 128, 64, "bf16"),
]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("decay", [1.0, 0.9])
def test_chunks_of_any_size(A, case, decay):
    rows, lens, heads, kvh, dim, page, dtype = CASES[case]
    check(A, Step(rows, lens, kvh, dim, page, dtype, seed=case), heads, kvh, dim, decay)


@pytest.mark.parametrize("rows,lens,heads,kvh,dim,page,dtype", [
    ([5], [0], 4, 1, 128, 16, "bf16"), ([40, 3, 33], [100, 0, 250], 8, 2, 128, 16, "bf16"), ([64, 1], [500, 127], 16, 4, 64, 64, "f16"),
    ([17, 9], [2047, 130], 16, 8, 256, 128, "f16"), ([100], [90], 6, 2, 128, 32, "bf16"), ([130, 70], [60, 0], 5, 1, 128, 16, "f16")])
def test_trees(A, rows, lens, heads, kvh, dim, page, dtype):
    check(A, Step(rows, lens, kvh, dim, page, dtype, tree=random_tree, seed=len(rows)), heads, kvh, dim, 0.95)


def test_rows_that_see_nothing_and_rows_that_do_not_see_themselves(A):
    def lonely(s, n):
        return [0 if i % 2 else (1 << (i // 2)) for i in range(n)], [0] * n
    for lens in ([0, 0], [50, 0]):
        step = Step([9, 40], lens, 2, 128, 16, "bf16", tree=lonely)
        _, _, _, lse, _, _ = check(A, step, 8, 2, 128)
        assert bool(torch.isinf(lse).any())


@pytest.mark.parametrize("stale", [math.inf, math.nan, -math.inf])
@pytest.mark.parametrize("rows,lens", [([1, 1], [100, 17]), ([70, 90], [33, 0])])
def test_what_no_row_sees_does_not_reach_a_weight(A, stale, rows, lens):
    check(A, Step(rows, lens, 2, 128, 64, "bf16", stale=stale), 8, 2, 128)
    check(A, Step(rows, lens, 2, 128, 64, "f16", tree=random_tree, stale=stale), 8, 2, 128)


@pytest.mark.parametrize("rows", [3, 60])
def test_a_bad_row_reaches_the_slots_it_sees_alone(A, rows):
    """NaN in a drafted row's query: the slots that row does not see keep their weights exactly; the others get NaN."""
    step = Step([rows], [200], 2, 128, 16, "bf16", tree=random_tree)
    cache, batch = step.device(A, rows=rows)
    q = queries(step, 8, 128)
    q[2, 1] = math.nan  # kv head 0
    old = old_weights(step, 2, 280)
    _, lse = A.tree_attention(cache, step.layer, batch, q, lse=True)
    w = A.attention_weight(cache, step.layer, batch, q, lse, old.cuda()).cpu()
    good = q.clone()
    good[2, 1] = 0
    seen = torch.zeros(280, dtype=torch.bool)
    seen[:200] = True
    for j in range(rows):
        seen[200 + j] = bool((int(step.tree[2, j // 32]) >> (j % 32)) & 1)
    assert bool(torch.isnan(w[0, 0, seen]).all()) and not bool(torch.isnan(w[0, 0, ~seen]).any())
    assert not bool(torch.isnan(w[0, 1]).any())
    # a NaN key is its own slot's
    step.k[step.layer][step.table[0, 3], 1, 5] = math.nan
    cache, batch = step.device(A, rows=rows)
    _, lse = A.tree_attention(cache, step.layer, batch, good, lse=True)
    lse = torch.nan_to_num(lse, nan=1.0)
    w = A.attention_weight(cache, step.layer, batch, good, lse, old.cuda()).cpu()
    assert torch.isnan(w).nonzero().tolist() == [[0, 1, 3 * 16 + 5]]


@pytest.mark.parametrize("heads,dim", [(2, 128), (8, 64), (4, 256)])
def test_a_bad_row_of_a_full_tile_wherever_it_lies(A, heads, dim):
    step = Step([256], [300], 2, dim, 64, "f16")
    cache, batch = step.device(A, rows=256)
    old = old_weights(step, 2, 560)
    for at in (0, 1, 2, 3, 4, 5, 6, 7, 130, 255):
        for head in range(heads // 2):
            q = queries(step, heads, dim)
            q[at, head] = math.nan
            _, lse = A.tree_attention(cache, step.layer, batch, q, lse=True)
            w = A.attention_weight(cache, step.layer, batch, q, lse, old.cuda())[0].isnan().cpu()
            assert bool(w[0, :300 + at + 1].all()) and not bool(w[0, 300 + at + 1:].any()) and not bool(w[1].any())


def test_probabilities_next_to_nothing_stay_above_zero(A):
    """Scores hundreds apart: what is below 2^-125 adds nothing, and no weight ends below zero."""
    for dim in (64, 128, 256):
        step = Step([256, 1, 40], [300, 500, 5], 2, dim, 64, "bf16")
        q = queries(step, 8, dim) * 40
        cache, batch = step.device(A, rows=step.row_start[-1])
        _, lse = A.tree_attention(cache, step.layer, batch, q, lse=True)
        w = A.attention_weight(cache, step.layer, batch, q, lse, torch.zeros((3, 2, 560), device="cuda"))
        assert bool((w >= 0).all()) and bool((w == 0).any()) and not bool(torch.signbit(w).any())


@pytest.mark.parametrize("pad", [1, 4, 8])
def test_queries_of_any_stride(A, pad):
    for rows, lens in (([1, 2], [40, 300]), ([90], [50])):
        step = Step(rows, lens, 2, 64, 16, "f16", layout="phd")
        check(A, step, 6, 2, 64, q=queries(step, 6, 64, pad=pad))


def test_heads_before_rows_and_broadcast_queries(A):
    step = Step([20], [100], 2, 128, 16, "bf16")
    q = queries(step, 8, 128)
    check(A, step, 8, 2, 128, q=q.transpose(0, 1).contiguous().transpose(0, 1))
    check(A, step, 8, 2, 128, q=q[:1].expand(20, 8, 128))
    check(A, step, 8, 2, 128, q=q[:, :1].expand(20, 8, 128), scale=0.3)


def test_a_prompt_of_many_rows(A):
    check(A, Step([2500], [300], 1, 128, 64, "bf16"), 4, 1, 128, 0.5)


def test_the_new_weights_sum_to_the_rows(A):
    """Each row and head spreads a weight of one: 2^-12 covers the terms' errors (the bound of each is below that)."""
    step = Step([40, 1, 7], [3000, 500, 0], 2, 128, 64, "bf16")
    cache, batch = step.device(A, rows=48)
    q = queries(step, 8, 128)
    _, lse = A.tree_attention(cache, step.layer, batch, q, lse=True)
    w = A.attention_weight(cache, step.layer, batch, q, lse, torch.zeros((3, 2, 3100), device="cuda"))
    want = 4.0 * torch.tensor(step.rows, dtype=torch.float64)[:, None]
    assert float((w.double().sum(-1).cpu() / want - 1).abs().max()) < 2.0 ** -12


def test_decay_zero_does_not_read_and_others_are_left(A):
    step = Step([2, 0, 5], [30, 40, 0], 2, 64, 16, "bf16")
    cache, batch = step.device(A, rows=7)
    q = queries(step, 4, 64)
    _, lse = A.tree_attention(cache, step.layer, batch, q, lse=True)
    zero = torch.zeros((3, 2, 60), device="cuda")
    want = A.attention_weight(cache, step.layer, batch, q, lse, zero.clone(), decay=0.0)
    bad = torch.full((3, 2, 60), math.nan, device="cuda")
    got = A.attention_weight(cache, step.layer, batch, q, lse, bad.clone(), decay=0.0)
    for s, n in ((0, 32), (1, 0), (2, 5)):
        assert torch.equal(got[s, :, :n], want[s, :, :n])
        assert bool(torch.isnan(got[s, :, n:]).all())


def test_a_layer_of_strided_weights(A):
    step = Step([3, 1], [100, 260], 2, 128, 16, "f16")
    cache, batch = step.device(A, rows=4)
    q = queries(step, 8, 128)
    _, lse = A.tree_attention(cache, step.layer, batch, q, lse=True)
    want = A.attention_weight(cache, step.layer, batch, q, lse, torch.ones((2, 2, 270), device="cuda"), decay=0.5)
    pool = torch.ones((2, 3, 2, 301), device="cuda")  # [kv head][layer][row][slot]
    view = pool.permute(1, 2, 0, 3)[1][..., 7:277]
    A.attention_weight(cache, step.layer, batch, q, lse, view, decay=0.5)
    assert torch.equal(view, want)
    view.fill_(1)
    assert bool((pool == 1).all())


def test_the_bits_do_not_depend_on_the_bounds_and_captures_replay(A):
    step = Step([70, 1, 9], [900, 2500, 0], 2, 128, 64, "bf16", tree=random_tree)
    q = queries(step, 16, 128)
    outs = []
    for most in (0, 2502, 5000):
        cache, batch = step.device(A, max_context=most, rows=80)
        if not outs:
            _, lse = A.tree_attention(cache, step.layer, batch, q, lse=True)
        outs.append(A.attention_weight(cache, step.layer, batch, q, lse, torch.ones((3, 2, 2600), device="cuda"), decay=0.5))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    w = torch.ones((3, 2, 2600), device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.attention_weight(cache, step.layer, batch, q, lse, w, decay=0.5)
    w.fill_(1)
    graph.replay()
    assert torch.equal(w, outs[0])
    # other contexts and rows in the captured tensors
    batch._keep[0].copy_(torch.tensor([0, 2, 2, 59], dtype=torch.int32))
    batch._keep[1].copy_(torch.tensor([500, 100, 7], dtype=torch.int32))
    w.fill_(1)
    graph.replay()
    fresh = A.attention_weight(cache, step.layer, batch, q, lse, torch.ones((3, 2, 2600), device="cuda"), decay=0.5)
    assert torch.equal(w, fresh) and bool((w[1] == 1).all()) and bool((w[0, :, 502:] == 1).all())


@pytest.mark.parametrize("rows", [(9, 3), (40, 130)])
def test_a_bound_on_the_rows_that_is_too_low_costs_time_alone(A, rows):
    step = Step(list(rows), [100, 300], 2, 128, 16, "bf16")
    cache, batch = step.device(A, rows=sum(rows))
    q = queries(step, 8, 128)
    _, lse = A.tree_attention(cache, step.layer, batch, q, lse=True)
    old = old_weights(step, 2, 440)
    want, off = E.weights(step.k[step.layer], q.cpu(), lse.cpu(), step.row_start, step.lens, step.table, 128 ** -0.5, 1.0, old)
    for most in (1, 2, 5):
        batch.raw.max_rows = most
        w = A.attention_weight(cache, step.layer, batch, q, lse, old.cuda())
        assert bool(((w.cpu().double() - want).abs() <= off).all())


def test_another_stream_and_padding_rows(A):
    step = Step([3, 2], [200, 40], 2, 128, 16, "bf16")
    cache, batch = step.device(A, rows=5)
    q = queries(step, 8, 128)
    _, lse = A.tree_attention(cache, step.layer, batch, q, lse=True)
    want = A.attention_weight(cache, step.layer, batch, q, lse, torch.ones((2, 2, 210), device="cuda"))
    w = torch.ones((2, 2, 210), device="cuda")
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    A.attention_weight(cache, step.layer, batch, q, lse, w, stream=st)
    st.synchronize()
    assert torch.equal(w, want)
    cache, batch = step.device(A, rows=9)  # four rows of padding
    more = (lambda t: torch.cat([t, torch.full((4, *t.shape[1:]), math.nan, dtype=t.dtype, device="cuda")]))
    w = A.attention_weight(cache, step.layer, batch, more(q), more(lse), torch.ones((2, 2, 210), device="cuda"))
    assert torch.equal(w, want)


def test_values_out_of_range_are_recorded_and_not_followed():
    from plugins_b200 import attention as A
    from plugins_b200 import quant as Q
    step = Step([3, 2], [200, 40], 2, 128, 16, "bf16")
    cache, batch = step.device(A, rows=5)
    q = queries(step, 8, 128)
    _, lse = A.tree_attention(cache, step.layer, batch, q, lse=True)
    Q.device_error(0, clear=True)
    want = A.attention_weight(cache, step.layer, batch, q, lse, torch.ones((2, 2, 203), device="cuda"))
    assert Q.device_error(0, clear=True) == 0
    # fewer slots than tokens: the first ones' weights, an error
    guard = torch.ones((2, 2, 203), device="cuda")
    A.attention_weight(cache, step.layer, batch, q, lse, guard[..., :100])
    assert torch.equal(guard[..., :100], want[..., :100]) and bool((guard[..., 100:] == 1).all())
    assert Q.device_error(0, clear=True) != 0
    # a page that does not exist: its keys count as zeros, as in the attention
    batch._keep[2][0, 2] = -1
    batch._keep[2][0, 3] = 10 ** 9
    w = A.attention_weight(cache, step.layer, batch, q, lse, torch.ones((2, 2, 203), device="cuda"))
    assert Q.device_error(0, clear=True) != 0
    assert torch.equal(w[0, :, :32], want[0, :, :32]) and torch.equal(w[0, :, 64:], want[0, :, 64:])
    zero = 1 + torch.exp(-lse[:3]).view(3, 2, 4).sum((0, 2))  # f32 exponentials: 2^-18 covers them
    assert float((w[0, :, 32:64] / zero[:, None] - 1).abs().max()) < 2.0 ** -18
    # a context beyond the table
    batch._keep[1][1] = 2 ** 31 - 1
    A.attention_weight(cache, step.layer, batch, q, lse, torch.ones((2, 2, 203), device="cuda"))
    assert Q.device_error(0, clear=True) != 0


@pytest.mark.parametrize("rows,lens", [([1, 1, 3], [2000, 5, 700]), ([200], [300])])
def test_steps_accumulate(A, rows, lens):
    """Three steps over growing rows: what was a row's own slot is the next step's context."""
    step = Step(rows, lens, 2, 128, 64, "bf16")
    w, want, off = None, None, 0
    for n in range(3):
        step.lens = [x + (r if n else 0) for x, r in zip(step.lens, step.rows)]
        held = max(-(-(r + x) // 64) for r, x in zip(step.rows, step.lens))
        table = torch.arange(len(rows) * held, dtype=torch.int32).view(len(rows), held)
        step.table = table
        if int(table.max()) >= step.pages:
            more = len(rows) * held - step.pages + 8
            step.k, step.v = (torch.cat([t, torch.randn((2, more, *t.shape[2:]), generator=torch.Generator().manual_seed(n)).to(t.dtype)], 1)
                              for t in (step.k, step.v))
            step.pages += more
        cache, batch = step.device(A, rows=step.row_start[-1])
        q = queries(step, 8, 128, seed=n)
        _, lse = A.tree_attention(cache, step.layer, batch, q, lse=True)
        if w is None:
            w, want = (torch.zeros((len(rows), 2, 3000), device=d) for d in ("cuda", "cpu"))
        A.attention_weight(cache, step.layer, batch, q, lse, w, decay=0.75)
        want, more = E.weights(step.k[step.layer], q.cpu(), lse.cpu(), step.row_start, step.lens, step.table, 128 ** -0.5, 0.75, want)
        off = 0.75 * off + more
        assert bool(((w.cpu().double() - want).abs() <= off).all())
