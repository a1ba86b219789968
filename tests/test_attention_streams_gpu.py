"""The attention side on a stream of its own (plugins_b200/attention.py): the tensors its work uses live until it is done."""
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


def cache_of(A, layers=2, pages=16, kv_heads=2, page=16, dim=64):
    g = torch.Generator(device="cuda").manual_seed(3)
    return A.KvCache(*(torch.randn((layers, pages, kv_heads, page, dim), generator=g, device="cuda").half() for _ in range(2)))


def batch_of(A):
    return A.TreeBatch(i32([0, 3, 5]), i32([20, 7]), i32([[4, 2, -1], [1, 9, -1]]), max_rows=3,
                       tree=i32([[1], [3], [5], [1], [2]]), position=i32([20, 21, 21, 7, 7]))


def state_of(A):
    refs = [0] * 16
    for p in (4, 2, 1, 9):
        refs[p] = 1
    return A.PageState(i32(refs), i32([[4, 2, -1], [1, 9, -1]]), i32([2, 2]), i32([20, 17]))


def rope_of(A):
    one = torch.ones(64, dtype=torch.float16, device="cuda")
    return A.NormRope(torch.ones(32, dtype=torch.float64, device="cuda"), one, one.clone())


CALLS = ["rope", "attention", "fork", "grow", "compact", "keep"]


def make(A, which):
    """(the call, the tensors it reads)"""
    cache = cache_of(A)
    x = torch.randn((5, 8, 64), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").half()
    if which in ("rope", "attention", "keep"):
        batch = batch_of(A)
        used = [cache.k, cache.v] + [t for t in batch._keep]
        if which == "rope":
            rope = rope_of(A)
            q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
            return lambda **kw: (A.qk_norm_rope(cache, 1, batch, q, k, v, rope, **kw), cache.k, cache.v), used + [q, k, v, *rope._keep]
        if which == "attention":
            q = x[:, :4]
            return lambda **kw: A.tree_attention(cache, 1, batch, q, lse=True, **kw), used + [q]
        path, kept = i32([[0, 2], [1, -1]]), i32([2, 1])
        batch.rows = batch.raw.rows = 5
        return lambda **kw: (A.cache_keep(cache, batch, path, kept, **kw), cache.k, cache.v), used + [path, kept]
    state = state_of(A)
    used = [state.refs, state.table, state.held, state.lens]
    flat = (lambda s: (s.refs, s.table, s.held, s.lens, cache.k, cache.v))
    if which == "fork":
        parent = i32([1, 1, 0])
        return lambda **kw: flat(A.cache_fork(cache, state, parent, **kw))[:4], used + [parent]  # (no key or value moves)
    if which == "grow":
        need = i32([40, 33])
        return lambda **kw: flat(A.cache_grow(cache, state, need, **kw)[0]), used + [need, cache.k, cache.v]
    return lambda **kw: flat(A.cache_compact(cache, state, **kw)), used + [cache.k, cache.v]


@pytest.mark.parametrize("which", CALLS)
def test_what_a_call_reads_is_recorded_on_its_stream(A, which, monkeypatch):
    call, used = make(A, which)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    seen = []
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: seen.append((t.data_ptr(), s)))
    call(stream=side)
    torch.cuda.synchronize()
    for t in used:
        assert (t.data_ptr(), side) in seen


@pytest.mark.parametrize("which", CALLS)
def test_a_call_behind_other_work_outlives_its_arguments(A, which):
    """The inputs are dropped right after the call, and their memory asked for again, while the side stream is still busy
    with something else."""
    want = [t.clone() for t in make(A, which)[0]()]
    torch.cuda.synchronize()
    call, used = make(A, which)
    shapes = [(t.shape, t.dtype) for t in used]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)  # some 50 ms
    got = call(stream=side)
    del call, used
    junk = [torch.full(s, 1, dtype=d, device="cuda") for s, d in shapes for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))
    del junk


@pytest.mark.parametrize("which", CALLS)
def test_results_do_not_take_memory_that_the_current_stream_let_go(A, which):
    """What was dropped on the current stream may still be in use there: a side stream that does not wait must not write
    to it."""
    call, used = make(A, which)
    side = torch.cuda.Stream()
    warm = call()
    made = [t for t in warm if all(t.data_ptr() != u.data_ptr() for u in used)]
    sizes = [(t.untyped_storage().nbytes(), t.untyped_storage().data_ptr()) for t in made]
    assert sizes
    torch.cuda.synchronize()
    let_go = set()
    freed = [torch.empty(n, dtype=torch.uint8, device="cuda") for n, _ in sizes for _ in range(4)]
    for t in freed + made:
        let_go.add(t.untyped_storage().data_ptr())
    del warm, made, freed, t
    got = call(stream=side)
    torch.cuda.current_stream().wait_stream(side)
    for t in got:
        if all(t.data_ptr() != u.data_ptr() for u in used):
            assert t.untyped_storage().data_ptr() not in let_go
