"""The calls that end a step (plugins_b200/attention.py): what they leave alone, and bounds that are not given."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.fixture()
def A():
    from plugins_b200 import attention
    from plugins_b200 import quant as Q
    Q.device_error(0, clear=True)
    yield attention
    assert Q.device_error(0, clear=True) == 0


def keeping(A):
    cache = A.KvCache.empty(3, 40, 16, 2, 64)
    cache.k.zero_(), cache.v.zero_()
    batch = A.TreeBatch(ints([0, 5, 5, 12]), ints([20, 9, 0]), ints([[0, 1, 2], [3, 4, 5], [6, 7, 8]]), max_rows=7, rows=12)
    return cache, batch, ints([[0, 2, 4, -1], [-1] * 4, [0, 1, 3, 6]]), ints([3, 0, 4])


def test_a_refused_keep_moves_no_weights(A):
    cache, batch, path, kept = keeping(A)
    w = torch.rand((3, 3, 2, 40), generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    before = w.clone()
    row_start, context, table = batch._keep[:3]
    both = torch.cat([kept, kept])
    for out, k in ((row_start[1:], kept), (table.view(-1)[3:6], kept), (path.view(-1)[:3], kept), (both[1:4], both[:3])):
        with pytest.raises(A.Exl3Error, match="lens lies over"):
            A.cache_keep(cache, batch, path, k, out=out, weight=w)
        assert torch.equal(w, before)
    assert A.cache_keep(cache, batch, path, kept, out=kept, weight=w) is kept and kept.tolist() == [23, 9, 4]
    assert not torch.equal(w, before)


def test_kept_weights_stay_inside_their_slots(A):
    """Weights as a strided part of a larger pool: what lies around each head's slots, and other rows, stay."""
    cache, batch, path, kept = keeping(A)
    pool = torch.rand((2, 3, 4, 57), generator=torch.Generator("cuda").manual_seed(2), device="cuda")  # [head][layer][row][slot]
    want = pool.clone()
    want[:, :, 0, 9 + 20:9 + 23] = pool[:, :, 0, [29, 31, 33]]
    want[:, :, 2, 9:13] = pool[:, :, 2, [9, 10, 12, 15]]
    A.cache_keep(cache, batch, path, kept, weight=pool.permute(1, 2, 0, 3)[:, :3, :, 9:49])
    assert torch.equal(pool, want)


def test_paths_are_as_deep_as_the_rows_where_no_bound_is_given(A):
    cache = A.KvCache.empty(1, 4, 16, 1, 64)
    n, vocab = 6, 50
    tokens = ints([3, 8, 1, 30, 7, 2, 40, 41])  # a chain that the model agrees with, then another sequence's one draft
    logits = torch.zeros((n + 2, vocab), device="cuda")
    logits[torch.arange(n - 1), tokens[1:n].long()] = 5.0
    logits[n - 1, 11], logits[n, 41], logits[n + 1, 9] = 5.0, 5.0, 5.0
    uniform = torch.full((n + 2, 2), 0.5, device="cuda")
    got = []
    for most in (n, 0):
        batch = A.TreeBatch(ints([0, n, n + 2]), ints([0, 0]), ints([[0], [1]]), max_rows=most, rows=n + 2)
        got.append(A.draft_verify(cache, batch, logits, tokens, None, uniform, torch.zeros(2, device="cuda")))
    for path, kept, token in got:
        assert kept.tolist() == [n, 2] and token.tolist() == [11, 9]
        assert path[0, :n].tolist() == list(range(n)) and path[1, :2].tolist() == [0, 1] and path[1, 2] == -1
