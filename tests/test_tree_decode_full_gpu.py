"""The decoder (plugins_b200/tree_decode.py) on a budget when its cache is nearly full of shared pages."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, HIDDEN, VOCAB, PAGE = 8, 2, 128, 512, 512, 16


@pytest.fixture(scope="module")
def make():
    from plugins_b200 import tree_decode as T
    layers = T.random_layers(2, HIDDEN, HEADS, KV, DIM, 1024, seed=3)
    embed = torch.randn((VOCAB, HIDDEN), generator=torch.Generator("cuda").manual_seed(1), device="cuda").bfloat16()
    return lambda pages: T.TreeDecoder(layers, embed, HEADS, KV, DIM, pages=pages, page_size=PAGE, nseq=2, max_pages=16,
                                       budget=40, sink=2, recent=8)


def test_forks_are_cut_one_after_the_other_where_pages_are_few(make):
    """Two rows of 49 tokens share their first two pages: cut together they ask for four free pages, of eight in all; one
    after the other for two."""
    few, many = make(8), make(40)
    out = []
    for dec in (few, many):
        out.append([dec.prompt([[3], [(5 * i + 1) % VOCAB for i in range(40)]])])
        dec.reorder([1, 1])
        for n in range(30):
            out[-1].append(dec.step([[(-1, n)], []]))
            out[-1].append(list(dec.lens))
        assert dec.state.lens.tolist() == dec.lens and max(dec.lens) <= 48
        refs = [0] * dec.cache.pages
        for row, held in zip(dec.state.table.tolist(), dec.state.held.tolist()):
            for p in row[:held]:
                refs[p] += 1
        assert dec.state.refs.tolist() == refs
    assert out[0] == out[1]


def test_rows_that_cannot_be_cut_keep_their_tokens(make):
    """One page short even for one row: the step's tokens are returned, the rows go on, and evict() says what is lacking."""
    few, many = make(7), make(40)
    for dec in (few, many):
        dec.prompt([[3], [(5 * i + 1) % VOCAB for i in range(40)]])
        dec.reorder([1, 1])
    for n in range(12):
        a, b = few.step([[], []]), many.step([[], []])
        assert [len(g) for g in a] == [1, 1]
        if few.lens[0] <= 48:
            assert a == b
    assert few.lens == [52, 52] and few.state.lens.tolist() == [52, 52] and many.lens[0] < 52
    before = few.weight.clone()
    with pytest.raises(RuntimeError, match="lacks"):
        few.evict()
    assert few.lens == [52, 52] and torch.equal(few.weight.view(torch.int32), before.view(torch.int32))
    few.reorder([1])  # the other row ends: the rest is its own, and is cut
    few.evict()
    assert few.lens == [40]
