"""The decoder (plugins_b200/tree_decode.py) beyond what draft_verify serves, and where no token has a probability."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, HIDDEN = 2, 1, 128, 256


@pytest.fixture(scope="module")
def make():
    from plugins_b200 import tree_decode as T
    layers = T.random_layers(1, HIDDEN, HEADS, KV, DIM, 512, seed=3)

    def build(vocab, nseq=1, poison=None, **kw):
        embed = torch.randn((vocab, HIDDEN), generator=torch.Generator("cuda").manual_seed(1), device="cuda").bfloat16()
        if poison is not None:
            embed[poison] = math.nan
        return T.TreeDecoder(layers, embed, HEADS, KV, DIM, pages=100, page_size=64, nseq=nseq, max_pages=40, **kw)
    return build


def test_a_greedy_tree_of_more_than_1024_rows(make):
    plain, dec = make(300), make(300)
    prompt = [[5, 9, 250]]
    assert plain.prompt(prompt) == dec.prompt(prompt)
    want = [plain.step([[]])[0][0] for _ in range(3)]
    tree = [(-1, t) for t in range(300) if t != want[0]] * 4  # 1196 wrong drafts, then two right ones
    tree += [(-1, want[0]), (len(tree), want[1])]
    assert len(tree) > 1024 and dec.step([tree])[0] == want
    assert dec.lens == plain.lens == [6] and dec.state.lens.tolist() == [6]


def test_a_greedy_vocabulary_of_more_than_393216(make):
    plain, dec = make(400000), make(400000)
    assert plain.prompt([[399999, 4]]) == dec.prompt([[399999, 4]])
    want = [plain.step([[]])[0][0] for _ in range(3)]
    assert dec.step([[(-1, want[0]), (-1, 3), (0, want[1])]])[0] == want


def test_sampling_from_logits_without_a_number_says_so_and_changes_nothing(make):
    dec = make(300, nseq=2, poison=7, temperature=50.0, seed=1)
    dec.prompt([[1, 2], [3, 4]])
    dec.last[1] = 7  # its hidden state is NaN, and all of its logits
    before = (list(dec.lens), list(dec.seen), list(dec.last), dec.state.lens.tolist())
    with pytest.raises(RuntimeError, match="sequence 1"):
        dec.step([[(-1, 3)], []])
    assert before == (dec.lens, dec.seen, dec.last, dec.state.lens.tolist())
    dec.last[1] = 8
    assert [len(g) >= 1 for g in dec.step([[], [(-1, 2)]])] == [True, True]
