"""The operators together: decoding with drafted trees gives what decoding one token at a time gives
(plugins_b200/tree_decode.py)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, HIDDEN, VOCAB = 8, 2, 128, 512, 512


def build(T, nseq):
    layers = T.random_layers(2, HIDDEN, HEADS, KV, DIM, 1024, seed=3)
    embed = torch.randn((VOCAB, HIDDEN), generator=torch.Generator("cuda").manual_seed(1), device="cuda").bfloat16()
    return lambda: T.TreeDecoder(layers, embed, HEADS, KV, DIM, pages=80, page_size=16, nseq=nseq, max_pages=16)


def test_drafted_trees_decode_as_single_tokens_do():
    from plugins_b200 import quant as Q
    from plugins_b200 import tree_decode as T
    make = build(T, 3)
    prompts = [[(5 * i + s) % VOCAB for i in range(n)] for s, n in enumerate((1, 17, 90))]
    plain = make()
    first = plain.prompt(prompts)
    want = [[], [], []]
    for _ in range(12):
        for w, g in zip(want, plain.step([[], [], []])):
            assert len(g) == 1
            w += g
    dec, got, steps = make(), [[], [], []], 0
    assert dec.prompt(prompts) == first
    while min(map(len, got)) < 12:
        trees = []
        for w, g in zip(want, got):
            right = w[len(g):len(g) + 3]
            wrong = [(-1, (right[0] + 1) % VOCAB)] if right else []
            trees.append(wrong + [(i - 1 + len(wrong) if i else -1, t) for i, t in enumerate(right)])
        for g, new in zip(got, dec.step(trees)):
            g += new
        steps += 1
    assert [g[:12] for g in got] == want and steps == 3  # three right drafts and the model's own next token a step
    assert dec.state.lens.tolist() == dec.lens
    assert Q.device_error(0, clear=True) == 0


def test_a_forked_sequence_decodes_as_its_parent_and_rows_give_pages_back():
    from plugins_b200 import attention as A
    from plugins_b200 import tree_decode as T
    make = build(T, 2)
    dec = make()
    dec.prompt([[1, 2, 3, 4, 5], list(range(40))])
    dec.step([[], []])
    used = int((dec.state.refs > 0).sum())
    dec.reorder([1, 1])  # sequence 0 ends, sequence 1 goes on twice
    assert int((dec.state.refs > 0).sum()) < used and dec.lens[0] == dec.lens[1] == 41
    for _ in range(12):
        a, b = dec.step([[], []])
        assert a == b
    assert dec.state.table[0].tolist() != dec.state.table[1].tolist()  # their own last pages
    dec.state = A.cache_compact(dec.cache, dec.state)
    live = int((dec.state.refs > 0).sum())
    assert bool((dec.state.refs[:live] > 0).all())
    a, b = dec.step([[], []])
    assert a == b
