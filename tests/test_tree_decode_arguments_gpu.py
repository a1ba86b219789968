"""What the decoder (plugins_b200/tree_decode.py) refuses before anything changes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_arguments_that_name_no_row_or_token():
    from plugins_b200 import tree_decode as T
    layers = T.random_layers(1, 256, 4, 2, 64, 512, seed=1)
    embed = torch.randn((64, 256), generator=torch.Generator("cuda").manual_seed(1), device="cuda").bfloat16()
    dec = T.TreeDecoder(layers, embed, 4, 2, 64, pages=16, page_size=16, nseq=2, max_pages=4)
    for prompts in ([[1, 2]], [[1], []], [[1], [2], [3]]):
        with pytest.raises(ValueError, match="prompt"):
            dec.prompt(prompts)
    dec.prompt([[1, 2, 3], [4]])
    before = (list(dec.lens), list(dec.last), dec.state.table.tolist())
    for trees in ([[]], [[], [(0, 5)]], [[(-2, 5)], []], [[(-1, 1), (1, 2)], []]):
        with pytest.raises(ValueError, match="tree"):
            dec.step(trees)
    for parent in ([-1, 0], [0, 2]):
        with pytest.raises(ValueError, match="parents"):
            dec.reorder(parent)
    assert before == (dec.lens, dec.last, dec.state.table.tolist())
    dec.reorder([1, 1])
    assert len(dec.step([[(-1, 3), (0, 4)], []])) == 2
