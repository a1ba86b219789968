"""exl3_attention_weight where one CTA has many query tiles, some of whose key blocks hold 128 keys or fewer: hundreds of
short contexts, causal prompts and trees whose last block is half empty.  Against the formula in 64 bits, with
tests/evict_ref.py's tolerance, and the same bits again; no device error."""
import numpy as np
import pytest
import torch

import evict_ref as E
from test_attention_gpu import A, Step, random_tree  # noqa: F401  (A: a fixture, which asserts that no error is recorded)
from test_attention_weight_gpu import check, queries

pytestmark = pytest.mark.gpu


def visible(ntok, ctx, keys, tree_rows=None, words=0):
    """tests/attention_ref.py's, for thousands of rows."""
    see = np.ones((ntok, keys), dtype=bool)
    if tree_rows is None:
        see[:, ctx:] = np.arange(keys - ctx) <= np.arange(ntok)[:, None]
    else:
        bits = np.unpackbits(tree_rows.numpy().view(np.uint8), axis=1, bitorder="little")
        see[:, ctx:] = bits[:, :keys - ctx]
    return torch.from_numpy(see)


@pytest.fixture(autouse=True)
def quick(monkeypatch):
    monkeypatch.setattr(E.R, "visible", visible)


def twice(A, step, heads, kvh, dim, pad=0):
    q = queries(step, heads, dim, pad=pad)
    cache, batch, q, lse, old, w = check(A, step, heads, kvh, dim, 0.9, q=q)
    again = A.attention_weight(cache, step.layer, batch, q, lse, old.cuda(), decay=0.9)
    assert torch.equal(again, w)


@pytest.mark.parametrize("heads,kvh,dim,dtype", [(8, 8, 64, "bf16"), (8, 8, 128, "bf16"), (8, 8, 256, "f16"), (16, 4, 128, "f16"), (32, 32, 128, "bf16")])
@pytest.mark.parametrize("most", [127, 300])
@pytest.mark.parametrize("pad", [0, 1])
def test_one_token_each_of_hundreds_of_short_sequences(A, heads, kvh, dim, dtype, most, pad):
    lens = [(37 * i + i // 7) % (most + 1) for i in range(256)]
    twice(A, Step([1] * 256, lens, kvh, dim, 16, dtype, layers=1), heads, kvh, dim, pad)


@pytest.mark.parametrize("rows,ctx,heads,kvh,dim", [
    (2000, 916, 24, 2, 128), (1900, 1044, 32, 2, 128), (2188, 500, 16, 2, 64), (2600, 78, 8, 1, 64), (1500, 146, 16, 2, 256)])
@pytest.mark.parametrize("pad", [0, 1])
def test_prompts_whose_last_block_is_half_empty(A, rows, ctx, heads, kvh, dim, pad):
    assert dim == 256 or 100 <= (rows + ctx) % 256 <= 128
    twice(A, Step([rows], [ctx], kvh, dim, 64, "bf16", layers=1), heads, kvh, dim, pad)


@pytest.mark.parametrize("rows,ctx,heads,kvh,dim", [(400, 14300, 8, 2, 128), (300, 14150, 8, 1, 64), (400, 4000, 8, 2, 256), (321, 15140, 16, 2, 128)])
def test_trees_of_hundreds_of_rows(A, rows, ctx, heads, kvh, dim):
    twice(A, Step([rows], [ctx], kvh, dim, 64, "f16", tree=random_tree, layers=1), heads, kvh, dim)


def test_short_and_long_sequences_by_turns(A):
    """Items of one and of many row tiles, of one half and of two, on one CTA's part."""
    rows = [1, 40, 1, 1, 3, 200, 1, 0, 9] * 20
    lens = [(53 * i) % 400 for i in range(len(rows))]
    for heads, kvh, dim in ((16, 2, 128), (16, 2, 64), (8, 1, 256)):
        twice(A, Step(rows, lens, kvh, dim, 16, "bf16", layers=1), heads, kvh, dim)
