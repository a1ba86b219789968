"""exl3_attention_weight's refusals, without a GPU (device 99 has no workspace anywhere), and the formula its GPU tests compare
with."""
import ctypes
import math

import pytest
import torch

import attention_ref as R
import evict_ref as E
from plugins_b200 import _lib as L
from test_attention_cpu import AT, batch, cache, heads, refused


def kv_weight(**kw):
    f = dict(size=ctypes.sizeof(L.KvWeight), layers=1, nseq=1, slots=100, data=500 * AT, layer_stride=200, row_stride=200,
             head_stride=100) | kw
    return L.KvWeight(**f)


def packed(**kw):
    return bytes(heads(**({"data": 600 * AT} | kw)))


def call(c=None, layer=0, b=None, q=None, scale=0.1, lse=700 * AT, decay=1.0, w=None):
    return L.lib().exl3_attention_weight(c or cache(device=99), layer, b or batch(), packed() if q is None else q, scale, lse,
                                         decay, None, w or kv_weight())


def test_what_is_served_fails_for_want_of_a_workspace_alone():
    for kw in (dict(), dict(decay=0.0), dict(w=kv_weight(row_stride=0)), dict(w=kv_weight(head_stride=1000)),
               dict(q=packed(heads=6, row_stride=0, head_stride=0)), dict(b=batch(tree=800 * AT, tree_words=1)),
               dict(c=cache(device=99, dtype=L.F16), q=packed(dtype=L.F16))):
        refused(call(**kw), L.EXL3_FAILED, "exl3_kv_register")


@pytest.mark.parametrize("kw,code,text", [
    (dict(size=0), L.EXL3_FAILED, "not a cache's weights"), (dict(data=None), L.EXL3_FAILED, "not a cache's weights"),
    (dict(layers=2), L.EXL3_FAILED, "other layers or rows"), (dict(nseq=2), L.EXL3_FAILED, "other layers or rows"),
    (dict(slots=0), L.EXL3_FAILED, "without slots"), (dict(data=500 * AT + 2), L.EXL3_UNSUPPORTED, "multiples of 4"),
    (dict(slots=(1 << 30) + 1), L.EXL3_TOO_LARGE, "2^30"), (dict(head_stride=99), L.EXL3_FAILED, "overlap"), (dict(head_stride=0), L.EXL3_FAILED, "overlap"),
    (dict(head_stride=-100), L.EXL3_FAILED, "overlap"),
])
def test_weights_are_refused_by_name(kw, code, text):
    refused(call(w=kv_weight(**kw)), code, text)


@pytest.mark.parametrize("kw,code,text", [
    (dict(layer=2), L.EXL3_FAILED, "layer"), (dict(layer=-1), L.EXL3_FAILED, "layer"),
    (dict(c=cache(size=3)), L.EXL3_FAILED, "not a key/value cache"), (dict(b=batch(size=0)), L.EXL3_FAILED, "not a batch"),
    (dict(b=batch(max_rows=9)), L.EXL3_FAILED, "max_rows"), (dict(q=packed(rows=3)), L.EXL3_FAILED, "q is"),
    (dict(q=packed(dim=128)), L.EXL3_FAILED, "q is"), (dict(q=packed(dtype=L.F32)), L.EXL3_UNSUPPORTED, "cache's dtype"),
    (dict(q=packed(heads=3)), L.EXL3_FAILED, "per kv head"), (dict(q=packed(heads=4098)), L.EXL3_TOO_LARGE, "4096"),
    (dict(scale=0.0), L.EXL3_UNSUPPORTED, "scale"), (dict(scale=-1.0), L.EXL3_UNSUPPORTED, "scale"),
    (dict(scale=math.nan), L.EXL3_UNSUPPORTED, "scale"), (dict(scale=math.inf), L.EXL3_UNSUPPORTED, "scale"),
    (dict(decay=-0.1), L.EXL3_UNSUPPORTED, "decay"), (dict(decay=1.5), L.EXL3_UNSUPPORTED, "decay"),
    (dict(decay=math.nan), L.EXL3_UNSUPPORTED, "decay"), (dict(lse=None), L.EXL3_FAILED, "log-sum-exp"),
])
def test_calls_are_refused_by_name(kw, code, text):
    refused(call(**kw), code, text)


def test_weights_over_the_arguments_are_refused():
    # [1][2][100] f32: 800 bytes; four rows of two heads: q 1024 bytes, lse 32
    for at in (600 * AT, 600 * AT + 1020, 700 * AT + 28, 700 * AT - 796, AT):
        refused(call(w=kv_weight(data=at)), L.EXL3_FAILED, "over the call's arguments")
    refused(call(w=kv_weight(data=700 * AT - 800)), L.EXL3_FAILED, "exl3_kv_register")
    tree = batch(tree=800 * AT, tree_words=3)
    refused(call(b=tree, w=kv_weight(data=800 * AT + 44)), L.EXL3_FAILED, "over the call's arguments")


def test_nothing_to_do_is_not_an_error():
    none = batch(nseq=0, rows=0, max_rows=0, row_start=None, context=None, table=None)
    assert call(b=none, q=packed(rows=0, data=None), lse=None, w=kv_weight(nseq=0, data=None)).ok


def test_the_formula_against_a_direct_sum_and_the_attention():
    g = torch.Generator().manual_seed(5)
    k = torch.randn((3, 2, 16, 8), generator=g, dtype=torch.float64)
    q = torch.randn((3, 4, 8), generator=g, dtype=torch.float64)
    table = torch.tensor([[2, 0, 1]])
    _, lse, _ = R.attention(k, k, q, [0, 3], [30], table, 0.5)
    old = torch.rand((1, 2, 40), generator=g)
    got, _ = E.weights(k, q, lse, [0, 3], [30], table, 0.5, 0.25, old)
    for h in range(2):
        for j in range(33):
            kj = k[int(table[0, j // 16]), h, j % 16]
            want = 0.25 * float(old[0, h, j]) if j < 30 else 0.0
            for i in range(3):
                if j <= 30 + i:
                    want += sum(math.exp(0.5 * float(q[i, 2 * h + e] @ kj) - float(lse[i, 2 * h + e])) for e in (0, 1))
            assert abs(float(got[0, h, j]) - want) < 1e-12
        assert float((got[0, h, :33].sum() - 0.25 * old[0, h, :30].double().sum() - 6).abs()) < 1e-12  # three rows of two heads
    assert torch.equal(got[:, :, 33:], old[:, :, 33:].double())
