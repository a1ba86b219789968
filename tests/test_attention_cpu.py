"""The attention side's refusals (include/exl3_b200.h), without a GPU: each is named before any launch, and the arrays
are device addresses that no check follows.  The 64-bit formulas the GPU tests compare with are checked here against
differences and identities of their own."""
import ctypes
import math

import pytest
import torch

import attention_ref as R
from plugins_b200 import _lib as L

AT = 1 << 20  # some aligned address; no refusal reads it


def cache(**kw):
    f = dict(size=ctypes.sizeof(L.KvCache), device=0, dtype=L.BF16, layers=2, pages=8, page_size=16, kv_heads=2,
             head_dim=64, k=AT, v=AT, layer_stride=8 * 2 * 16 * 64, page_stride=2 * 16 * 64, head_stride=16 * 64,
             token_stride=64) | kw
    return L.KvCache(**f)


def batch(**kw):
    f = dict(size=ctypes.sizeof(L.TreeBatch), nseq=1, rows=4, max_rows=4, max_context=0, max_pages=4, tree_words=0,
             row_start=AT, context=AT, table=AT, tree=None, position=None) | kw
    return L.TreeBatch(**f)


def heads(**kw):
    f = dict(data=AT, dtype=L.BF16, rows=4, heads=2, dim=64, row_stride=128, head_stride=64) | kw
    return L.Heads(**f)


def rope(**kw):
    f = dict(size=ctypes.sizeof(L.NormRope), rot_dims=64, adjacent=0, weight_dtype=L.BF16, eps=1e-6, weight_offset=0.0,
             q_weight=AT, k_weight=AT, inv_freq=AT) | kw
    return L.NormRope(**f)


def state(**kw):
    f = dict(size=ctypes.sizeof(L.PageState), nseq=2, max_pages=4, refs=AT, table=AT, held=AT, lens=AT) | kw
    return L.PageState(**f)


def refused(v, code, text):
    assert v.code == code and text in v.message(), (v.code, v.message())


@pytest.mark.parametrize("kw,code,text", [
    (dict(size=4), L.EXL3_FAILED, "not a key/value cache"), (dict(k=None), L.EXL3_FAILED, "not a key/value cache"),
    (dict(dtype=L.F32), L.EXL3_UNSUPPORTED, "f16 or bf16"), (dict(head_dim=96), L.EXL3_UNSUPPORTED, "head_dim"),
    (dict(page_size=8), L.EXL3_UNSUPPORTED, "page_size"), (dict(page_size=48), L.EXL3_UNSUPPORTED, "page_size"),
    (dict(page_size=512), L.EXL3_UNSUPPORTED, "page_size"), (dict(pages=0), L.EXL3_FAILED, "empty"),
    (dict(pages=1 << 23), L.EXL3_TOO_LARGE, "pages"), (dict(kv_heads=2000), L.EXL3_TOO_LARGE, "kv heads"),
    (dict(v=AT + 8), L.EXL3_UNSUPPORTED, "aligned"), (dict(token_stride=68), L.EXL3_UNSUPPORTED, "aligned"),
    (dict(token_stride=32), L.EXL3_FAILED, "overlap"), (dict(page_stride=0), L.EXL3_FAILED, "overlap"),
    (dict(head_stride=15 * 64), L.EXL3_FAILED, "overlap"),
])
def test_a_cache_is_refused_by_name(kw, code, text):
    c = cache(**kw)
    refused(L.lib().exl3_kv_register(c), code, text)
    refused(L.lib().exl3_tree_attention(c, 0, batch(), heads(), 0.1, None, heads(), None), code, text)
    refused(L.lib().exl3_cache_compact(c, state(), None, state(refs=AT * 2)), code, text)


def test_pages_of_token_major_pools_are_served():
    # [pages][token][head] rows: no GPU here, so what follows the checks is refused for want of one
    v = L.lib().exl3_kv_register(cache(head_stride=64, token_stride=128, device=99))
    refused(v, L.EXL3_UNSUPPORTED, "device index")


@pytest.mark.parametrize("kw,code,text", [
    (dict(size=0), L.EXL3_FAILED, "not a batch"), (dict(nseq=-1), L.EXL3_FAILED, "negative"),
    (dict(rows=-4), L.EXL3_FAILED, "negative"), (dict(nseq=70000), L.EXL3_TOO_LARGE, "sequences"),
    (dict(table=None), L.EXL3_FAILED, "lacks its arrays"), (dict(max_pages=0), L.EXL3_FAILED, "lacks its arrays"),
    (dict(tree=AT), L.EXL3_FAILED, "without words"), (dict(rows=1 << 25), L.EXL3_TOO_LARGE, "rows"),
])
def test_a_batch_is_refused_by_name(kw, code, text):
    b = batch(**kw)
    refused(L.lib().exl3_tree_attention(cache(), 0, b, heads(), 0.1, None, heads(), None), code, text)
    refused(L.lib().exl3_qk_norm_rope(cache(), 0, b, heads(), heads(), heads(), rope(), None, heads()), code, text)
    refused(L.lib().exl3_cache_keep(cache(), b, AT, 4, AT, None, AT), code, text)


@pytest.mark.parametrize("q,out,scale,layer,code,text", [
    (dict(rows=5), {}, 1, 0, L.EXL3_FAILED, "q is"), (dict(dim=128), {}, 1, 0, L.EXL3_FAILED, "q is"),
    (dict(data=None), {}, 1, 0, L.EXL3_FAILED, "q is"), ({}, dict(rows=3), 1, 0, L.EXL3_FAILED, "out is"),
    (dict(dtype=L.F16), {}, 1, 0, L.EXL3_UNSUPPORTED, "cache's dtype"),
    (dict(dtype=L.F32), {}, 1, 0, L.EXL3_UNSUPPORTED, "cache's dtype"),
    (dict(heads=3), dict(heads=3), 1, 0, L.EXL3_FAILED, "per kv head"),
    (dict(heads=4), dict(heads=2), 1, 0, L.EXL3_FAILED, "per kv head"),
    ({}, {}, 0.0, 0, L.EXL3_UNSUPPORTED, "scale"), ({}, {}, -1.0, 0, L.EXL3_UNSUPPORTED, "scale"),
    ({}, {}, math.nan, 0, L.EXL3_UNSUPPORTED, "scale"), ({}, {}, math.inf, 0, L.EXL3_UNSUPPORTED, "scale"),
    ({}, dict(head_stride=0), 1, 0, L.EXL3_FAILED, "overlap"), ({}, dict(row_stride=64), 1, 0, L.EXL3_FAILED, "overlap"),
    ({}, dict(head_stride=63), 1, 0, L.EXL3_FAILED, "overlap"),
    ({}, {}, 1, 2, L.EXL3_FAILED, "layer"), ({}, {}, 1, -1, L.EXL3_FAILED, "layer"),
])
def test_attention_is_refused_by_name(q, out, scale, layer, code, text):
    refused(L.lib().exl3_tree_attention(cache(), layer, batch(), heads(**q), scale, None, heads(**out), None), code, text)


@pytest.mark.parametrize("q,k,v,o,opts,code,text", [
    (dict(dim=32), {}, {}, {}, {}, L.EXL3_FAILED, "q is"), ({}, dict(rows=1), {}, {}, {}, L.EXL3_FAILED, "k is"),
    ({}, {}, dict(dim=8), {}, {}, L.EXL3_FAILED, "v is"), ({}, dict(heads=1), {}, {}, {}, L.EXL3_FAILED, "kv heads"),
    ({}, {}, {}, dict(heads=4), {}, L.EXL3_FAILED, "q's heads"),
    (dict(dtype=L.I32), {}, {}, {}, {}, L.EXL3_UNSUPPORTED, "f16, bf16 or f32"),
    (dict(dtype=L.F32), {}, {}, {}, {}, L.EXL3_UNSUPPORTED, "one dtype"),
    ({}, {}, {}, dict(dtype=L.F16), {}, L.EXL3_UNSUPPORTED, "q_out"),
    ({}, {}, {}, dict(dtype=L.F32), {}, L.EXL3_UNSUPPORTED, "q_out"),
    ({}, {}, {}, dict(row_stride=0), {}, L.EXL3_FAILED, "overlap"),
    ({}, {}, {}, dict(row_stride=512), {}, L.EXL3_FAILED, "another layout"),
    ({}, {}, {}, {}, dict(size=1), L.EXL3_FAILED, "options"), ({}, {}, {}, {}, dict(rot_dims=66), L.EXL3_UNSUPPORTED, "rot_dims"),
    ({}, {}, {}, {}, dict(rot_dims=24), L.EXL3_UNSUPPORTED, "rot_dims"),
    ({}, {}, {}, {}, dict(rot_dims=7, adjacent=1), L.EXL3_UNSUPPORTED, "rot_dims"),
    ({}, {}, {}, {}, dict(inv_freq=None), L.EXL3_FAILED, "frequencies"),
    ({}, {}, {}, {}, dict(weight_dtype=L.I32), L.EXL3_UNSUPPORTED, "weights"),
    ({}, {}, {}, {}, dict(eps=-1.0), L.EXL3_FAILED, "eps"), ({}, {}, {}, {}, dict(eps=math.nan), L.EXL3_FAILED, "eps"),
])
def test_norm_rope_is_refused_by_name(q, k, v, o, opts, code, text):
    refused(L.lib().exl3_qk_norm_rope(cache(), 0, batch(), heads(**q), heads(**k), heads(**v), rope(**opts), None,
                                      heads(**o)), code, text)


def test_page_calls_are_refused_by_name():
    lib = L.lib()
    other = dict(refs=2 * AT, table=2 * AT, held=2 * AT, lens=2 * AT)
    for a, b, text in ((dict(size=1), other, "not a page state"), ({}, other | dict(refs=None), "not a page state"),
                       ({}, other | dict(max_pages=5), "one width"), ({}, other | dict(table=AT), "own arrays"),
                       ({}, other | dict(refs=AT), "own arrays")):
        refused(lib.exl3_cache_fork(cache(), state(**a), AT, None, state(**b)), L.EXL3_FAILED, text)
        refused(lib.exl3_cache_grow(cache(), state(**a), AT, None, state(**b), AT), L.EXL3_FAILED, text)
        refused(lib.exl3_cache_compact(cache(), state(**a), None, state(**b)), L.EXL3_FAILED, text)
    # a cache that was not registered has no workspace
    refused(lib.exl3_cache_fork(cache(), state(), AT, None, state(**other)), L.EXL3_FAILED, "exl3_kv_register")
    refused(lib.exl3_cache_keep(cache(), batch(), AT, 0, AT, None, AT), L.EXL3_FAILED, "without depth")
    refused(lib.exl3_cache_keep(cache(), batch(), AT, 1, None, None, AT), L.EXL3_FAILED, "without its arrays")
    refused(lib.exl3_tree_attention(cache(), 0, batch(), heads(), 1.0, None, heads(data=2 * AT), None), L.EXL3_FAILED,
            "exl3_kv_register")
    refused(lib.exl3_tree_attention(cache(), 0, batch(), heads(), 1.0, None, heads(), None), L.EXL3_FAILED, "out is not q")
    refused(lib.exl3_tree_attention(cache(), 0, batch(max_rows=5), heads(), 1.0, None, heads(data=2 * AT), None),
            L.EXL3_FAILED, "max_rows")


def test_nothing_to_do_is_not_an_error():
    lib = L.lib()
    none = batch(nseq=0, rows=0, max_rows=0, row_start=None, context=None, table=None)
    h = heads(rows=0, data=None)
    assert lib.exl3_tree_attention(cache(), 0, none, h, 1.0, None, h, None).ok
    assert lib.exl3_qk_norm_rope(cache(), 0, none, h, h, h, rope(), None, h).ok
    assert lib.exl3_cache_keep(cache(), none, AT, 1, AT, None, AT).ok


# ------------------------------------------------------------------ the formulas themselves

def test_the_rotation_keeps_lengths_and_relative_angles():
    g = torch.Generator().manual_seed(0)
    x, y = (torch.randn((1, 1, 32), generator=g, dtype=torch.float64) for _ in range(2))
    inv = 100.0 ** (-torch.arange(16, dtype=torch.float64) / 16)
    for adjacent in (False, True):
        turn = (lambda z, p: R.norm_rotate(z, None, torch.tensor([p]), inv, 0, adjacent))
        assert abs(float((turn(x, 7) ** 2).sum() - (x ** 2).sum())) < 1e-12
        a, b = float((turn(x, 9) * turn(y, 4)).sum()), float((turn(x, 105) * turn(y, 100)).sum())
        assert abs(a - b) < 1e-11


def test_the_attention_formula_against_a_direct_sum():
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn((2, 1, 16, 8), generator=g, dtype=torch.float64) for _ in range(2))
    q = torch.randn((2, 1, 8), generator=g, dtype=torch.float64)
    out, lse, _ = R.attention(k, v, q, [0, 2], [15], torch.tensor([[1, 0]]), 0.5)
    keys = [(1, i) for i in range(16)] + [(0, 0)]
    for row, n in ((0, 16), (1, 17)):
        e = [math.exp(0.5 * float(q[row, 0] @ k[p, 0, o])) for p, o in keys[:n]]
        want = sum(x * v[p, 0, o] for x, (p, o) in zip(e, keys)) / sum(e)
        assert float((out[row, 0] - want).abs().max()) < 1e-13
        assert abs(float(lse[row, 0]) - math.log(sum(e))) < 1e-13
