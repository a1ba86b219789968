"""exl3_draft_verify's refusals, without a GPU: each is named before any launch, and the arrays are device addresses that no
check follows (device 99 has no workspace, here or on a GPU box)."""
import ctypes

import pytest

from plugins_b200 import _lib as L
from test_attention_cpu import AT, batch, cache, refused


def draft(**kw):
    f = dict(size=ctypes.sizeof(L.Draft), vocab=1000, logits_dtype=L.F32, draft_dtype=L.BF16, logits_stride=1000,
             draft_stride=1008, logits=100 * AT, draft=200 * AT, tokens=300 * AT, parent=301 * AT, uniform=302 * AT,
             temperature=303 * AT) | kw
    return L.Draft(**f)


def verify(c=None, b=None, d=None, path=400 * AT, depth=4, kept=401 * AT, token=402 * AT):
    return L.lib().exl3_draft_verify(c or cache(device=99), b or batch(), d or draft(), None, path, depth, kept, token)


def test_what_is_served_fails_for_want_of_a_workspace_alone():
    for d in (draft(), draft(draft=None), draft(parent=None), draft(temperature=None), draft(vocab=1), draft(vocab=393216),
              draft(logits_dtype=L.F16, logits=100 * AT + 2), draft(logits_stride=0)):
        refused(verify(d=d), L.EXL3_FAILED, "exl3_kv_register")


@pytest.mark.parametrize("kw,code,text", [
    (dict(size=0), L.EXL3_FAILED, "not a draft"), (dict(vocab=0), L.EXL3_FAILED, "vocabulary"),
    (dict(vocab=-5), L.EXL3_FAILED, "vocabulary"), (dict(vocab=393217), L.EXL3_TOO_LARGE, "393216"),
    (dict(logits_dtype=L.I32), L.EXL3_UNSUPPORTED, "f16, bf16 or f32"),
    (dict(draft_dtype=L.U16), L.EXL3_UNSUPPORTED, "f16, bf16 or f32"),
    (dict(logits=None), L.EXL3_FAILED, "without its arrays"), (dict(tokens=None), L.EXL3_FAILED, "without its arrays"),
    (dict(uniform=None), L.EXL3_FAILED, "without its arrays"), (dict(logits=100 * AT + 2), L.EXL3_UNSUPPORTED, "multiples"),
    (dict(draft=200 * AT + 1), L.EXL3_UNSUPPORTED, "multiples"),
])
def test_a_draft_is_refused_by_name(kw, code, text):
    refused(verify(d=draft(**kw)), code, text)


def test_batches_caches_and_results_are_refused_by_name():
    refused(verify(c=cache(size=1)), L.EXL3_FAILED, "not a key/value cache")
    refused(verify(b=batch(size=0)), L.EXL3_FAILED, "not a batch")
    refused(verify(b=batch(max_rows=5)), L.EXL3_FAILED, "max_rows")
    refused(verify(b=batch(rows=1025, max_rows=1025)), L.EXL3_TOO_LARGE, "1024")
    refused(verify(b=batch(rows=1025, max_rows=0)), L.EXL3_TOO_LARGE, "1024")  # (no bound given: all rows may be one's)
    refused(verify(b=batch(rows=5000, max_rows=1024)), L.EXL3_FAILED, "exl3_kv_register")
    refused(verify(depth=0), L.EXL3_FAILED, "depth")
    for kw in (dict(path=None), dict(kept=None), dict(token=None)):
        refused(verify(**kw), L.EXL3_FAILED, "without its arrays")
    # four rows of 1000 f32: the last ends 16000 bytes on
    for kw in (dict(path=100 * AT + 15984), dict(kept=200 * AT), dict(token=300 * AT + 12), dict(path=301 * AT - 12),
               dict(kept=302 * AT + 28), dict(token=303 * AT), dict(kept=AT + 4)):
        refused(verify(**kw), L.EXL3_FAILED, "over its arguments")
    for kw in (dict(kept=400 * AT + 12), dict(token=401 * AT), dict(token=400 * AT)):
        refused(verify(**kw), L.EXL3_FAILED, "over one another")
    assert verify(b=batch(nseq=0, rows=0, max_rows=0, row_start=None, context=None, table=None)).ok
