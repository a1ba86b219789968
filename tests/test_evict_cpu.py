"""exl3_cache_evict's refusals, without a GPU (device 99 has no workspace anywhere), and the plain Python eviction its GPU tests
compare with."""
import math

import pytest
import torch

import evict_ref as E
from plugins_b200 import _lib as L
from test_attention_cpu import AT, cache, refused, state
from test_attention_weight_cpu import kv_weight

OLD = dict(refs=AT, table=2 * AT, held=3 * AT, lens=4 * AT)
NEW = dict(refs=5 * AT, table=6 * AT, held=7 * AT, lens=8 * AT)


def weights(**kw):  # [2][2][2][100]
    return kv_weight(**({"layers": 2, "nseq": 2, "layer_stride": 400} | kw))


def evict(c=None, old=None, new=None, w=None, budget=20 * AT, sink=1, recent=2, kept=None, missing=30 * AT):
    return L.lib().exl3_cache_evict(c or cache(device=99), state(**(OLD if old is None else old)), w or weights(), budget, sink,
                                    recent, None, state(**(NEW if new is None else new)), kept or w or weights(), missing)


def test_what_is_served_fails_for_want_of_a_workspace_alone():
    apart = weights(data=600 * AT)
    for kw in (dict(), dict(kept=apart), dict(sink=0, recent=0), dict(sink=2 ** 31 - 1, recent=2 ** 31 - 1),
               dict(kept=weights(data=500 * AT + 3200)), dict(w=weights(row_stride=400, layer_stride=200))):
        refused(evict(**kw), L.EXL3_FAILED, "exl3_kv_register")


@pytest.mark.parametrize("kw,code,text", [
    (dict(c=cache(size=0)), L.EXL3_FAILED, "not a key/value cache"), (dict(old=OLD | dict(size=3)), L.EXL3_FAILED, "not a page state"),
    (dict(new=NEW | dict(refs=None)), L.EXL3_FAILED, "not a page state"), (dict(new=NEW | dict(nseq=3)), L.EXL3_FAILED, "keeps the rows"),
    (dict(old=OLD | dict(nseq=5000), new=NEW | dict(nseq=5000)), L.EXL3_TOO_LARGE, "4096 rows"),
    (dict(sink=-1), L.EXL3_FAILED, "negative counts"), (dict(recent=-1), L.EXL3_FAILED, "negative counts"),
    (dict(w=weights(size=0)), L.EXL3_FAILED, "not a cache's weights"), (dict(w=weights(layers=1)), L.EXL3_FAILED, "other layers"),
    (dict(w=weights(nseq=3)), L.EXL3_FAILED, "other layers"), (dict(kept=weights(slots=99)), L.EXL3_FAILED, "number of slots"),
    (dict(kept=weights(layers=3)), L.EXL3_FAILED, "other layers"), (dict(w=weights(slots=101)), L.EXL3_FAILED, "overlap"),
    (dict(w=weights(layer_stride=399)), L.EXL3_FAILED, "overlap"), (dict(budget=None), L.EXL3_FAILED, "without its arrays"),
    (dict(missing=None), L.EXL3_FAILED, "without its arrays"), (dict(kept=weights(data=500 * AT + 400)), L.EXL3_FAILED, "another layout"),
    (dict(kept=weights(row_stride=400, layer_stride=200)), L.EXL3_FAILED, "another layout"),
    (dict(new=NEW | dict(max_pages=5)), L.EXL3_FAILED, "one width"), (dict(new=NEW | dict(table=2 * AT)), L.EXL3_FAILED, "own arrays"),
    (dict(new=NEW | dict(lens=20 * AT)), L.EXL3_FAILED, "over the call's arguments"),
    (dict(missing=20 * AT + 4), L.EXL3_FAILED, "over the call's arguments"), (dict(missing=7 * AT), L.EXL3_FAILED, "over the call's arguments"),
])
def test_calls_are_refused_by_name(kw, code, text):
    refused(evict(**kw), code, text)


def test_weights_over_the_page_state_are_refused():
    for at in (AT, 2 * AT, 3 * AT, 4 * AT, 5 * AT, 6 * AT, 7 * AT, 8 * AT, 20 * AT, 30 * AT):
        refused(evict(w=weights(data=at)), L.EXL3_FAILED, "over the page state")
        refused(evict(kept=weights(data=at)), L.EXL3_FAILED, "over the page state")


def test_keeping_weights_is_refused_by_name():
    from test_attention_cpu import batch
    keep = (lambda c=None, b=None, path=40 * AT, depth=3, kept=41 * AT, w=None:
            L.lib().exl3_weight_keep(c or cache(device=99), b or batch(nseq=2), path, depth, kept, None, w or weights()))
    refused(keep(), L.EXL3_FAILED, "exl3_kv_register")
    refused(keep(c=cache(size=1)), L.EXL3_FAILED, "not a key/value cache")
    refused(keep(b=batch(size=1)), L.EXL3_FAILED, "not a batch")
    refused(keep(w=weights(nseq=1)), L.EXL3_FAILED, "other layers or rows")
    refused(keep(kept=None), L.EXL3_FAILED, "without its arrays")
    refused(keep(depth=0), L.EXL3_FAILED, "without depth")
    for at in (40 * AT, 41 * AT, AT):
        refused(keep(w=weights(data=at)), L.EXL3_FAILED, "over the call's arguments")
    assert keep(path=None).ok and keep(b=batch(nseq=0, rows=0, max_rows=0), w=weights(nseq=0)).ok


def test_the_plain_eviction():
    w = [0.5, 3.0, math.nan, 0.0, 3.0, 1.0, 2.0, 0.0]
    assert E.kept_slots(w, 8, 3, 0, 0) == [1, 2, 4]
    assert E.kept_slots(w, 8, 2, 0, 0) == [1, 2]
    assert E.kept_slots(w, 8, 4, 1, 1) == [0, 1, 2, 7]
    assert E.kept_slots([0.0] * 6, 6, 3, 0, 1) == [0, 1, 5]
    assert E.kept_slots([math.inf, math.nan, -math.inf, 0.0], 4, 1, 0, 0) == [1]
    k = torch.arange(4 * 16, dtype=torch.float32).view(1, 4, 1, 16, 1)
    weight = torch.zeros((1, 2, 1, 20))
    weight[0, 0, 0, 17], weight[0, 0, 0, 3] = 5.0, 4.0
    # two rows share page 2; the first is cut to 2 tokens of 18
    k2, _, w2, refs, table, held, lens, missing = E.evict(k, k, weight, [0, 1, 2, 0], [[2, 1], [2, -1]], [2, 1], [18, 4], [2, 9], 0, 0)
    assert (refs, table, held, lens, missing) == ([1, 0, 1, 0], [[0, -1], [2, -1]], [1, 1], [2, 4], 0)
    assert k2[0, 0, 0, :2, 0].tolist() == [35.0, 17.0] and torch.equal(k2[0, 1:], k[0, 1:]) and w2[0, 0, 0, :2].tolist() == [4.0, 5.0]
