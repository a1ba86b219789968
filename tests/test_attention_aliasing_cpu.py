"""Results that lie over what a call still reads are refused by name, those that lie beside it are served
(include/exl3_b200.h); the checks come before any launch, on addresses that nothing follows."""
import random

import pytest

from plugins_b200 import _lib as L
from test_attention_cpu import AT, batch, cache, heads, refused, rope, state

SERVED = "exl3_kv_register"  # what stops a call that passed its checks: device 99 has no workspace, on any machine


def attention(q, out, lse=None, rows=4):
    return L.lib().exl3_tree_attention(cache(device=99), 0, batch(rows=rows, max_rows=rows), q, 0.1, None, out, lse)


def append(q, k, v, out, rows=4):
    return L.lib().exl3_qk_norm_rope(cache(device=99), 0, batch(rows=rows, max_rows=rows), q, k, v, rope(), None, out)


def addresses(h):
    size = 4 if h.dtype == L.F32 else 2
    return {h.data + (r * h.row_stride + c * h.head_stride) * size + e
            for r in range(h.rows) for c in range(h.heads) for e in range(0, h.dim * size, 2)}


@pytest.mark.parametrize("offset,text", [(0, "out is not q"), (128, "out is not q"), (-2, "out is not q"), (1022, "out is not q"),
                                         (1024, SERVED), (-1024, SERVED), (-1022, "out is not q")])
def test_out_shifted_into_q(offset, text):
    refused(attention(heads(), heads(data=AT + offset)), L.EXL3_FAILED, text)


@pytest.mark.parametrize("at,text", [(0, "lse lies over"), (1020, "lse lies over"), (1024, SERVED), (-32, SERVED), (-28, "lse lies over"),
                                     (4096, "lse lies over"), (4096 + 1024, SERVED)])
def test_lse_over_q_or_out(at, text):
    refused(attention(heads(), heads(data=AT + 4096), AT + at), L.EXL3_FAILED, text)


def test_slices_of_one_row_buffer():
    """q, k, v and a result as head slices of rows of 8 heads: beside one another served, over one another refused."""
    def part(first, n):
        return heads(data=AT + first * 128, heads=n, row_stride=8 * 64)
    refused(append(part(0, 4), part(4, 2), part(6, 2), part(0, 4)), L.EXL3_FAILED, SERVED)  # in place
    refused(append(part(0, 2), part(4, 2), part(6, 2), part(2, 2)), L.EXL3_FAILED, SERVED)
    refused(append(part(0, 4), part(4, 2), part(6, 2), part(1, 4)), L.EXL3_FAILED, "another layout")
    refused(append(part(0, 2), part(2, 2), part(6, 2), part(3, 2)), L.EXL3_FAILED, "over k or v")
    refused(append(part(0, 2), part(2, 2), part(6, 2), part(5, 2)), L.EXL3_FAILED, "over k or v")
    refused(append(part(0, 2), part(2, 2), part(4, 2), part(6, 2)), L.EXL3_FAILED, SERVED)
    refused(attention(part(0, 4), part(4, 4)), L.EXL3_FAILED, SERVED)
    refused(attention(part(0, 4), part(3, 4)), L.EXL3_FAILED, "out is not q")
    # one row: its stride means nothing
    one = heads(rows=1, row_stride=999)
    refused(append(one, heads(data=2 * AT, rows=1), heads(data=3 * AT, rows=1), heads(rows=1), rows=1), L.EXL3_FAILED, SERVED)
    # a query repeated for every row and head, and a result over it
    refused(attention(heads(row_stride=0, head_stride=0), heads(data=AT + 128)), L.EXL3_FAILED, SERVED)
    refused(attention(heads(row_stride=0, head_stride=0), heads(data=AT - 256)), L.EXL3_FAILED, "out is not q")
    # interleaved with a gate: [head][query | gate]
    refused(attention(heads(heads=4, row_stride=512, head_stride=128), heads(data=AT + 128, heads=4, row_stride=512, head_stride=128)),
            L.EXL3_FAILED, SERVED)


def test_in_place_is_one_layout_and_dtype():
    f32 = dict(dtype=L.F32)
    k, v = heads(data=2 * AT, **f32), heads(data=3 * AT, **f32)
    refused(append(heads(**f32), k, v, heads(**f32)), L.EXL3_FAILED, SERVED)
    refused(append(heads(**f32), k, v, heads()), L.EXL3_FAILED, "another layout")
    refused(append(heads(**f32), k, v, heads(data=AT + 2 * 1024)), L.EXL3_FAILED, SERVED)


def test_against_the_elements_themselves():
    r = random.Random(5)
    count = {True: 0, False: 0}
    for _ in range(4000):
        def some(data):
            return heads(data=data, rows=rows, heads=r.choice([2, 4]), row_stride=r.choice([0, 64, 65, 128, 192, 200, 256, 512, -256, 640]),
                         head_stride=r.choice([0, 64, 64, 70, 128, 192, 512, -64]))
        rows = r.choice([1, 2, 3, 5])
        q, out = some(AT), some(AT + 2 * r.randrange(-2000, 2000))
        out.heads = q.heads
        v = attention(q, out, rows=rows)
        if "overlap" in v.message():
            continue
        over = bool(addresses(q) & addresses(out))
        refused(v, L.EXL3_FAILED, "out is not q" if over else SERVED)
        count[over] += 1
    assert min(count.values()) > 300


@pytest.mark.parametrize("at,text", [("context", SERVED), ("kept", SERVED), ("path", "lies over"), ("table", "lies over"),
                                     ("row_start", "lies over"), (8, "lies over"), (4, "lies over"), (12, SERVED)])
def test_keep_lengths_over_what_it_reads(at, text):
    where = dict(context=AT, kept=2 * AT, path=3 * AT, table=4 * AT, row_start=5 * AT)
    b = batch(nseq=3, context=where["context"], table=where["table"], row_start=where["row_start"])
    lens = where[at] if isinstance(at, str) else AT + at
    refused(L.lib().exl3_cache_keep(cache(device=99), b, where["path"], 4, where["kept"], None, lens), L.EXL3_FAILED, text)


def test_page_states_over_one_another_and_over_the_arguments():
    lib = L.lib()
    old = dict(refs=AT, table=2 * AT, held=3 * AT, lens=4 * AT)
    new = dict(refs=5 * AT, table=6 * AT, held=7 * AT, lens=8 * AT)
    for name, at, text in (("refs", AT + 28, "own arrays"), ("refs", AT + 32, SERVED), ("table", 2 * AT - 28, "own arrays"),
                           ("held", 2 * AT + 28, "own arrays"), ("lens", 4 * AT + 4, "own arrays"), ("lens", 4 * AT + 8, SERVED),
                           ("held", 3 * AT - 4, "own arrays"), ("refs", 9 * AT + 4, "arguments"), ("refs", 9 * AT + 8, SERVED)):
        for call in (lambda a, b: lib.exl3_cache_fork(cache(device=99), a, 9 * AT, None, b),
                     lambda a, b: lib.exl3_cache_grow(cache(device=99), a, 9 * AT, None, b, 10 * AT)):
            refused(call(state(**old), state(**new | {name: at})), L.EXL3_FAILED, text)
    for missing, text in ((AT + 4, "own arrays"), (7 * AT, "arguments"), (9 * AT + 4, "arguments"), (10 * AT, SERVED)):
        refused(lib.exl3_cache_grow(cache(device=99), state(**old), 9 * AT, None, state(**new), missing), L.EXL3_FAILED, text)
