"""exl3_draft_verify of a batch without rows, without a GPU: it still reads row_start and temperature, and writes its results."""
import pytest

from plugins_b200 import _lib as L
from test_attention_cpu import AT, batch, refused
from test_draft_verify_cpu import draft, verify


@pytest.mark.parametrize("which", ["path", "kept", "token"])
def test_results_over_what_is_read_are_refused(which):
    b = batch(nseq=3, rows=0, max_rows=0)
    refused(verify(b=b), L.EXL3_FAILED, "exl3_kv_register")  # what is served fails for want of a workspace alone
    for at in (b.row_start, b.row_start + 12, draft().temperature + 8):
        refused(verify(b=b, **{which: at}), L.EXL3_FAILED, "lie over its arguments")
    # what is not read without rows may lie anywhere
    refused(verify(b=b, **{which: draft().tokens}), L.EXL3_FAILED, "exl3_kv_register")
