"""The attention side's Python wrappers where no GPU is needed (plugins_b200/attention.py)."""
from plugins_b200 import _lib as L
from plugins_b200 import attention as A
from test_attention_cpu import AT, cache, refused, state


def test_a_second_thread_never_sees_half_the_calls(monkeypatch):
    """KvCache loads the calls when `rope` is missing: `rope` has to come last."""
    lib = A.L.lib()
    seen = []

    class Watched:
        def __getattr__(self, name):
            seen.append((name, A._Calls.rope))
            return getattr(lib, name)

    monkeypatch.setattr(A._Calls, "rope", None)
    monkeypatch.setattr(A._Calls, "attention", None)
    monkeypatch.setattr(A.L, "lib", Watched)
    A._Calls.load()
    assert {n for n, _ in seen} == {"exl3_qk_norm_rope", "exl3_tree_attention"}
    assert all(rope is None for _, rope in seen) and A._Calls.rope is not None and A._Calls.attention is not None


def test_a_fork_whose_search_would_not_end_is_refused():
    """Every old row looks through all new ones: the pairs are bounded."""
    far = dict(refs=5 * AT, table=64 * AT, held=128 * AT, lens=192 * AT, max_pages=1)
    old = dict(table=256 * AT, held=320 * AT, lens=384 * AT, max_pages=1)
    fork = L.lib().exl3_cache_fork
    refused(fork(cache(device=99), state(**old, nseq=65537), 448 * AT, None, state(**far, nseq=65536)), L.EXL3_TOO_LARGE, "2^32 pairs")
    refused(fork(cache(device=99), state(**old, nseq=65536), 448 * AT, None, state(**far, nseq=65536)), L.EXL3_FAILED, "exl3_kv_register")
