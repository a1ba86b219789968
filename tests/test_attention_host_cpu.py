"""The attention side's Python wrappers where no GPU is needed (plugins_b200/attention.py)."""
from plugins_b200 import attention as A


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
