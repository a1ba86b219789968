"""A layer's attention side over a paged key/value cache: what runs between its q|k|v linears and its o linear, and what
ends a step after the last layer.

    cache = A.KvCache.empty(layers=36, pages=4096, page_size=64, kv_heads=8, head_dim=128, dtype=torch.bfloat16)
    batch = A.TreeBatch(row_start, context, table, max_rows=..., tree=bits, position=pos)     # once per step
    for layer in ...:
        q = A.qk_norm_rope(cache, layer, batch, q, k, v, rope)      # norms, rotation, k and v into the cache
        o = A.tree_attention(cache, layer, batch, q)                # one token, a drafted tree, or a prompt chunk
    path, kept, token = A.draft_verify(cache, batch, logits, tokens, parent, uniform, temperature)
    lens = A.cache_keep(cache, batch, path, kept)                   # the accepted path stays

and the pages between steps: :func:`cache_fork` (fork, reorder, free), :func:`cache_grow` (new pages, copy on write),
:func:`cache_compact`, and :func:`cache_evict`, which keeps a row's tokens inside a budget by how much they were attended to
(:func:`attention_weight`, after each layer's attention).  Every call goes through the C ABI (include/exl3_b200.h says what each computes) on the current
torch stream or ``stream``; refusals raise :class:`Exl3Error`.
"""
from __future__ import annotations

import ctypes
import functools
import struct

import torch

from . import _lib as L
from ._lib import Exl3Error, check
from .quant import _TORCH_DT, _stream

__all__ = ["Exl3Error", "KvCache", "TreeBatch", "NormRope", "PageState", "qk_norm_rope", "tree_attention", "cache_fork",
           "cache_grow", "cache_keep", "cache_compact", "cache_evict", "draft_verify",
           "attention_weight"]


def _refuse(why: str, code: int = L.EXL3_FAILED):
    raise Exl3Error(code, "exl3_b200: " + why)


def _ints(t, shape, what: str, device=None, optional: bool = False):
    """A contiguous int32 GPU tensor of this shape (None in a place takes any size)."""
    if t is None and optional:
        return None
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.int32 or not t.is_contiguous():
        _refuse(f"{what} is a contiguous int32 tensor on the GPU")
    if t.dim() != len(shape) or any(want is not None and want != got for want, got in zip(shape, t.shape)):
        _refuse(f"{what} has shape {list(t.shape)}, not {['any' if s is None else s for s in shape]}")
    if device is not None and t.device != device:
        _refuse(f"{what} lies on another device")
    return t


# exl3_heads as bytes: a ctypes structure costs more than the rest of the checks
_HEADS = struct.Struct("@Piiiiqq")
assert _HEADS.size == ctypes.sizeof(L.Heads)


def _heads(t: torch.Tensor, index: int, what: str) -> bytes:
    dt = _TORCH_DT.get(t.dtype)
    if t.get_device() != index:
        _refuse(f"{what} does not lie on the cache's GPU")
    if dt is None:
        _refuse(f"dtype {t.dtype} is not served", L.EXL3_UNSUPPORTED)
    shape, stride = t.shape, t.stride()
    if len(shape) != 3:
        _refuse(f"{what} is [rows, heads, head_dim]")
    if stride[2] != 1 and shape[2] > 1:
        _refuse(f"{what}'s head vectors must be contiguous")
    return _HEADS.pack(t.data_ptr(), dt, shape[0], shape[1], shape[2], stride[0], stride[1])


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _on(stream, index: int) -> int:
    """The stream's handle; without one, the current stream of the cache's GPU."""
    if stream is not None:
        return _stream(stream)
    return _raw_stream(index) if _raw_stream is not None else torch.cuda.current_stream(index).cuda_stream


def _check(v: L.Verdict) -> None:
    if v.code:
        check(v)


class _Calls:
    """The library's per-layer calls taking addresses and packed structures."""
    rope = attention = None

    @classmethod
    def load(cls) -> None:
        p, c = ctypes.c_void_p, ctypes.c_char_p
        lib = L.lib()
        proto = ctypes.CFUNCTYPE(L.Verdict, p, ctypes.c_int32, p, c, ctypes.c_float, p, c, p)
        cls.attention = proto(ctypes.cast(lib.exl3_tree_attention, p).value)
        proto = ctypes.CFUNCTYPE(L.Verdict, p, ctypes.c_int32, p, c, c, c, p, p, c)
        cls.rope = proto(ctypes.cast(lib.exl3_qk_norm_rope, p).value)  # last: another thread takes it for all there


class _StepCalls:
    """Likewise the calls that end a step (exl3_kv_weight and exl3_draft as bytes)."""
    weight = evict = verify = None

    @classmethod
    def load(cls) -> None:
        p, c, i, f = ctypes.c_void_p, ctypes.c_char_p, ctypes.c_int32, ctypes.c_float
        lib = L.lib()
        proto = ctypes.CFUNCTYPE(L.Verdict, p, i, p, c, f, p, f, p, c)
        cls.weight = proto(ctypes.cast(lib.exl3_attention_weight, p).value)
        proto = ctypes.CFUNCTYPE(L.Verdict, p, p, c, p, i, i, p, p, c, p)
        cls.evict = proto(ctypes.cast(lib.exl3_cache_evict, p).value)
        proto = ctypes.CFUNCTYPE(L.Verdict, p, p, c, p, p, i, p, p)
        cls.verify = proto(ctypes.cast(lib.exl3_draft_verify, p).value)  # last, as above


_KV_WEIGHT = struct.Struct("@IiiiPqqq")
_DRAFT = struct.Struct("@IiiiqqPPPPPP")
assert _KV_WEIGHT.size == ctypes.sizeof(L.KvWeight) and _DRAFT.size == ctypes.sizeof(L.Draft)


def _used_on(stream, *tensors) -> None:
    """Tensors the caching allocator must not hand out again before `stream` is done with them: all that a call reads or
    writes there.  (A stream given by its handle is the caller's to wait for.)"""
    if stream is not None and isinstance(stream, torch.cuda.Stream):
        for t in tensors:
            if t is not None:
                t.record_stream(stream)


def _made_on(stream, make, *args, **kw) -> torch.Tensor:
    current = torch.cuda.current_stream(stream.device)
    with torch.cuda.stream(stream):
        t = make(*args, **kw)
    t.record_stream(current)
    return t


def _maker(stream, make):
    """`make` for a result that `stream` writes: from that stream's own memory (what the current stream has let go of it may
    still be using), and kept for the current stream's later use of it."""
    return functools.partial(_made_on, stream, make) if isinstance(stream, torch.cuda.Stream) else make


def _overlap(a, b) -> bool:
    """Whether two contiguous tensors of one device share memory (None has none)."""
    return b is not None and a.data_ptr() < b.data_ptr() + b.nbytes and b.data_ptr() < a.data_ptr() + a.nbytes


class KvCache:
    """The paged cache of every layer: ``k`` and ``v`` [layers, pages, kv_heads, page_size, head_dim], f16 or bf16, of
    any strides (the same for both) with contiguous head vectors -- so also the transposed view of a pool stored
    [layers, pages, page_size, kv_heads, head_dim]."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        for t in (k, v):
            if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dim() != 5:
                _refuse("the cache is two GPU tensors [layers, pages, kv_heads, page_size, head_dim]")
        if k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype or k.device != v.device:
            _refuse("k and v have one shape, one dtype, the same strides and one device")
        if k.stride(4) != 1:
            _refuse("the cache's head vectors must be contiguous")
        dt = _TORCH_DT.get(k.dtype)
        if dt not in (L.F16, L.BF16):
            _refuse("the cache holds f16 or bf16", L.EXL3_UNSUPPORTED)
        self.k, self.v, self.device = k, v, k.device
        layers, pages, kv_heads, page_size, dim = k.shape
        sl, sp, sh, st, _ = k.stride()
        self.raw = L.KvCache(ctypes.sizeof(L.KvCache), k.device.index, dt, layers, pages, page_size, kv_heads, dim,
                             k.data_ptr(), v.data_ptr(), sl, sp, sh, st)
        self._at, self._index = ctypes.addressof(self.raw), k.device.index
        self._scale = dim ** -0.5
        check(L.lib().exl3_kv_register(self.raw))
        if _Calls.rope is None:
            _Calls.load()
        if _StepCalls.verify is None:
            _StepCalls.load()

    @classmethod
    def empty(cls, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=torch.bfloat16,
              device=None) -> "KvCache":
        """A new pool, its slots uninitialised (nothing reads a slot that no row sees)."""
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        shape = (layers, pages, kv_heads, page_size, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))

    @property
    def page_size(self) -> int:
        return self.raw.page_size

    @property
    def pages(self) -> int:
        return self.raw.pages


class TreeBatch:
    """One step's new tokens: sequence s owns rows ``row_start[s]`` .. ``row_start[s + 1]`` - 1 (int32 [nseq + 1]),
    which follow its ``context[s]`` cached tokens (int32 [nseq]) in the pages ``table[s]`` (int32 [nseq, max_pages]).

    ``tree`` (int32 [rows, words]): bit j of a row says whether it sees row j of its own sequence; without it row i sees
    rows 0 .. i.  ``position`` (int32 [rows]): what the rotation turns by, without it context + i.  ``rows``: all rows
    (rows past row_start[nseq] are padding); ``max_rows``: the most rows of one sequence; ``max_context``: a bound on
    context + rows (what the table spans, if not given).  The tensors are read when the calls' work runs, so a step in a
    CUDA graph may change their values between replays."""

    def __init__(self, row_start, context, table, max_rows: int, rows: int | None = None, max_context: int = 0,
                 tree=None, position=None):
        _ints(row_start, (None,), "row_start")
        dev = row_start.device
        nseq = row_start.shape[0] - 1
        if nseq < 0:
            _refuse("row_start has nseq + 1 entries")
        _ints(context, (nseq,), "context", dev)
        _ints(table, (nseq, None), "table", dev)
        if rows is None:
            rows = next((t.shape[0] for t in (tree, position) if t is not None), None)
        _ints(tree, (rows, None), "tree", dev, optional=True)
        if tree is not None and tree.shape[1] == 0:
            _refuse("a tree without words")  # (whose address is null: it would read as no tree)
        _ints(position, (rows,), "position", dev, optional=True)
        self.rows, self.nseq, self.device = rows, nseq, dev
        self._keep = (row_start, context, table, tree, position)
        ptr = (lambda t: t.data_ptr() if t is not None else None)
        self.raw = L.TreeBatch(ctypes.sizeof(L.TreeBatch), nseq, rows or 0, int(max_rows), int(max_context),
                               table.shape[1], tree.shape[1] if tree is not None else 0, ptr(row_start), ptr(context),
                               ptr(table), ptr(tree), ptr(position))
        self._at, self._index = ctypes.addressof(self.raw), dev.index

    def _for(self, cache: KvCache, rows: int):
        if self.rows is None:  # neither tree nor position nor rows said how many
            self.rows = self.raw.rows = rows
        if rows != self.rows:
            _refuse(f"the batch has {self.rows} rows, not {rows}")
        if self._index != cache._index:
            _refuse("the batch lies on another device than the cache")
        return self._at


class NormRope:
    """The norms and rotation of :func:`qk_norm_rope`: ``inv_freq`` (float64 [rot_dims / 2], radians per position) or
    None for no rotation, the heads' norm weights ([head_dim], one dtype) or None for no norm, ``adjacent`` pairs
    (2i, 2i + 1) instead of (i, i + rot_dims / 2), ``weight_offset`` added to the weights (1 for weights stored around
    zero)."""

    def __init__(self, inv_freq=None, q_weight=None, k_weight=None, eps: float = 1e-6, adjacent: bool = False,
                 weight_offset: float = 0.0):
        if inv_freq is not None and (not inv_freq.is_cuda or inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or
                                     not inv_freq.is_contiguous()):
            _refuse("inv_freq is a contiguous float64 vector on the GPU")
        weights = [w for w in (q_weight, k_weight) if w is not None]
        for w in weights:
            if not w.is_cuda or w.dim() != 1 or not w.is_contiguous() or w.dtype != weights[0].dtype:
                _refuse("norm weights are contiguous vectors on the GPU in one dtype")
        wdt = _TORCH_DT.get(weights[0].dtype) if weights else L.F32
        if wdt is None:
            _refuse("norm weights are f16, bf16 or f32", L.EXL3_UNSUPPORTED)
        self.dim = weights[0].shape[0] if weights else None
        if any(w.shape[0] != self.dim for w in weights):
            _refuse("norm weights are [head_dim]")
        self._keep = (inv_freq, q_weight, k_weight)
        self.device = next((t.device for t in self._keep if t is not None), None)
        if any(t is not None and t.device != self.device for t in self._keep):
            _refuse("the norm weights and frequencies lie on one device")
        ptr = (lambda t: t.data_ptr() if t is not None else None)
        self.raw = L.NormRope(ctypes.sizeof(L.NormRope), 0 if inv_freq is None else 2 * inv_freq.shape[0],
                              int(bool(adjacent)), wdt, float(eps), float(weight_offset), ptr(q_weight), ptr(k_weight),
                              ptr(inv_freq))
        self._at = ctypes.addressof(self.raw)


def qk_norm_rope(cache: KvCache, layer: int, batch: TreeBatch, q, k, v, rope: NormRope, out=None, stream=None):
    """q [rows, heads, head_dim] normed and rotated (returned, in ``out`` if given: in q's dtype or the cache's, q
    itself allowed), k and v [rows, kv_heads, head_dim] written to their slots of ``layer``: k normed and rotated, v as it is."""
    if out is None:
        out = _maker(stream, torch.empty_like)(q)
    if rope.dim is not None and rope.dim != cache.raw.head_dim:
        _refuse("norm weights are [head_dim]")
    if rope.device is not None and rope.device != cache.device:
        _refuse("the norm weights lie on another device than the cache")
    i = cache._index
    hq, hk, hv, ho = _heads(q, i, "q"), _heads(k, i, "k"), _heads(v, i, "v"), _heads(out, i, "out")
    if stream is not None:
        _used_on(stream, q, k, v, out, cache.k, cache.v, *batch._keep, *rope._keep)
    _check(_Calls.rope(cache._at, layer, batch._for(cache, q.shape[0]), hq, hk, hv, rope._at, _on(stream, i), ho))
    return out


def tree_attention(cache: KvCache, layer: int, batch: TreeBatch, q, scale: float | None = None, lse=None, out=None,
                   stream=None):
    """Attention of the batch's rows q [rows, heads, head_dim] over ``layer`` -> [rows, heads, head_dim] in the cache's
    dtype.  ``scale`` defaults to head_dim ** -0.5.  ``lse``: True returns (out, lse), the log-sum-exp f32
    [rows, heads] of each row's scores; a tensor receives it."""
    i = cache._index
    if out is None:
        out = _maker(stream, torch.empty_like)(q)
    hq, ho = _heads(q, i, "q"), _heads(out, i, "out")
    if lse is True:
        lse = _maker(stream, torch.empty)(q.shape[:2], dtype=torch.float32, device=q.device)
    elif lse is False:
        lse = None
    elif lse is not None and (lse.dtype != torch.float32 or lse.device != cache.device or not lse.is_contiguous() or
                              lse.shape != q.shape[:2]):
        _refuse("lse is a contiguous f32 tensor [rows, heads] on the cache's GPU")
    if stream is not None:
        _used_on(stream, q, out, lse, cache.k, cache.v, *batch._keep)
    _check(_Calls.attention(cache._at, layer, batch._for(cache, q.shape[0]), hq, cache._scale if scale is None else scale,
                            _on(stream, i), ho, None if lse is None else lse.data_ptr()))
    return out if lse is None else (out, lse)


def _kv_weight(t, layers: int, nseq: int, cache: KvCache, dims: int = 4) -> tuple:
    """The fields of exl3_kv_weight: f32 [layers,] rows, kv_heads, slots on the cache's GPU, a head's slots contiguous."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.get_device() != cache._index:
        _refuse("weights are an f32 tensor on the cache's GPU")
    shape, stride = t.shape, t.stride()
    if len(shape) != dims:
        _refuse("weights are [layers, rows, kv_heads, slots]" if dims == 4 else "a layer's weights are [rows, kv_heads, slots]")
    if dims == 3:
        shape, stride = (1, *shape), (0, *stride)
    if shape[0] != layers or shape[1] != nseq or shape[2] != cache.raw.kv_heads:
        _refuse(f"the weights have shape {list(shape)}, not {[layers, nseq, cache.raw.kv_heads, 'any']}")
    if stride[3] != 1 and shape[3] > 1:
        _refuse("the weights of a head's slots must be contiguous")
    return _KV_WEIGHT.size, layers, nseq, shape[3], t.data_ptr(), stride[0], stride[1], stride[2]


def attention_weight(cache: KvCache, layer: int, batch: TreeBatch, q, lse, weight, scale: float | None = None,
                     decay: float = 1.0, stream=None):
    """How much the batch's rows attended to each cached token of ``layer``, added to ``weight`` (f32
    [nseq, kv_heads, slots], in place, returned): slots of the context keep ``decay`` of what they had, the rows' own slots
    begin anew.  ``q``, ``scale`` and ``lse`` (f32 [rows, heads]) are :func:`tree_attention`'s, which comes first."""
    i = cache._index
    hq = _heads(q, i, "q")
    _floats(lse, q.shape[:2], "lse", i)
    raw = _KV_WEIGHT.pack(*_kv_weight(weight, 1, batch.nseq, cache, 3))
    if stream is not None:
        _used_on(stream, q, lse, weight, cache.k, cache.v, *batch._keep)
    _check(_StepCalls.weight(cache._at, layer, batch._for(cache, q.shape[0]), hq, cache._scale if scale is None else scale,
                             lse.data_ptr(), decay, _on(stream, i), raw))
    return weight


class PageState:
    """The page bookkeeping: ``refs`` (int32 [pages], rows that hold each page; 0 free), ``table`` (int32
    [nseq, max_pages], -1 past the held ones), ``held`` and ``lens`` (int32 [nseq], pages and tokens of each row)."""

    def __init__(self, refs, table, held, lens):
        _ints(refs, (None,), "refs")
        dev, nseq = refs.device, held.shape[0]
        _ints(table, (nseq, None), "table", dev)
        _ints(held, (nseq,), "held", dev)
        _ints(lens, (nseq,), "lens", dev)
        self.refs, self.table, self.held, self.lens = refs, table, held, lens
        self.raw = L.PageState(ctypes.sizeof(L.PageState), nseq, table.shape[1], refs.data_ptr(), table.data_ptr(),
                               held.data_ptr(), lens.data_ptr())

    @classmethod
    def empty(cls, cache: KvCache, nseq: int, max_pages: int) -> "PageState":
        """All pages free, ``nseq`` empty rows."""
        z = (lambda *s: torch.zeros(s, dtype=torch.int32, device=cache.device))
        return cls(z(cache.pages), z(nseq, max_pages) - 1, z(nseq), z(nseq))

    def _tensors(self):
        return self.refs, self.table, self.held, self.lens

    def _like(self, n: int, stream) -> "PageState":
        pages, width = self.refs.shape[0], self.raw.max_pages
        flat = _maker(stream, torch.empty)(pages + n * (width + 2), dtype=torch.int32, device=self.refs.device)
        refs, table, held, lens = flat.split_with_sizes((pages, n * width, n, n))
        new = PageState.__new__(PageState)  # (nothing to check)
        new.refs, new.table, new.held, new.lens = refs, table.view(n, width), held, lens
        at = flat.data_ptr()
        new.raw = L.PageState(ctypes.sizeof(L.PageState), n, width, at, at + 4 * pages, at + 4 * (pages + n * width),
                              at + 4 * (pages + n * width + n))
        return new


def _states(cache: KvCache, state: PageState, out: PageState | None, stream, nseq: int | None = None):
    if state.refs.shape[0] != cache.pages or (out is not None and out.refs.shape[0] != cache.pages):
        _refuse("refs counts the cache's pages")
    if state.refs.device != cache.device or (out is not None and out.refs.device != cache.device):
        _refuse("the page state lies on another device than the cache")
    n = state.raw.nseq if nseq is None else nseq
    if out is None:
        out = state._like(n, stream)
    elif out.raw.nseq != n:
        _refuse(f"the new page state has {out.raw.nseq} rows, not {n}")
    return out


def cache_fork(cache: KvCache, state: PageState, parent, out: PageState | None = None, stream=None) -> PageState:
    """Fork, reorder and free: row i of the result is row ``parent[i]`` (int32; -1: an empty row) sharing its pages; the
    pages of rows nobody names become free."""
    _ints(parent, (None,), "parent", cache.device)
    out = _states(cache, state, out, stream, parent.shape[0])
    if stream is not None:
        _used_on(stream, parent, *state._tensors(), *out._tensors())
    check(L.lib().exl3_cache_fork(cache.raw, state.raw, parent.data_ptr(), _on(stream, cache._index), out.raw))
    return out


def cache_grow(cache: KvCache, state: PageState, need, out: PageState | None = None, missing=None, stream=None):
    """Pages for ``need[i]`` (int32) tokens in every row, each shared page that row i will write (slots ``lens[i]`` to
    ``need[i]`` - 1) replaced by one of its own, with a copy where it holds tokens of the row -> (the new state,
    ``missing``: an int32 scalar tensor, 0, or the pages lacking: then nothing changed)."""
    _ints(need, (state.raw.nseq,), "need", cache.device)
    out = _states(cache, state, out, stream)
    if missing is None:
        missing = _maker(stream, torch.empty)((), dtype=torch.int32, device=cache.device)
    else:
        _ints(missing, (), "missing", cache.device)
    if stream is not None:
        _used_on(stream, need, missing, cache.k, cache.v, *state._tensors(), *out._tensors())
    check(L.lib().exl3_cache_grow(cache.raw, state.raw, need.data_ptr(), _on(stream, cache._index), out.raw,
                                  missing.data_ptr()))
    return out, missing


def cache_keep(cache: KvCache, batch: TreeBatch, path, kept, out=None, stream=None, weight=None):
    """The accepted rows of each drafted tree, ``path[s][:kept[s]]`` (int32 [nseq, depth], ascending; None: the first
    kept rows), moved behind the context in every layer -> the sequences' new lengths, context + kept (``out`` may be the
    batch's own context tensor).  ``weight`` ([layers, nseq, kv_heads, slots]): the rows' weights move likewise, first."""
    _ints(kept, (batch.nseq,), "kept", cache.device)
    _ints(path, (batch.nseq, None), "path", cache.device, optional=True)
    if out is None:
        out = _maker(stream, torch.empty)(batch.nseq, dtype=torch.int32, device=cache.device)
    else:
        _ints(out, (batch.nseq,), "lens", cache.device)
    if batch.rows is None:
        _refuse("the batch does not know its rows yet: give rows to TreeBatch")
    if stream is not None:
        _used_on(stream, path, kept, out, cache.k, cache.v, *batch._keep)
    batch._for(cache, batch.rows)
    if weight is not None:
        raw = L.KvWeight(*_kv_weight(weight, cache.raw.layers, batch.nseq, cache))
        # what exl3_cache_keep refuses, before the weights move (a second call would move them again)
        row_start, context, table = batch._keep[:3]
        if any(_overlap(out, t) for t in (row_start, table, path)) or \
                any(_overlap(out, t) and out.data_ptr() != t.data_ptr() for t in (context, kept)):
            _refuse("exl3_b200: lens lies over the call's arguments")
        if stream is not None:
            _used_on(stream, weight)
        check(L.lib().exl3_weight_keep(cache.raw, batch.raw, None if path is None else path.data_ptr(),
                                       0 if path is None else path.shape[1], kept.data_ptr(), _on(stream, cache._index), raw))
    check(L.lib().exl3_cache_keep(cache.raw, batch.raw, None if path is None else path.data_ptr(),
                                  0 if path is None else path.shape[1], kept.data_ptr(), _on(stream, cache._index),
                                  out.data_ptr()))
    return out


def cache_compact(cache: KvCache, state: PageState, out: PageState | None = None, stream=None) -> PageState:
    """The live pages moved into the lowest ids, in every layer; tables and reference counts follow."""
    out = _states(cache, state, out, stream)
    if stream is not None:
        _used_on(stream, cache.k, cache.v, *state._tensors(), *out._tensors())
    check(L.lib().exl3_cache_compact(cache.raw, state.raw, _on(stream, cache._index), out.raw))
    return out


def cache_evict(cache: KvCache, state: PageState, weight, budget, sink: int = 0, recent: int = 0,
                out: PageState | None = None, weight_out=None, missing=None, stream=None):
    """Rows of more than max(``budget[i]`` (int32), ``sink`` + ``recent``) tokens keep that many: in every layer and kv head the
    first ``sink``, the last ``recent`` and the heaviest of the others by ``weight`` (f32 [layers, rows, kv_heads, slots]),
    moved together in their order -> (the new state, ``missing``: an int32 scalar tensor, 0, or the free pages lacking to part
    from shared ones: then nothing changed).  The tokens' weights move with them, in place or to ``weight_out``."""
    n = state.raw.nseq
    if not (0 <= sink < 1 << 31 and 0 <= recent < 1 << 31):
        _refuse("counts of tokens that always stay are not negative")
    _ints(budget, (n,), "budget", cache.device)
    raw = _KV_WEIGHT.pack(*_kv_weight(weight, cache.raw.layers, n, cache))
    kept = raw if weight_out is None else _KV_WEIGHT.pack(*_kv_weight(weight_out, cache.raw.layers, n, cache))
    out = _states(cache, state, out, stream)
    if missing is None:
        missing = _maker(stream, torch.empty)((), dtype=torch.int32, device=cache.device)
    else:
        _ints(missing, (), "missing", cache.device)
    if stream is not None:
        _used_on(stream, budget, missing, weight, weight_out, cache.k, cache.v, *state._tensors(), *out._tensors())
    _check(_StepCalls.evict(cache._at, ctypes.addressof(state.raw), raw, budget.data_ptr(), sink, recent,
                            _on(stream, cache._index), ctypes.addressof(out.raw), kept, missing.data_ptr()))
    return out, missing


def _floats(t, shape, what: str, index: int):
    """A contiguous f32 tensor of this shape on the cache's GPU."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.get_device() != index or not t.is_contiguous():
        _refuse(f"{what} is a contiguous f32 tensor on the cache's GPU")
    if t.shape != shape:
        _refuse(f"{what} has shape {list(t.shape)}, not {list(shape)}")


def _vocab_rows(t, rows: int, vocab, what: str, index: int):
    """[rows, vocab] with contiguous rows -> its dtype."""
    if not isinstance(t, torch.Tensor) or t.get_device() != index or t.dim() != 2 or t.shape[0] != rows or \
            (vocab is not None and t.shape[1] != vocab) or (t.stride(1) != 1 and t.shape[1] > 1):
        _refuse(f"{what} is [rows, vocab] on the cache's GPU, its rows contiguous")
    dt = _TORCH_DT.get(t.dtype)
    if dt not in (L.F16, L.BF16, L.F32):
        _refuse(f"{what} is f16, bf16 or f32", L.EXL3_UNSUPPORTED)
    return dt


def draft_verify(cache: KvCache, batch: TreeBatch, logits, tokens, parent, uniform, temperature=None, draft=None,
                 depth: int | None = None, path=None, kept=None, token=None, stream=None):
    """Which drafted tokens stay, and the token after them -> (``path`` [nseq, depth], ``kept`` [nseq], as
    :func:`cache_keep` takes them, ``token`` [nseq]; int32).

    Row 0 of a sequence is its newest token, the others are drafts: ``tokens`` (int32 [rows]) and ``parent`` (int32 [rows],
    rows of the same sequence, a parent before its children; None: chains).  ``logits`` [rows, vocab]: the target's, f16, bf16
    or f32; ``draft`` [rows, vocab]: the probabilities that the children of each row were drawn from (None: a drafter without
    any).  ``uniform`` (f32 [rows, 2], in [0, 1)): a number for the row's own token and one for the token that follows the
    row.  ``temperature`` (f32 [nseq], 0: greedy; None: 1).  The path and the token are distributed as tokens drawn one by one
    from softmax(logits / temperature).  ``depth``: the most rows of a path (if not given max_rows, or all rows without such a
    bound)."""
    dev, n, i = cache.device, batch.nseq, cache._index
    rows = batch.rows if batch.rows is not None else logits.shape[0]
    dt = _vocab_rows(logits, rows, None, "logits", i)
    vocab = logits.shape[1]
    qt = L.F32 if draft is None else _vocab_rows(draft, rows, vocab, "draft", i)
    for t, what in ((tokens, "tokens"), (parent, "parent")):
        # (the common case at a glance; the other says what is wrong, or that there are no parents)
        if t is None or t.dtype != torch.int32 or t.shape != (rows,) or t.get_device() != i or not t.is_contiguous():
            _ints(t, (rows,), what, dev, optional=what == "parent")
    _floats(uniform, (rows, 2), "uniform", i)
    if temperature is not None:
        _floats(temperature, (n,), "temperature", i)
    depth = max(1, batch.raw.max_rows or rows) if depth is None else int(depth)  # (max_rows 0: no bound is given)
    if depth < 1:
        _refuse("a path without depth")
    make = _maker(stream, torch.empty)
    if path is None and kept is None and token is None:  # one allocation
        path, kept, token = make(n * (depth + 2), dtype=torch.int32, device=dev).split_with_sizes((n * depth, n, n))
        path = path.view(n, depth)
    else:
        path = make((n, depth), dtype=torch.int32, device=dev) if path is None else _ints(path, (n, depth), "path", dev)
        kept = make(n, dtype=torch.int32, device=dev) if kept is None else _ints(kept, (n,), "kept", dev)
        token = make(n, dtype=torch.int32, device=dev) if token is None else _ints(token, (n,), "token", dev)
    if stream is not None:
        _used_on(stream, logits, tokens, parent, uniform, temperature, draft, path, kept, token, *batch._keep)
    raw = _DRAFT.pack(_DRAFT.size, vocab, dt, qt, logits.stride(0), 0 if draft is None else draft.stride(0), logits.data_ptr(),
                      0 if draft is None else draft.data_ptr(), tokens.data_ptr(), 0 if parent is None else parent.data_ptr(),
                      uniform.data_ptr(), 0 if temperature is None else temperature.data_ptr())
    _check(_StepCalls.verify(cache._at, batch._for(cache, rows), raw, _on(stream, i), path.data_ptr(), depth, kept.data_ptr(),
                             token.data_ptr()))
    return path, kept, token
