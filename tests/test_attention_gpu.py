"""The attention side of a layer on the GPU (plugins_b200/attention.py) against its formulas in 64 bits."""
import math
import random

import pytest
import torch

import attention_ref as R
from plugins_b200 import _lib as L

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # half an ulp, relative
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133, torch.float32: 2.0 ** -150}


@pytest.fixture()
def A():
    from plugins_b200 import attention
    from plugins_b200 import quant as Q
    Q.device_error(0, clear=True)
    yield attention
    assert Q.device_error(0, clear=True) == 0


def cuda(t):
    return None if t is None else t.cuda()


class Step:
    """A cache with `lens` tokens, and `rows` new tokens per sequence."""

    def __init__(self, rows, lens, kv_heads, dim, page, dtype, tree=None, seed=0, layers=2, layout="hpd", stale=None,
                 spare=3):
        g = torch.Generator().manual_seed(seed)
        self.rows, self.lens, self.page, self.dtype = rows, lens, page, DT[dtype]
        held = [-(-(r + n) // page) for r, n in zip(rows, lens)]
        self.pages, width = sum(held) + spare, max(held + [1]) + 1
        ids = list(range(self.pages))
        random.Random(seed).shuffle(ids)
        self.table = torch.full((len(rows), width), -1, dtype=torch.int32)
        at = 0
        for s, h in enumerate(held):
            self.table[s, :h] = torch.tensor(ids[at:at + h], dtype=torch.int32)
            at += h
        self.row_start = [0]
        for r in rows:
            self.row_start.append(self.row_start[-1] + r)
        shape = (layers, self.pages, kv_heads, page, dim)
        self.k = torch.randn(shape, generator=g).to(self.dtype)
        self.v = torch.randn(shape, generator=g).to(self.dtype)
        if stale is not None:  # every slot no sequence owns
            used = torch.zeros((self.pages, page), dtype=torch.bool)
            for s in range(len(rows)):
                used[R.slots(self.table[s], page, 0, lens[s] + rows[s])] = True
            for t in (self.k, self.v):
                t.permute(1, 3, 0, 2, 4)[~used] = stale
        self.layout = layout
        self.layer = layers - 1
        self.tree = self.position = None
        if tree is not None:
            words = max(1, -(-max(rows) // 32))
            self.tree = torch.zeros((self.row_start[-1], words), dtype=torch.int32)
            pos = []
            for s, n in enumerate(rows):
                bits, depth = tree(s, n)
                for i, b in enumerate(bits):
                    for w in range(words):
                        x = (b >> (32 * w)) & 0xFFFFFFFF
                        self.tree[self.row_start[s] + i, w] = x - (1 << 32) if x >> 31 else x
                pos += [lens[s] + d for d in depth]
            self.position = torch.tensor(pos, dtype=torch.int32)

    def device(self, A, max_context=0, rows=None):
        if self.layout == "hpd":
            k, v = self.k.cuda(), self.v.cuda()
        else:  # pages of [token][head] rows
            k, v = (t.transpose(2, 3).contiguous().cuda().transpose(2, 3) for t in (self.k, self.v))
        cache = A.KvCache(k, v)
        batch = A.TreeBatch(torch.tensor(self.row_start, dtype=torch.int32).cuda(),
                            torch.tensor(self.lens, dtype=torch.int32).cuda(), self.table.cuda(),
                            max_rows=max(self.rows), max_context=max_context, tree=cuda(self.tree),
                            position=cuda(self.position), rows=rows)
        return cache, batch

    def want(self, q, scale):
        return R.attention(self.k[self.layer], self.v[self.layer], q.cpu(), self.row_start, self.lens, self.table, scale,
                           self.tree)


def chain(s, n):
    return [(2 << i) - 1 for i in range(n)], list(range(n))


def random_tree(s, n):
    r = random.Random(97 * s + n)
    bits, depth = [], []
    for i in range(n):
        p = r.randrange(max(0, i - 5), i) if i and r.random() < 0.9 else None
        bits.append((bits[p] if p is not None else 0) | (1 << i))
        depth.append(depth[p] + 1 if p is not None else 0)
    return bits, depth


def check_attention(out, lse, want, wlse, mass, dtype):
    """The result's rounding (u |o|), the probabilities' rounding to 16 bits for the product with v (u sum p |v|), and
    the f32 sums and exponentials: a score's error of up to D additions at 2^-23 of sum |q k| scale (below 2^-14 at these
    sizes) is a relative error of its probability."""
    u = U[dtype]
    tol = u * want.abs() + (u + 2.0 ** -13) * mass + TINY[dtype]
    err = (out.cpu().double() - want).abs()
    assert bool((err <= tol).all()), f"worst {float((err / tol.clamp(min=1e-30)).max()):.2f} x the tolerance"
    got = lse.cpu().double()
    inf = torch.isinf(wlse)
    assert torch.equal(torch.isinf(got), inf) and bool((got[inf] < 0).all())
    assert bool(((got - wlse)[~inf].abs() <= 2.0 ** -13 + 2.0 ** -21 * wlse[~inf].abs()).all())


CASES = [
    # rows, lens, heads, kv_heads, dim, page
    ([1], [0], 4, 4, 128, 16),
    ([1], [1], 8, 2, 128, 16),
    ([1], [300], 32, 8, 128, 16),
    ([1, 1, 1], [15, 16, 17], 8, 8, 64, 16),
    ([1, 1], [127, 1025], 16, 8, 256, 128),
    ([3, 0, 7, 1], [0, 50, 64, 129], 12, 4, 128, 32),
    ([16, 5], [63, 700], 32, 8, 128, 64),
    ([33], [200], 10, 2, 128, 64),
    ([64, 40], [130, 513], 8, 2, 64, 64),
    ([20], [70], 16, 8, 256, 256),
    ([100], [37], 5, 1, 128, 64),
    ([70, 65], [0, 260], 8, 8, 128, 128),
    ([17, 1, 31, 0, 64], [129, 700, 0, 3, 255], 8, 2, 128, 16),
    ([130, 40], [120, 9], 4, 1, 256, 16),
    ([300], [200], 2, 1, 64, 32),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kind", ["causal", "tree"])
@pytest.mark.parametrize("rows,lens,heads,kv_heads,dim,page", CASES)
def test_attention(A, rows, lens, heads, kv_heads, dim, page, kind, dtype):
    st = Step(rows, lens, kv_heads, dim, page, dtype, tree=random_tree if kind == "tree" else None, seed=len(rows) + dim,
              stale=math.nan)
    cache, batch = st.device(A)
    q = torch.randn((st.row_start[-1], heads, dim), generator=torch.Generator().manual_seed(1)).to(st.dtype)
    out, lse = A.tree_attention(cache, st.layer, batch, q.cuda(), lse=True)
    check_attention(out, lse, *st.want(q, dim ** -0.5), st.dtype)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [2, 12, 40, 70])
def test_attention_long_keys_split_over_the_gpu(A, dim, rows):
    st = Step([rows], [6001], 2, dim, 64, "bf16", tree=chain, seed=5, layers=1)
    cache, batch = st.device(A, max_context=6001 + rows)
    q = torch.randn((rows, 8, dim), generator=torch.Generator().manual_seed(2)).to(st.dtype) * 2
    out, lse = A.tree_attention(cache, 0, batch, q.cuda(), lse=True)
    check_attention(out, lse, *st.want(q, dim ** -0.5), st.dtype)
    for _ in range(3):  # the joins leave their counters clear, and the order of arrival does not show
        again, lse2 = A.tree_attention(cache, 0, batch, q.cuda(), lse=True)
        assert torch.equal(again, out) and torch.equal(lse2, lse)


@pytest.mark.parametrize("layout", ["hpd", "phd"])
def test_attention_strides_scale_and_unaligned_rows(A, layout):
    st = Step([5, 2], [90, 33], 2, 128, 32, "f16", tree=random_tree, seed=8, layout=layout, stale=math.inf)
    cache, batch = st.device(A)
    wide = torch.randn((7, 6 * 128 + 3), generator=torch.Generator().manual_seed(3)).half()
    q = wide[:, 3:].unflatten(1, (6, 128))  # rows 2 bytes off any vector's alignment
    buf = torch.full((7, 6 * 128 + 5), 7.0, dtype=torch.float16, device="cuda")
    out = buf[:, 5:].unflatten(1, (6, 128))
    big = wide.cuda()
    lse = torch.empty((7, 6), device="cuda")
    A.tree_attention(cache, st.layer, batch, big[:, 3:].unflatten(1, (6, 128)), scale=0.3, out=out, lse=lse)
    check_attention(out, lse, *st.want(q, 0.3), st.dtype)
    assert bool((buf[:, :5] == 7).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [6, 40])
def test_rows_that_see_nothing_and_other_branches_infinities(A, dtype, rows):
    """Row 1 of a sequence without context sees nothing; the odd rows' v hold infinities and NaN, their k NaN, that only
    the rows that see them may show."""
    def tree(s, n):
        return [0 if i == 1 else (1 << i) | (1 if i else 0) for i in range(n)], [0] * n
    st = Step([rows, rows], [0, 50], 2, 128, 16, dtype, tree=tree, seed=3)
    for s in range(2):
        pg, of = R.slots(st.table[s], 16, st.lens[s], st.lens[s] + rows)
        st.v[st.layer, pg[3], 1, of[3], 5] = math.inf
        st.v[st.layer, pg[4], 0, of[4], 77] = -math.inf
        st.v[st.layer, pg[5], :, of[5], 64:] = math.nan
        st.k[st.layer, pg[2], :, of[2]] = math.nan
    cache, batch = st.device(A)
    q = torch.randn((2 * rows, 4, 128), generator=torch.Generator().manual_seed(4)).to(st.dtype)
    out, lse = A.tree_attention(cache, st.layer, batch, q.cuda(), lse=True)
    want, wlse, mass = st.want(q, 128 ** -0.5)
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(out.cpu()), torch.isnan(want))
    assert torch.equal(torch.isinf(out.cpu()), torch.isinf(want)) and bool((out.cpu().double()[torch.isinf(want)] == want[torch.isinf(want)]).all())
    assert bool((out[1] == 0).all()) and bool(torch.isneginf(lse[1]).all())
    nan = torch.isnan(wlse)
    assert torch.equal(torch.isnan(lse.cpu()), nan)
    clean = torch.where(odd, 0.0, want)
    check_attention(torch.where(odd.cuda(), 0.0, out), torch.where(nan.cuda(), 0.0, lse), clean,
                    torch.where(nan, 0.0, wlse), torch.where(torch.isfinite(mass), mass, 0.0), st.dtype)


def test_attention_large_scores_and_equal_keys(A):
    """Scores in the hundreds (the running maximum moves late), and one value repeated."""
    st = Step([4], [517], 1, 128, 64, "f16", seed=9, layers=1)
    st.k[:] = st.k[:].sort(dim=3).values * 6
    cache, batch = st.device(A)
    q = torch.randn((4, 4, 128), generator=torch.Generator().manual_seed(5)).half() * 3
    out, lse = A.tree_attention(cache, 0, batch, q.cuda(), lse=True)
    want, wlse, mass = st.want(q, 128 ** -0.5)
    # scores reach some 10^3: their f32 sums carry 2^-23 of sum |q k| scale each, so the probabilities 2^-10
    tol = U[st.dtype] * want.abs() + (U[st.dtype] + 2.0 ** -9) * mass + 1e-6
    assert bool(((out.cpu().double() - want).abs() <= tol).all())
    assert bool(((lse.cpu().double() - wlse).abs() <= 2.0 ** -9 + 2.0 ** -20 * wlse.abs()).all())


def test_attention_padding_rows_and_no_rows(A):
    st = Step([2, 3], [20, 0], 2, 64, 16, "bf16", seed=11)
    cache, batch = st.device(A, rows=9)
    q = torch.randn((9, 4, 64), generator=torch.Generator().manual_seed(6)).bfloat16()
    out = torch.full((9, 4, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((9, 4), 3.0, device="cuda")
    A.tree_attention(cache, st.layer, batch, q.cuda(), out=out, lse=lse)
    want, wlse, mass = st.want(q[:5], 64 ** -0.5)
    check_attention(out[:5], lse[:5], want, wlse, mass, st.dtype)
    assert bool((out[5:] == 3).all()) and bool((lse[5:] == 3).all())
    empty = A.TreeBatch(torch.zeros(1, dtype=torch.int32).cuda(), torch.zeros(0, dtype=torch.int32).cuda(),
                        torch.zeros((0, 1), dtype=torch.int32).cuda(), max_rows=0)
    assert A.tree_attention(cache, 0, empty, q[:0].cuda()).shape == (0, 4, 64)


def test_attention_in_a_graph_on_another_stream(A):
    st = Step([1, 1], [100, 40], 2, 128, 16, "bf16", seed=12)
    cache, batch = st.device(A)
    q = torch.randn((2, 8, 128), generator=torch.Generator().manual_seed(7)).bfloat16().cuda()
    plain = A.tree_attention(cache, st.layer, batch, q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = A.tree_attention(cache, st.layer, batch, q, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(plain, other)
    out = torch.empty_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        A.tree_attention(cache, st.layer, batch, q, out=out)
    batch._keep[1].fill_(7)  # other contexts, other queries: the replay reads them
    q.mul_(-1)
    g.replay()
    st.lens = [7, 7]
    want, wlse, mass = st.want(q.cpu(), 128 ** -0.5)
    check_attention(out, wlse, want, wlse, mass, st.dtype)


def test_device_values_out_of_range_are_recorded_not_followed(A):
    from plugins_b200 import quant as Q
    st = Step([2], [40], 2, 128, 16, "f16", seed=13)
    st.table[0, 1] = st.pages + 1000
    cache, batch = st.device(A)
    q = torch.randn((2, 2, 128)).half().cuda()
    A.tree_attention(cache, st.layer, batch, q)
    assert Q.device_error(0, clear=True) & L.ERR_BAD_SHAPE
    batch._keep[1].fill_(10 ** 6)
    A.tree_attention(cache, st.layer, batch, q)
    assert Q.device_error(0, clear=True) & L.ERR_BAD_SHAPE
    rope = A.NormRope(torch.ones(64, dtype=torch.float64).cuda())
    A.qk_norm_rope(cache, st.layer, batch, q, q, q, rope)
    assert Q.device_error(0, clear=True) & L.ERR_BAD_SHAPE


# ------------------------------------------------------------------ norms and rotation

def check_rounded(got, want, scale, dtype):
    """One rounding of the result, and f32 arithmetic: the sum of dim squares (relative 2^-22), a reciprocal root, two
    products and one sum, the sine and cosine of an angle good to 2^-24 turns: 2^-20 of the vector's size."""
    tol = U[dtype] * want.abs() + 2.0 ** -20 * scale + TINY[dtype]
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), f"worst {float((err / tol).max()):.2f} x the tolerance"


@pytest.mark.parametrize("dim,rot,adjacent", [(128, 128, False), (128, 128, True), (128, 96, False), (64, 16, False),
                                              (64, 10, True), (256, 64, False), (256, 256, True), (128, 0, False)])
@pytest.mark.parametrize("dtype,cdtype", [("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16"), ("f32", "f16"),
                                          ("bf16", "f16")])
@pytest.mark.parametrize("layout", ["hpd", "phd"])
def test_norm_rope(A, dim, rot, adjacent, dtype, cdtype, layout):
    st = Step([1, 0, 37, 4], [0, 9, 100, 70000], 2, dim, 32, cdtype, seed=dim + rot, layout=layout, layers=2)
    cache, batch = st.device(A)
    g = torch.Generator().manual_seed(rot)
    n, heads = 42, 6
    qkv = (torch.randn((n, heads + 4, dim), generator=g) * 3).to(DT[dtype])
    qw, kw = ((1 + 0.2 * torch.randn(dim, generator=g)).to(DT[dtype]) for _ in range(2))
    inv = 1e6 ** (-torch.arange(rot // 2, dtype=torch.float64) / max(1, rot // 2))
    rope = A.NormRope(inv.cuda() if rot else None, qw.cuda(), kw.cuda(), eps=1e-5, adjacent=adjacent)
    dev = qkv.cuda()
    out = A.qk_norm_rope(cache, st.layer, batch, dev[:, :heads], dev[:, heads:heads + 2], dev[:, heads + 2:], rope)
    pos = torch.cat([torch.arange(c, c + r) for r, c in zip(st.rows, st.lens)])
    size = lambda x, w: (x.double() / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + 1e-5) * w.double()).abs().amax(-1, keepdim=True)  # noqa: E731
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + 2], qkv[:, heads + 2:]
    check_rounded(out, R.norm_rotate(q, qw, pos, inv, 1e-5, adjacent), size(q, qw), DT[dtype])
    wk, wv = st.k.double(), st.v.double()
    ks = torch.zeros_like(wk)
    nk = R.norm_rotate(k, kw, pos, inv, 1e-5, adjacent)
    for s in range(4):
        a, b = st.row_start[s], st.row_start[s + 1]
        pg, of = R.slots(st.table[s], 32, st.lens[s], st.lens[s] + b - a)
        wk[st.layer, pg, :, of] = nk[a:b]
        wv[st.layer, pg, :, of] = v[a:b].to(st.dtype).double()
        ks[st.layer, pg, :, of] = size(k[a:b], kw).expand(-1, -1, dim)
    check_rounded(cache.k, wk, ks, st.dtype)
    assert torch.equal(cache.v.cpu().double(), wv)


def test_norm_rope_in_place_narrowed_offset_and_given_positions(A):
    st = Step([3, 9], [5, 60], 1, 128, 16, "bf16", tree=random_tree, seed=21)
    cache, batch = st.device(A)
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn((12, h, 128), generator=g) for h in (4, 1, 1))
    qw, kw = (0.3 * torch.randn(128, generator=g) for _ in range(2))
    inv = 1e4 ** (-torch.arange(64, dtype=torch.float64) / 64)
    rope = A.NormRope(inv.cuda(), qw.cuda(), kw.cuda(), eps=1e-6, weight_offset=1.0)
    want = R.norm_rotate(q, qw, st.position, inv, 1e-6, False, offset=1.0)
    size = want.abs().amax(-1, keepdim=True) * 2
    narrow = A.qk_norm_rope(cache, st.layer, batch, q.cuda(), k.cuda(), v.cuda(), rope,
                            out=torch.empty((12, 4, 128), dtype=torch.bfloat16, device="cuda"))
    check_rounded(narrow, want, size, torch.bfloat16)
    dev = q.cuda()
    assert A.qk_norm_rope(cache, st.layer, batch, dev, k.cuda(), v.cuda(), rope, out=dev) is dev
    check_rounded(dev, want, size, torch.float32)
    only = A.NormRope(None)  # neither norm nor rotation: a copy and an append
    same = A.qk_norm_rope(cache, st.layer, batch, q.cuda(), k.cuda(), v.cuda(), only)
    assert torch.equal(same.cpu(), q)


def test_norm_rope_unaligned_rows_and_padding(A):
    st = Step([2], [3], 2, 64, 16, "f16", seed=22)
    cache, batch = st.device(A, rows=4)
    wide = torch.randn((4, 8 * 64 + 1), generator=torch.Generator().manual_seed(1)).half()
    rows = wide.cuda()[:, 1:].unflatten(1, (8, 64))
    inv = 1e4 ** (-torch.arange(32, dtype=torch.float64) / 32)
    before = cache.k.clone()
    out = torch.full((4, 4, 64), 5.0, dtype=torch.float16, device="cuda")
    A.qk_norm_rope(cache, st.layer, batch, rows[:, :4], rows[:, 4:6], rows[:, 6:], A.NormRope(inv.cuda()), out=out)
    want = R.norm_rotate(wide[:2, 1:].unflatten(1, (8, 64))[:, :4], None, torch.tensor([3, 4]), inv, 0, False)
    check_rounded(out[:2], want, want.abs().amax(-1, keepdim=True) * 2, torch.float16)
    assert bool((out[2:] == 5).all())
    assert int((cache.k != before).any(-1).sum()) == 4  # two tokens, two heads


def test_norm_rope_many_rows_and_sequences(A):
    """Rows of many sequences (the search for a row's owner), some of them empty."""
    r = random.Random(3)
    rows = [r.choice([0, 1, 1, 2, 5]) for _ in range(1500)]
    st = Step(rows, [r.randrange(40) for _ in rows], 1, 64, 16, "bf16", seed=23, layers=1)
    cache, batch = st.device(A)
    n = st.row_start[-1]
    x = torch.randn((n, 3, 64), generator=torch.Generator().manual_seed(2)).bfloat16()
    dev = x.cuda()
    A.qk_norm_rope(cache, 0, batch, dev[:, :1], dev[:, 1:2], dev[:, 2:], A.NormRope(None))
    seq = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor(rows))
    at = torch.arange(n) - torch.tensor(st.row_start)[seq] + torch.tensor(st.lens)[seq]
    pg = st.table[seq, at // 16].long()
    assert torch.equal(cache.v.cpu()[0][pg, 0, at % 16], x[:, 2])
    assert torch.equal(cache.k.cpu()[0][pg, 0, at % 16], x[:, 1])


@pytest.mark.parametrize("which", ["q", "k"])
@pytest.mark.parametrize("dim,heads,kv_heads,rows", [(128, 40, 12, 700), (64, 3, 1, 900), (256, 7, 3, 650)])
def test_norm_rope_one_norm_many_heads_and_rows(A, which, dim, heads, kv_heads, rows):
    """A norm of the queries or of the keys alone (their heads share warps), several rows and batches of heads a CTA."""
    st = Step([rows // 2, rows - rows // 2], [17, 0], kv_heads, dim, 32, "bf16", seed=dim)
    cache, batch = st.device(A)
    g = torch.Generator().manual_seed(heads)
    x = (torch.randn((rows, heads + 2 * kv_heads, dim), generator=g) * 3).bfloat16()
    w = (1 + 0.2 * torch.randn(dim, generator=g)).bfloat16()
    inv = 1e4 ** (-torch.arange(dim // 2, dtype=torch.float64) / (dim // 2))
    rope = A.NormRope(inv.cuda(), w.cuda() if which == "q" else None, w.cuda() if which == "k" else None)
    dev = x.cuda()
    parts = (x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:])
    out = A.qk_norm_rope(cache, st.layer, batch, dev[:, :heads], dev[:, heads:heads + kv_heads],
                         dev[:, heads + kv_heads:], rope)
    pos = torch.cat([torch.arange(c, c + r) for r, c in zip(st.rows, st.lens)])
    want_q = R.norm_rotate(parts[0], w if which == "q" else None, pos, inv, 1e-6, False)
    want_k = R.norm_rotate(parts[1], w if which == "k" else None, pos, inv, 1e-6, False)
    check_rounded(out, want_q, want_q.abs().amax(-1, keepdim=True) * 2, st.dtype)
    seq = torch.repeat_interleave(torch.arange(2), torch.tensor(st.rows))
    at = torch.arange(rows) - torch.tensor(st.row_start)[seq] + torch.tensor(st.lens)[seq]
    pg = st.table[seq, at // 32].long()
    got_k = cache.k[st.layer].cpu()[pg, :, at % 32]
    check_rounded(got_k, want_k, want_k.abs().amax(-1, keepdim=True) * 2, st.dtype)
    assert torch.equal(cache.v[st.layer].cpu()[pg, :, at % 32], parts[2])


@pytest.mark.parametrize("rows", [2, 24])
def test_slots_past_two_to_the_31_elements(A, rows):
    """A pool of 2.3e9 elements, the sequence in its last pages: append, attention, and a copy of pages out there."""
    pages, kvh, page, dim = 70000, 8, 64, 64
    k, v = (torch.empty((1, pages, kvh, page, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    st = Step([rows], [70], kvh, dim, page, "bf16", tree=chain, seed=31, layers=1, spare=0)
    lo = pages - st.pages
    k[:, lo:], v[:, lo:] = st.k.cuda(), st.v.cuda()
    cache = A.KvCache(k, v)
    batch = A.TreeBatch(torch.tensor(st.row_start, dtype=torch.int32).cuda(), torch.tensor(st.lens, dtype=torch.int32).cuda(),
                        torch.where(st.table >= 0, st.table + lo, -1).int().cuda(), max_rows=rows, tree=st.tree.cuda())
    g = torch.Generator().manual_seed(1)
    q, kk, vv = (torch.randn((rows, h, dim), generator=g).bfloat16() for h in (16, kvh, kvh))
    A.qk_norm_rope(cache, 0, batch, q.cuda(), kk.cuda(), vv.cuda(), A.NormRope(None))
    pg, of = R.slots(st.table[0], page, 70, 70 + rows)
    st.k[0, pg, :, of], st.v[0, pg, :, of] = kk, vv
    assert torch.equal(k[:, lo:].cpu(), st.k)
    out, lse = A.tree_attention(cache, 0, batch, q.cuda(), lse=True)
    check_attention(out, lse, *st.want(q, dim ** -0.5), st.dtype)
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[pages - 1] = 2
    refs[:pages - 3] = 1
    i32 = (lambda x: torch.tensor(x, dtype=torch.int32).cuda())
    state = A.PageState(refs.cuda(), i32([[pages - 1], [pages - 1]]), i32([1, 1]), i32([9, 9]))
    grown, missing = A.cache_grow(cache, state, i32([10, 9]))
    assert int(missing) == 0 and grown.table.tolist() == [[pages - 3], [pages - 1]]
    assert torch.equal(k[0, pages - 3], k[0, pages - 1]) and torch.equal(v[0, pages - 3], v[0, pages - 1])


def test_broadcast_queries_and_one_key_for_all_heads(A):
    """Inputs of stride 0: one query vector for every row and head, one k and v vector for every kv head."""
    st = Step([3], [20], 2, 64, 16, "f16", seed=41)
    cache, batch = st.device(A)
    x = torch.randn((3, 1, 64), generator=torch.Generator().manual_seed(3)).half()
    one = x.cuda().expand(3, 2, 64)
    A.qk_norm_rope(cache, st.layer, batch, x.cuda()[:1].expand(3, 4, 64), one, one, A.NormRope(None))
    pg, of = R.slots(st.table[0], 16, 20, 23)
    st.k[st.layer, pg, :, of] = st.v[st.layer, pg, :, of] = x.expand(3, 2, 64)
    assert torch.equal(cache.k.cpu(), st.k) and torch.equal(cache.v.cpu(), st.v)
    q = x[:1].expand(3, 4, 64)
    out, lse = A.tree_attention(cache, st.layer, batch, x.cuda()[:1].expand(3, 4, 64), lse=True,
                                out=torch.empty((3, 4, 64), dtype=torch.float16, device="cuda"))
    check_attention(out, lse, *st.want(q, 64 ** -0.5), st.dtype)
