"""The attention side's kernels where their arithmetic is at its limits (plugins_b200/attention.py)."""
import math

import pytest
import torch

import attention_ref as R
from plugins_b200 import _lib as L

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half an ulp, relative


@pytest.fixture()
def A():
    from plugins_b200 import attention
    from plugins_b200 import quant as Q
    Q.device_error(0, clear=True)
    yield attention
    assert Q.device_error(0, clear=True) == 0


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def close(out, lse, want, wlse, mass, dtype):
    """One rounding of the result and one of the probabilities, relative to what they weigh; scores and sums in f32 (the
    scores here stay below 2^5, their sums' errors below 2^-13)."""
    tol = U[dtype] * want.abs() + (U[dtype] + 2.0 ** -13) * mass + 2.0 ** -25
    err = (out.cpu().double() - want).abs()
    assert bool((err <= tol).all()), f"worst {float((err / tol).max()):.2f} x the tolerance"
    assert bool(((lse.cpu().double() - wlse).abs() <= 2.0 ** -13 + 2.0 ** -21 * wlse.abs()).all())


@pytest.mark.parametrize("context", [2 ** 31 - 1, 2 ** 31 - 40, 1 << 30, 97])
@pytest.mark.parametrize("rows", [2, 24, 90])
@pytest.mark.parametrize("tree", [False, True])
def test_a_context_past_the_table_harms_no_other_sequence(A, context, rows, tree):
    """Contexts whose sums with a row's place pass 32 bits (and one slot too many): recorded, nothing of the sequence is
    written, the sequences beside it are right."""
    from plugins_b200 import quant as Q
    g = torch.Generator().manual_seed(rows)
    page, dim, dtype = 16, 128, torch.bfloat16
    k, v = (torch.randn((1, 30, 2, page, dim), generator=g).to(dtype) for _ in range(2))
    ids = torch.randperm(30, generator=g).int()
    table = torch.full((3, 12), -1, dtype=torch.int32)
    table[0, :12], table[1, :6], table[2, :12] = ids[:12], ids[12:18], ids[18:30]
    lens = [70, context, 100]
    if context == 97:  # the last new row of sequence 1 does not fit its table's six pages, and the seventh is -1
        lens[1] = 6 * page - rows + 1
    start = [0, rows, 2 * rows, 3 * rows]
    bits = None
    if tree:  # a chain
        seen = [[((2 << i) - 1) >> (32 * w) & 0xFFFFFFFF for w in range(3)] for i in range(rows)]
        bits = torch.tensor([[w - (1 << 32) if w >> 31 else w for w in row] for row in seen], dtype=torch.int32).repeat(3, 1)
    cache = A.KvCache(k.cuda(), v.cuda())
    batch = A.TreeBatch(i32(start), i32(lens), table.cuda(), max_rows=rows, rows=3 * rows,
                        tree=None if bits is None else bits.cuda())
    q = torch.randn((3 * rows, 8, dim), generator=g).to(dtype)
    out, lse = A.tree_attention(cache, 0, batch, q.cuda(), lse=True)
    assert Q.device_error(0, clear=True) == L.ERR_BAD_SHAPE
    for s in (0, 2):
        a, b = start[s], start[s + 1]
        want = R.attention(k[0], v[0], q[a:b], [0, rows], [lens[s]], table[s:s + 1], dim ** -0.5,
                           None if bits is None else bits[a:b])
        close(out[a:b], lse[a:b], *want, dtype)
    x = torch.randn((3 * rows, 4, dim), generator=g).to(dtype).cuda()
    A.qk_norm_rope(cache, 0, batch, x[:, :2], x[:, :2], x[:, 2:], A.NormRope(None))
    assert Q.device_error(0, clear=True) == L.ERR_BAD_SHAPE
    for s in (0, 2):
        pg, of = R.slots(table[s], page, lens[s], lens[s] + rows)
        k[0, pg, :, of], v[0, pg, :, of] = x[start[s]:start[s + 1], :2].cpu(), x[start[s]:start[s + 1], 2:].cpu()
    if context == 97:  # those of its rows that have a slot
        pg, of = R.slots(table[1], page, lens[1], 6 * page)
        k[0, pg, :, of], v[0, pg, :, of] = x[rows:2 * rows - 1, :2].cpu(), x[rows:2 * rows - 1, 2:].cpu()
    assert torch.equal(cache.k.cpu(), k) and torch.equal(cache.v.cpu(), v)
    lens2 = A.cache_keep(cache, batch, None, i32([1, 1, 1]))
    if context != 97:
        assert Q.device_error(0, clear=True) == L.ERR_BAD_SHAPE and lens2.tolist() == [71, context, 101]


@pytest.mark.parametrize("rows,dim,page", [(2, 128, 16), (40, 128, 16), (90, 128, 64), (24, 64, 32), (40, 256, 16), (24, 256, 128)])
@pytest.mark.parametrize("bad", [-1, 10 ** 6])
def test_a_page_that_is_not_there_reads_as_zeros(A, rows, dim, page, bad):
    """A page id out of range is recorded; its slots count as zero keys and values, whatever the kernel, and nothing that an
    earlier launch or another sequence left on the chip shows."""
    from plugins_b200 import quant as Q
    g = torch.Generator().manual_seed(rows + dim)
    dtype, ctx = torch.float16, 1000
    held = -(-(ctx + rows) // page)
    k, v = (torch.randn((1, held + 1, 2, page, dim), generator=g).to(dtype) for _ in range(2))
    k[0, held], v[0, held] = 0, 0  # what the missing pages read as
    table = torch.randperm(held, generator=g).int()[None]
    lost = [held // 3, held // 2] if held > 8 else [held // 2]
    cache = A.KvCache(k.cuda(), v.cuda())
    q = torch.randn((rows, 8, dim), generator=g).to(dtype)

    def run(t):
        batch = A.TreeBatch(i32([0, rows]), i32([ctx]), t.cuda(), max_rows=rows, rows=rows)
        return A.tree_attention(cache, 0, batch, q.cuda(), lse=True)

    run(table)  # (leaves other keys behind)
    assert Q.device_error(0, clear=True) == 0
    holes = table.clone()
    holes[0, lost] = bad
    out, lse = run(holes)
    assert Q.device_error(0, clear=True) == L.ERR_BAD_SHAPE
    holes[0, lost] = held
    close(out, lse, *R.attention(k[0], v[0], q, [0, rows], [ctx], holes, dim ** -0.5), dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,dim", [(1, 64), (24, 64), (40, 128), (20, 256)])
def test_many_small_probabilities_beside_a_large_one(A, dtype, rows, dim):
    """2^18 keys of some 2^-23.4 of the first one's probability each, which is below f16's full precision (and its smallest
    numbers): together they are the whole result, since the first key's value is zero.  Enough sequences over the same
    pages that a CTA's part of the keys is long."""
    page, keys, nseq = 256, 1 << 18, 300 if rows == 1 else 40
    dev = dict(dtype=dtype, device="cuda")
    k, v = (torch.zeros((1, keys // page + 1, 1, page, dim), **dev) for _ in range(2))
    v[:] = torch.linspace(0.5, 1.5, dim, **dev)
    c = 23.4 * math.log(2) / math.sqrt(dim)
    k[0, 0, 0, 0], v[0, 0, 0, 0] = c, 0
    table = torch.arange(keys // page + 1, dtype=torch.int32)[None].expand(nseq, -1).contiguous().cuda()
    start = [rows * s for s in range(nseq + 1)]
    batch = A.TreeBatch(i32(start), i32([keys - 1] * nseq), table, max_rows=rows, rows=start[-1])
    q = torch.ones((start[-1], 1, dim), **dev)
    out, lse = A.tree_attention(A.KvCache(k, v), 0, batch, q, lse=True)
    first = math.exp(float(k[0, 0, 0, 0].double().sum()) / math.sqrt(dim))
    rest = torch.tensor([keys - 1 + i for i in range(rows)], dtype=torch.float64).repeat(nseq)[:, None]
    want = (rest / (first + rest))[:, :, None] * v[0, 1, 0, 0].double().cpu()
    close(out, lse, want, torch.log(first + rest), want, dtype)


@pytest.mark.parametrize("rows,dim", [(1, 128), (4, 64), (20, 128), (40, 64), (10, 256)])
@pytest.mark.parametrize("tree", [False, True])
def test_more_sequences_than_threads(A, rows, dim, tree):
    """The line of work is scanned in several runs of sequences, many of them without rows; launches follow one another."""
    nseq, page, dtype = 1000, 16, torch.bfloat16
    g = torch.Generator().manual_seed(rows)
    lens = torch.randint(0, 60, (nseq,), generator=g).tolist()
    count = [rows if x < 0.7 else (1 if x < 0.8 else 0) for x in torch.rand(nseq, generator=g).tolist()]
    start = [0]
    for c in count:
        start.append(start[-1] + c)
    width = (60 + rows) // page + 1
    pages = 512  # (read only: the sequences may share them)
    table = torch.randint(0, pages, (nseq, width), generator=g).int()
    k, v = (torch.randn((1, pages, 1, page, dim), generator=g).to(dtype) for _ in range(2))
    bits = torch.randint(0, 1 << 30, (start[-1], 2), generator=g).int() if tree else None
    batch = A.TreeBatch(i32(start), i32(lens), table.cuda(), max_rows=rows, rows=start[-1], tree=None if bits is None else bits.cuda())
    cache = A.KvCache(k.cuda(), v.cuda())
    q = torch.randn((start[-1], 2, dim), generator=g).to(dtype)
    dev = q.cuda()
    outs = [A.tree_attention(cache, 0, batch, dev, lse=True) for _ in range(4)]
    for out, lse in outs[1:]:
        assert torch.equal(out, outs[0][0]) and torch.equal(lse, outs[0][1])
    out, lse = outs[0]
    sample = [0, 1, 255, 256, 257, 383, 384, 385, 640, nseq - 1] + torch.randint(0, nseq, (25,), generator=g).tolist()
    for s in sample:
        a, b = start[s], start[s + 1]
        want, wlse, mass = R.attention(k[0], v[0], q[a:b], [0, b - a], [lens[s]], table[s:s + 1], dim ** -0.5,
                                       None if bits is None else bits[a:b])
        empty = torch.isneginf(wlse)
        assert torch.equal(torch.isneginf(lse[a:b].cpu()), empty)
        close(out[a:b], torch.where(empty, 0.0, lse[a:b].cpu()), want, torch.where(empty, 0.0, wlse), mass, dtype)


def test_a_tree_without_words_is_refused(A):
    with pytest.raises(A.Exl3Error, match="without words"):
        A.TreeBatch(i32([0, 2]), i32([3]), i32([[0]]), max_rows=2, tree=torch.empty((2, 0), dtype=torch.int32, device="cuda"))
