"""Greedy decoding with drafted trees over EXL3 layers: the linears of :mod:`plugins_b200.quant` and the attention side
of :mod:`plugins_b200.attention` run together as a serving loop runs them.

A step takes every sequence's last token and a tree of drafted continuations through the layers at once (one row per
token), follows the model's own choices down each tree, keeps the accepted rows in the cache and frees nothing it may
still need:

    dec = TreeDecoder(layers, embed, heads=32, kv_heads=8, head_dim=128, pages=4096, page_size=64, nseq=8)
    first = dec.prompt(prompts)                   # causal chunks of any lengths -> each sequence's next token
    got = dec.step([tree, ...])                   # tree: [(parent, token), ...] below the last token (parent -1)

    python -m plugins_b200.tree_decode            # a small random stack, decoded with and without drafts
"""
from __future__ import annotations

import dataclasses

import torch

from . import attention as A
from . import quant as Q


@dataclasses.dataclass
class Layer:
    """One transformer layer: stacked q|k|v and gate|up linears, o and down, and the norms' weights (the model's)."""
    qkv: Q.Weight
    o: Q.Weight
    gate_up: Q.Weight
    down: Q.Weight
    attn_norm: torch.Tensor
    mlp_norm: torch.Tensor
    rope: A.NormRope


def rms(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    f = x.float()
    return (f * torch.rsqrt((f * f).mean(-1, keepdim=True) + eps) * weight.float()).to(x.dtype)


class TreeDecoder:
    """``embed`` [vocab, hidden] embeds tokens and, transposed, scores them."""

    def __init__(self, layers: list[Layer], embed: torch.Tensor, heads: int, kv_heads: int, head_dim: int, pages: int,
                 page_size: int, nseq: int, max_pages: int | None = None, eps: float = 1e-6):
        self.layers, self.embed, self.eps = layers, embed, eps
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.cache = A.KvCache.empty(len(layers), pages, page_size, kv_heads, head_dim, embed.dtype, embed.device)
        self.state = A.PageState.empty(self.cache, nseq, max_pages or pages)
        self.lens = [0] * nseq    # tokens in the cache, the host's copy
        self.last = [None] * nseq  # each sequence's newest token, not in the cache yet

    def _ints(self, v) -> torch.Tensor:
        return torch.tensor(v, dtype=torch.int32, device=self.embed.device)

    def forward(self, tokens: torch.Tensor, batch: A.TreeBatch) -> torch.Tensor:
        """The rows' hidden states after the last layer."""
        x = self.embed[tokens]
        rows, dim = tokens.shape[0], self.head_dim
        for i, la in enumerate(self.layers):
            q, k, v = Q.segment_outputs(la.qkv, Q.matmul(la.qkv, rms(x, la.attn_norm, self.eps)), rows)
            q, k, v = (t.view(rows, -1, dim) for t in (q, k, v))
            q = A.qk_norm_rope(self.cache, i, batch, q, k, v, la.rope, out=q)
            x = x + Q.matmul(la.o, A.tree_attention(self.cache, i, batch, q).view(rows, -1))
            g, u = Q.segment_outputs(la.gate_up, Q.matmul(la.gate_up, rms(x, la.mlp_norm, self.eps)), rows)
            x = x + Q.matmul(la.down, (torch.nn.functional.silu(g.float()) * u.float()).to(x.dtype))
        return x

    def _batch(self, counts: list[int], tree=None, depth=None) -> A.TreeBatch:
        """Pages for the new rows, and the step's description."""
        need = [n + c for n, c in zip(self.lens, counts)]
        self.state, missing = A.cache_grow(self.cache, self.state, self._ints(need))
        if int(missing):
            raise RuntimeError(f"the cache lacks {int(missing)} pages")
        start = [0]
        for c in counts:
            start.append(start[-1] + c)
        return A.TreeBatch(self._ints(start), self.state.lens, self.state.table, max_rows=max(counts), rows=start[-1],
                           max_context=max(need), tree=tree, position=depth)

    def _choices(self, x: torch.Tensor) -> list[int]:
        return (x.float() @ self.embed.float().T).argmax(-1).tolist()

    def _commit(self, batch: A.TreeBatch, path, kept: list[int]) -> None:
        A.cache_keep(self.cache, batch, path, self._ints(kept), out=self.state.lens)
        self.lens = [n + k for n, k in zip(self.lens, kept)]

    def prompt(self, prompts: list[list[int]]) -> list[int]:
        """Every sequence's prompt in one pass -> its next token."""
        if len(prompts) != len(self.lens) or not all(prompts):
            raise ValueError(f"a prompt of at least one token for each of the {len(self.lens)} sequences")
        batch = self._batch([len(p) for p in prompts])
        x = self.forward(torch.tensor([t for p in prompts for t in p], device=self.embed.device), batch)
        ends = [0]
        for p in prompts:
            ends.append(ends[-1] + len(p))
        self.last = self._choices(x[[e - 1 for e in ends[1:]]])
        self._commit(batch, None, [len(p) for p in prompts])
        return list(self.last)

    def step(self, trees: list[list[tuple[int, int]]]) -> list[list[int]]:
        """One pass over every sequence's last token (row 0 of its tree) and its drafts -> the tokens each gained."""
        if len(trees) != len(self.lens) or any(not -1 <= p < i for tree in trees for i, (p, _) in enumerate(tree)):
            raise ValueError(f"a tree for each of the {len(self.lens)} sequences, every parent -1 or before its child")
        tokens, parents, counts = [], [], []
        for last, tree in zip(self.last, trees):
            tokens += [last] + [t for _, t in tree]
            parents.append([None] + [p + 1 for p, _ in tree])
            counts.append(len(tree) + 1)
        words = -(-max(counts) // 32)
        bits, place = [], []
        for n, par in zip(self.lens, parents):
            seen, depth = [], []
            for i, p in enumerate(par):
                seen.append((seen[p] if p is not None else 0) | 1 << i)
                depth.append(depth[p] + 1 if p is not None else 0)
            for s, d in zip(seen, depth):
                w = [(s >> (32 * k)) & 0xFFFFFFFF for k in range(words)]
                bits.append([x - (1 << 32) if x >> 31 else x for x in w])
                place.append(n + d)
        batch = self._batch(counts, self._ints(bits), self._ints(place))
        choice = self._choices(self.forward(torch.tensor(tokens, device=self.embed.device), batch))
        got, paths, row0 = [], [], 0
        for par, count in zip(parents, counts):
            path, at = [0], 0
            while True:  # the drafted child the model would have chosen
                nxt = next((i for i in range(at + 1, count) if par[i] == at and tokens[row0 + i] == choice[row0 + at]), None)
                if nxt is None:
                    break
                path.append(nxt)
                at = nxt
            got.append([choice[row0 + i] for i in path])
            paths.append(path)
            row0 += count
        deep = max(map(len, paths))
        self._commit(batch, self._ints([p + [-1] * (deep - len(p)) for p in paths]), [len(p) for p in paths])
        self.last = [g[-1] for g in got]
        return got

    def reorder(self, parent: list[int]) -> None:
        """Row i becomes row parent[i] (a fork when named twice); rows nobody names give their pages back."""
        if not all(0 <= p < len(self.lens) for p in parent):
            raise ValueError(f"parents are among the {len(self.lens)} rows")
        self.state = A.cache_fork(self.cache, self.state, self._ints(parent))
        self.lens, self.last = [self.lens[p] for p in parent], [self.last[p] for p in parent]


def random_layers(count: int, hidden: int, heads: int, kv_heads: int, head_dim: int, inter: int, seed: int = 0,
                  dtype=torch.bfloat16, theta: float = 1e6) -> list[Layer]:
    """Layers of random EXL3 linears (4 bits) and norms near one."""
    from . import encoder as E
    g = torch.Generator(device="cuda").manual_seed(seed)
    inv = theta ** (-torch.arange(head_dim // 2, dtype=torch.float64, device="cuda") / (head_dim // 2))

    def linear(i, o, s):
        return Q.weight_from_tensors(*E.random_linear(i, o, 64, seed=seed * 1000 + s))

    def norm(n):
        return (1 + 0.1 * torch.randn(n, generator=g, device="cuda")).to(dtype)

    out = []
    for c in range(count):
        s = 10 * c
        qkv = Q.stack([linear(hidden, heads * head_dim, s), linear(hidden, kv_heads * head_dim, s + 1),
                       linear(hidden, kv_heads * head_dim, s + 2)])
        out.append(Layer(qkv, linear(heads * head_dim, hidden, s + 3),
                         Q.stack([linear(hidden, inter, s + 4), linear(hidden, inter, s + 5)]), linear(inter, hidden, s + 6),
                         norm(hidden), norm(hidden), A.NormRope(inv, norm(head_dim), norm(head_dim))))
    return out


def main() -> None:
    heads, kv_heads, dim, hidden, vocab = 8, 2, 128, 1024, 2048
    layers = random_layers(4, hidden, heads, kv_heads, dim, 2048)
    embed = torch.randn((vocab, hidden), generator=torch.Generator("cuda").manual_seed(9), device="cuda").bfloat16()
    prompts = [[(7 * i + s) % vocab for i in range(20 + 13 * s)] for s in range(3)]

    def decoder():
        return TreeDecoder(layers, embed, heads, kv_heads, dim, pages=64, page_size=16, nseq=3, max_pages=16)

    plain, want = decoder(), [[], [], []]
    first = plain.prompt(prompts)
    for _ in range(16):
        for w, g in zip(want, plain.step([[]] * 3)):
            w += g
    drafted, got, steps = decoder(), [[], [], []], 0
    assert drafted.prompt(prompts) == first
    while min(map(len, got)) < 16:
        # a drafter that is right for two tokens and then wrong, beside a wrong branch
        trees = []
        for w, g in zip(want, got):
            right = w[len(g):len(g) + 2]
            trees.append([(i - 1, t) for i, t in enumerate(right)] + [(len(right) - 1, 0), (-1, 1), (len(right) + 1, 2)])
        for g, new in zip(got, drafted.step(trees)):
            g += new
        steps += 1
    same = all(g[:16] == w for g, w in zip(got, want))
    print(f"{sum(map(len, got))} tokens in {steps} drafted steps, as one token at a time: {same}")


if __name__ == "__main__":
    main()
