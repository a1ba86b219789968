"""Decoding with drafted trees over EXL3 layers: the linears of :mod:`plugins_b200.quant` and the attention side
of :mod:`plugins_b200.attention` run together as a serving loop runs them.

A step takes every sequence's last token and a tree of drafted continuations through the layers at once (one row per
token), accepts drafts by the model's probabilities (its own choices, at temperature 0), keeps the accepted rows in the cache
and frees nothing it may still need.  With a budget, rows that outgrow it keep the tokens that were attended to most:

    dec = TreeDecoder(layers, embed, heads=32, kv_heads=8, head_dim=128, pages=4096, page_size=64, nseq=8,
                      temperature=0.8, budget=2048)
    first = dec.prompt(prompts)                   # causal chunks of any lengths -> each sequence's next token
    got = dec.step([tree, ...])                   # tree: [(parent, token), ...] below the last token (parent -1)

    python -m plugins_b200.tree_decode            # a small random stack, decoded with and without drafts, and on a budget
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
    """``embed`` [vocab, hidden] embeds tokens and, transposed, scores them.  ``temperature`` (0: greedy) and ``seed`` are of
    the sampled tokens.  ``budget``: once a row has more than ``budget`` + ``recent`` tokens, the rows are cut to ``budget`` of
    them: the first ``sink``, the last ``recent`` and the most attended to (rejected drafts' attention counts too), what they
    had falling by ``decay`` a step."""

    def __init__(self, layers: list[Layer], embed: torch.Tensor, heads: int, kv_heads: int, head_dim: int, pages: int,
                 page_size: int, nseq: int, max_pages: int | None = None, eps: float = 1e-6, temperature: float = 0.0,
                 seed: int = 0, budget: int | None = None, sink: int = 4, recent: int = 32, decay: float = 1.0):
        if budget is not None and budget < sink + recent:
            raise ValueError("a budget below the tokens that always stay")
        self.layers, self.embed, self.eps = layers, embed, eps
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.cache = A.KvCache.empty(len(layers), pages, page_size, kv_heads, head_dim, embed.dtype, embed.device)
        self.state = A.PageState.empty(self.cache, nseq, max_pages or pages)
        self.temperature, self.random = float(temperature), torch.Generator(embed.device).manual_seed(seed)
        self.budget, self.sink, self.recent, self.decay = budget, sink, recent, decay
        self.weight = None  # how much each cached token was attended to
        if budget is not None:
            self.weight = torch.zeros((len(layers), nseq, kv_heads, (max_pages or pages) * page_size), device=embed.device)
        self.lens = [0] * nseq    # tokens in the cache, the host's copy
        self.seen = [0] * nseq    # tokens a row has had: the next one's position
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
            if self.weight is None:
                o = A.tree_attention(self.cache, i, batch, q)
            else:
                o, lse = A.tree_attention(self.cache, i, batch, q, lse=True)
                A.attention_weight(self.cache, i, batch, q, lse, self.weight[i], decay=self.decay)
            x = x + Q.matmul(la.o, o.view(rows, -1))
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

    def _logits(self, x: torch.Tensor) -> torch.Tensor:
        return x.float() @ self.embed.float().T

    def _verify(self, x: torch.Tensor, batch: A.TreeBatch, tokens: torch.Tensor, parent, depth: int, draft=None):
        """Which of the rows stay, by their hidden states, and each sequence's token after them (on the device and here)."""
        n, dev = batch.nseq, self.embed.device
        uniform = torch.rand((x.shape[0], 2), generator=self.random, device=dev)
        path, kept, token = A.draft_verify(self.cache, batch, self._logits(x), tokens, parent, uniform,
                                           torch.full((n,), self.temperature, device=dev), draft, depth=depth)
        after = token.tolist()
        if min(after) < 0:
            raise RuntimeError(f"no token has a probability in sequence {after.index(-1)}: its logits are NaN or -inf")
        return path, kept, after

    def _choices(self, x: torch.Tensor) -> list[int]:
        return self._logits(x).argmax(-1).tolist()

    def _follow(self, choice: list[int], tokens: list[int], parents: list[list], counts: list[int]):
        """The model's own choices down each tree -> its path, and the choice after it (trees and vocabularies of any size)."""
        paths, after, row0 = [], [], 0
        for par, count in zip(parents, counts):
            path, at = [0], 0
            while True:  # the drafted child the model would have chosen
                nxt = next((i for i in range(at + 1, count) if par[i] == at and tokens[row0 + i] == choice[row0 + at]), None)
                if nxt is None:
                    break
                path.append(nxt)
                at = nxt
            paths.append(path)
            after.append(choice[row0 + at])
            row0 += count
        return paths, after

    def _commit(self, batch: A.TreeBatch, path, kept: torch.Tensor, counts: list[int]) -> None:
        A.cache_keep(self.cache, batch, path, kept, out=self.state.lens, weight=self.weight)
        self.lens = [n + k for n, k in zip(self.lens, counts)]
        self.seen = [n + k for n, k in zip(self.seen, counts)]
        if self.budget is not None and max(self.lens) > self.budget + self.recent:
            self._cut()  # (rows that cannot be cut yet are left to the next step: this one's tokens are not lost)

    def evict(self) -> None:
        """Cuts every row to the budget."""
        missing = self._cut()
        if missing:
            raise RuntimeError(f"the cache lacks {missing} pages")

    def _cut(self) -> int:
        """Cuts the rows to the budget, together, or, where the free pages do not suffice for all that share some, one after the
        other: a row that is cut gives pages back, and those it shared may be another's alone by then -> the pages lacking for
        the rows that had to be left."""
        def cut(rows) -> int:
            budget = self._ints([self.budget if i in rows else 0x7FFFFFFF for i in range(len(self.lens))])
            self.state, missing = A.cache_evict(self.cache, self.state, self.weight, budget, self.sink, self.recent)
            lacking = int(missing)
            if not lacking:
                self.lens = [min(n, self.budget) if i in rows else n for i, n in enumerate(self.lens)]
            return lacking

        lacking = cut(range(len(self.lens)))
        left, before = [i for i, n in enumerate(self.lens) if lacking and n > self.budget], None
        while left and left != before:
            before = left
            left = [i for i in left if cut((i,))]
        return cut(left) if left else 0

    def prompt(self, prompts: list[list[int]]) -> list[int]:
        """Every sequence's prompt in one pass -> its next token."""
        if len(prompts) != len(self.lens) or not all(prompts):
            raise ValueError(f"a prompt of at least one token for each of the {len(self.lens)} sequences")
        counts = [len(p) for p in prompts]
        places = [n + i for n, c in zip(self.seen, counts) for i in range(c)]
        batch = self._batch(counts, depth=self._ints(places))
        tokens = self._ints([t for p in prompts for t in p])
        x = self.forward(tokens, batch)
        ends = [0]
        for c in counts:
            ends.append(ends[-1] + c)
        rows = [e - 1 for e in ends[1:]]
        if self.temperature == 0:
            self.last = self._choices(x[rows])
        else:
            last = A.TreeBatch(self._ints(list(range(len(rows) + 1))), self.state.lens, self.state.table, max_rows=1, rows=len(rows))
            self.last = self._verify(x[rows], last, tokens[rows], None, 1)[2]
        self._commit(batch, None, self._ints(counts), counts)
        return list(self.last)

    def step(self, trees: list[list[tuple[int, int]]], draft: torch.Tensor | None = None) -> list[list[int]]:
        """One pass over every sequence's last token (row 0 of its tree) and its drafts -> the tokens each gained.  ``draft``
        [rows, vocab]: the probabilities each row's children were drawn from, where the drafter has any."""
        if len(trees) != len(self.lens) or any(not -1 <= p < i for tree in trees for i, (p, _) in enumerate(tree)):
            raise ValueError(f"a tree for each of the {len(self.lens)} sequences, every parent -1 or before its child")
        tokens, parents, counts = [], [], []
        for last, tree in zip(self.last, trees):
            tokens += [last] + [t for _, t in tree]
            parents.append([None] + [p + 1 for p, _ in tree])
            counts.append(len(tree) + 1)
        words = -(-max(counts) // 32)
        bits, place = [], []
        for n, par in zip(self.seen, parents):
            seen, depth = [], []
            for i, p in enumerate(par):
                seen.append((seen[p] if p is not None else 0) | 1 << i)
                depth.append(depth[p] + 1 if p is not None else 0)
            for s, d in zip(seen, depth):
                w = [(s >> (32 * k)) & 0xFFFFFFFF for k in range(words)]
                bits.append([x - (1 << 32) if x >> 31 else x for x in w])
                place.append(n + d)
        batch = self._batch(counts, self._ints(bits), self._ints(place))
        rows = self._ints(tokens)
        x = self.forward(rows, batch)
        if self.temperature == 0:
            paths, self.last = self._follow(self._choices(x), tokens, parents, counts)
            stay = [len(p) for p in paths]
            path, kept = self._ints([p + [-1] * (max(stay) - len(p)) for p in paths]), self._ints(stay)
        else:
            parent = self._ints([-1 if p is None else p for par in parents for p in par])
            deep = max(p - n for n, c, at in zip(self.seen, counts, self._starts(counts)) for p in place[at:at + c]) + 1
            path, kept, self.last = self._verify(x, batch, rows, parent, deep, draft)
            paths, stay = path.tolist(), kept.tolist()
        self._commit(batch, path, kept, stay)
        return [[tokens[at + i] for i in p[1:k]] + [t] for at, p, k, t in zip(self._starts(counts), paths, stay, self.last)]

    @staticmethod
    def _starts(counts: list[int]) -> list[int]:
        return [sum(counts[:i]) for i in range(len(counts))]

    def reorder(self, parent: list[int]) -> None:
        """Row i becomes row parent[i] (a fork when named twice); rows nobody names give their pages back."""
        if not all(0 <= p < len(self.lens) for p in parent):
            raise ValueError(f"parents are among the {len(self.lens)} rows")
        self.state = A.cache_fork(self.cache, self.state, self._ints(parent))
        self.lens, self.last, self.seen = ([v[p] for p in parent] for v in (self.lens, self.last, self.seen))
        if self.weight is not None:
            self.weight = self.weight[:, parent]


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
    small = TreeDecoder(layers, embed, heads, kv_heads, dim, pages=64, page_size=16, nseq=3, max_pages=16, temperature=80,
                        budget=32, sink=2, recent=8)
    small.prompt(prompts)
    count = sum(len(g) for _ in range(16) for g in small.step([[(-1, 5), (0, 6)]] * 3))
    print(f"{count} sampled tokens on a budget of 32: {small.lens} cached of {small.seen}")


if __name__ == "__main__":
    main()
