"""The operators together in the decoder (plugins_b200/tree_decode.py): drafts verified by probabilities, attention weights
kept with the tokens they belong to, rows cut to a budget."""
import pytest
import torch

import evict_ref as E

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, HIDDEN, VOCAB, PAGE = 8, 2, 128, 512, 512, 16
# (the random stack's hidden states are not normalised: its logits spread over a few hundred, hence temperatures of 80)


@pytest.fixture(scope="module")
def make():
    from plugins_b200 import tree_decode as T
    layers = T.random_layers(2, HIDDEN, HEADS, KV, DIM, 1024, seed=3)
    embed = torch.randn((VOCAB, HIDDEN), generator=torch.Generator("cuda").manual_seed(1), device="cuda").bfloat16()
    return lambda nseq, **kw: T.TreeDecoder(layers, embed, HEADS, KV, DIM, pages=120, page_size=PAGE, nseq=nseq, max_pages=16, **kw)


def prompts(*lens):
    return [[(5 * i + s) % VOCAB for i in range(n)] for s, n in enumerate(lens)]


def test_a_budget_that_is_not_reached_changes_nothing(make):
    plain, kept = make(3), make(3, budget=200, recent=16)
    p = prompts(1, 17, 90)
    assert plain.prompt(p) == kept.prompt(p)
    for n in range(8):
        trees = [[(-1, n), (0, 7), (-1, 11)], [], [(-1, 3)]]
        assert plain.step(trees) == kept.step(trees)
    assert plain.lens == kept.lens == kept.seen


def test_the_weights_of_a_step_are_those_of_one_token_at_a_time(make):
    """Drafts that are all accepted: the same rows attend to the same slots, in one step or in several; the bf16
    activations of the two ways differ by a few roundings, which move a weight by a few per cent at most -- a weight
    left at another slot would be off by its whole size."""
    one, drafted = make(1, budget=200), make(1, budget=200)
    p = prompts(40)
    assert one.prompt(p) == drafted.prompt(p)
    got = []
    for _ in range(6):
        got += one.step([[]])[0]
    wrong = (got[0] + 1) % VOCAB
    new = drafted.step([[(-1, wrong)] + [(i if i else -1, t) for i, t in enumerate(got[:5])]])[0]
    assert new == got and drafted.lens == one.lens == [46]
    a, b = one.weight[:, 0, :, 40:46], drafted.weight[:, 0, :, 40:46]  # the new tokens' own
    # the rejected draft sees the context, the last token (slot 40, which it adds to) and itself, none of the accepted drafts
    assert float((a - b)[..., 1:].abs().max()) < 0.1 * float(a[..., 1:].max())
    assert bool((b[..., 0] > a[..., 0]).all())


def test_cut_rows_hold_what_the_plain_eviction_keeps(make):
    from plugins_b200 import quant as Q
    dec = make(3, budget=40, sink=3, recent=10, decay=0.9)
    dec.budget = None  # by hand
    dec.prompt(prompts(30, 77, 50))
    for n in range(3):
        dec.step([[(-1, n)], [], [(-1, 9), (0, 4)]])
    dec.budget = 40
    st = dec.state
    cpu = (lambda t: t.cpu().clone())
    want = E.evict(cpu(dec.cache.k), cpu(dec.cache.v), cpu(dec.weight), st.refs.tolist(), [r[:h] for r, h in zip(st.table.tolist(), st.held.tolist())],
                   st.held.tolist(), st.lens.tolist(), [40] * 3, 3, 10)
    seen = list(dec.seen)
    dec.evict()
    assert torch.equal(dec.cache.k.cpu(), want[0]) and torch.equal(dec.cache.v.cpu(), want[1]) and torch.equal(dec.weight.cpu(), want[2])
    assert dec.state.lens.tolist() == dec.lens == want[6] and dec.seen == seen
    assert Q.device_error(0, clear=True) == 0


def test_decoding_on_a_budget_stays_inside_it(make):
    from plugins_b200 import quant as Q
    dec = make(3, budget=40, sink=3, recent=12, temperature=80.0, seed=4)
    dec.prompt(prompts(30, 77, 5))
    assert dec.lens == [30, 40, 5] and dec.seen == [30, 77, 5]
    total = 0
    for n in range(60):
        new = dec.step([[(-1, n), (0, 7)], [(-1, 3)], []])
        total += sum(map(len, new))
        assert max(dec.lens) <= 52 and dec.state.lens.tolist() == dec.lens
    assert sum(dec.seen) == 112 + total and dec.seen[2] == 65
    refs = [0] * 120
    for row, held in zip(dec.state.table.tolist(), dec.state.held.tolist()):
        for p in row[:held]:
            refs[p] += 1
    assert dec.state.refs.tolist() == refs
    assert Q.device_error(0, clear=True) == 0


def test_forks_on_a_budget_decode_alike(make):
    dec = make(2, budget=40, sink=2, recent=8)
    dec.prompt(prompts(20, 60))
    dec.step([[], []])
    dec.reorder([1, 1])
    for _ in range(30):  # through evictions, which part their pages
        a, b = dec.step([[(-1, 1)], [(-1, 1)]])
        assert a == b
    assert dec.lens[0] == dec.lens[1] and dec.state.table[0].tolist() != dec.state.table[1].tolist()


def test_seeds_and_temperatures(make):
    def run(**kw):
        dec = make(2, **kw)
        out = [dec.prompt(prompts(9, 20))]
        return out + [dec.step([[(-1, i), (-1, i + 1)], []]) for i in range(10)]
    assert run(temperature=80.0, seed=5) == run(temperature=80.0, seed=5)
    assert run(temperature=80.0, seed=5) != run(temperature=80.0, seed=6)
    assert run() == run(seed=6)
    with pytest.raises(ValueError, match="budget"):
        make(1, budget=10, sink=4, recent=8)


def test_the_drafters_probabilities(make):
    """A drafter that draws from the model's own distribution at the root is always accepted there."""
    dec = make(1, temperature=80.0, seed=2)
    dec.prompt(prompts(25))
    last = dec.last[0]
    probe = make(1, temperature=80.0, seed=2)
    probe.prompt(prompts(25))
    x = probe.forward(probe._ints([last]), probe._batch([1], depth=probe._ints(probe.seen)))
    q = torch.softmax((x.float() @ probe.embed.float().T) / 80, 1)
    t = int(torch.multinomial(q[0], 1, generator=torch.Generator("cuda").manual_seed(1)))
    draft = torch.cat([q, q])
    # two rows go through the layers instead of one: their logits differ by bf16 roundings, the ratio p / q stays near 1
    dec.random.manual_seed(0)
    got = dec.step([[(-1, t)]], draft=draft)[0]
    assert got[0] == t and len(got) == 2


def test_the_weights_follow_the_path():
    from plugins_b200 import attention as A
    from plugins_b200 import quant as Q
    cache = A.KvCache.empty(3, 40, 16, 2, 64)
    i = (lambda v: torch.tensor(v, dtype=torch.int32, device="cuda"))
    batch = A.TreeBatch(i([0, 5, 5, 12]), i([20, 9, 0]), i([[0, 1, 2], [3, 4, 5], [6, 7, 8]]), max_rows=7, rows=12)
    w = torch.rand((3, 3, 2, 40), generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    path, kept = i([[0, 2, 4, -1], [-1] * 4, [0, 1, 3, 6]]), i([3, 0, 4])
    want = w.clone()
    want[:, 0, :, 20:23] = w[:, 0, :, [20, 22, 24]]
    want[:, 2, :, 0:4] = w[:, 2, :, [0, 1, 3, 6]]
    got = w.clone()
    lens = A.cache_keep(cache, batch, path, kept, weight=got)
    assert torch.equal(got, want) and lens.tolist() == [23, 9, 4]
    assert torch.equal(w, w) and Q.device_error(0, clear=True) == 0
    same = w.clone()
    A.cache_keep(cache, batch, None, kept, weight=same)
    assert torch.equal(same, w)
    bad = i([[2, 1, 4, -1], [-1] * 4, [0, 1, 3, 9]])  # not ascending; past the rows
    A.cache_keep(cache, batch, bad, kept, weight=same)
    assert torch.equal(same, w) and Q.device_error(0, clear=True) != 0
