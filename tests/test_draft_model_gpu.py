"""Trees of drafted tokens through a small model: ``core.draft_step`` and ``core.GraphedDraftStep`` over a ``PagedKVCache``, ``ops.verify_drafts`` on their logits, the accepted
paths kept, forked sequences, and the generator with drafts.  What plain steps give is the reference (bf16 activations rounded along two routes: the tolerance of
those tests)."""
import random

import pytest
import torch

from daisy_amd import core, ops
from test_core_gpu import DEV, _close
from test_paged_model_gpu import alone, generator, model_and_prompts, paged

pytestmark = pytest.mark.gpu


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def path_to(parents, node):
    out = [node]
    while out[-1] != 0:
        up = parents[out[-1]]
        out.append(up if 0 <= up < out[-1] else 0)      # (any other root has no path from node 0; trees here have none)
    return out[::-1]


def random_tree(r, T):
    return [-1] + [r.randrange(0, i) for i in range(1, T)]


def page_rows(cache, slot):
    """All keys and values of a sequence, in order: [2, L, H, n, D]."""
    n = cache.length(slot)
    pages = cache.page_table[slot, :-(-n // cache.page_size)].long()
    rows = [t[:, pages].permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :n] for t in (cache.k, cache.v)]
    return torch.stack(rows)


@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("D,dtype,window,keep", [(128, torch.bfloat16, 48, None), (64, torch.float16, 20, 32)])
def test_every_node_gives_what_its_path_gives_alone(D, dtype, window, keep, recorded):
    """Trees of two sequences, drafted twice: behind the prompts, and behind an accepted path."""
    T, r = 11, random.Random(5)
    model, prompts, g = model_and_prompts([37, 1], window, D)
    cache = paged(model, 3, dtype=dtype, window=keep)
    with torch.inference_mode():
        core.admit(model, prompts, cache)
        step = core.GraphedDraftStep(model, cache, T) if recorded else lambda *a: core.draft_step(model, a[0], a[1], cache, a[2])
        said = [[], []]                                       # what was accepted of each
        for draft in range(3):
            print(f"draft {draft}", flush=True)
            trees = [random_tree(r, T) for _ in range(3)]
            nodes = [T, 7, 0]
            tokens = torch.randint(2, 96, (3, T), generator=g, device=DEV)
            logits = step(tokens, ints(*trees), nodes).clone()
            torch.cuda.synchronize()
            paths = [path_to(trees[b], r.randrange(nodes[b])) for b in range(2)]
            for b in range(2):
                for node in {0, nodes[b] - 1, paths[b][-1]}:
                    steps = said[b] + [tokens[b, i] for i in path_to(trees[b], node)]
                    _close(logits[b, node], alone(model, prompts[b], steps)[-1], f"draft {draft}, sequence {b}, node {node}")
            path = ints(*([p + [-1] * (T - len(p)) for p in paths + [[]]]))
            assert cache.accept(path, ints(*(len(p) for p in paths), 0)) == [len(paths[0]), len(paths[1]), 0]
            for b in range(2):
                said[b] += [tokens[b, i] for i in paths[b]]
            # a plain step goes on from the accepted path
            token = torch.randint(2, 96, (3,), generator=g, device=DEV)
            got = core.step(model, token, cache)
            for b in range(2):
                said[b].append(token[b])
                _close(got[b], alone(model, prompts[b], said[b])[-1], f"step behind draft {draft}, sequence {b}")
        cache.check()


def test_a_chain_that_is_accepted_leaves_what_plain_steps_leave():
    """Keys and values of the first layer depend on tokens and positions alone: of an accepted path they are bit for bit what single steps write."""
    model, prompts, g = model_and_prompts([30, 16, 5])
    a, b = paged(model, 3), paged(model, 3)
    parents = [-1, 0, 0, 1, 1, 4, 2]
    paths = [[0, 1, 4, 5], [0], [0, 2, 6]]
    tokens = torch.randint(2, 96, (3, 7), generator=g, device=DEV)
    with torch.inference_mode():
        for c in (a, b):
            core.admit(model, prompts, c)
        core.draft_step(model, tokens, ints(*parents), a)
        a.accept(ints(*(p + [-1] * (7 - len(p)) for p in paths)), ints(*(len(p) for p in paths)))
        for n in range(4):
            live = [s for s in range(3) if n < len(paths[s])]
            core.step(model, torch.stack([tokens[s, paths[s][min(n, len(paths[s]) - 1)]] for s in range(3)]), b)
            for s in set(range(3)) - set(live):
                if b.length(s) is not None:
                    assert torch.equal(page_rows(a, s)[:, 0], page_rows(b, s)[:, 0, :, :a.length(s)])
                    b.release(s)
        assert torch.equal(page_rows(a, 0)[:, 0], page_rows(b, 0)[:, 0])
        a.check()
        b.check()


def test_recorded_drafts_are_the_eager_ones_while_sequences_come_and_go():
    T, r = 6, random.Random(1)
    model, prompts, g = model_and_prompts([5, 33, 12])
    a, b = paged(model, 3), paged(model, 3)
    with torch.inference_mode():
        recorded = core.GraphedDraftStep(model, a, T)
        for c in (a, b):
            core.admit(model, prompts[:2], c)
        for n in range(8):
            print(f"recorded draft {n}", flush=True)
            trees, nodes = [random_tree(r, T) for _ in range(3)], [r.randint(0, T) for _ in range(3)]
            tokens = torch.randint(2, 96, (3, T), generator=g, device=DEV)
            x, y = recorded(tokens, ints(*trees), nodes), core.draft_step(model, tokens, ints(*trees), b, nodes)
            torch.cuda.synchronize()
            for s in range(3):
                if b.length(s) is not None:
                    assert torch.equal(x[s, :nodes[s]], y[s, :nodes[s]]), (n, s)
            path, counts, following = ops.verify_drafts(y, tokens, ints(*trees), nodes=ints(*nodes))
            assert a.accept(path, counts) == b.accept(path, counts)
            if n == 2:
                for c in (a, b):
                    core.admit(model, prompts[2:], c)
            if n == 5:
                for c in (a, b):
                    c.release(0)
        for c in (a, b):
            c.check()
        assert a.positions.tolist() == b.positions.tolist() and a._length == b._length
        for s in (1, 2):
            assert torch.equal(page_rows(a, s)[:, [0, 1, 3]], page_rows(b, s)[:, [0, 1, 3]])


@pytest.mark.parametrize("length", [1, 16, 40])
def test_forks_go_on_as_the_sequence_itself_does(length):
    model, prompts, g = model_and_prompts([9, length])
    cache = paged(model, 4)
    with torch.inference_mode():
        core.admit(model, prompts, cache)
        assert cache.fork(1, 2) == [2, 3]
        for s in (2, 3):
            assert torch.equal(page_rows(cache, s), page_rows(cache, 1))
        before = page_rows(cache, 1)
        tokens = torch.randint(2, 96, (20, 4), generator=g, device=DEV)
        for n, t in enumerate(tokens):
            got = core.step(model, t, cache)
            for s in (1, 2, 3):
                _close(got[s], alone(model, prompts[1], tokens[:n + 1, s])[-1], f"fork {s}, step {n}") if n in (0, 1, 19) else None
        assert torch.equal(page_rows(cache, 1)[:, [0, 1, 3]][:, :, :, :length], before[:, [0, 1, 3]])
        cache.release(1)                                     # the others keep the shared pages
        core.admit(model, [prompts[0]], cache)
        got = core.step(model, tokens[0], cache)
        _close(got[3], alone(model, prompts[1], [*tokens[:, 3], tokens[0, 3]])[-1], "a fork without its source")
        cache.check()


# ---------------------------------------------------------------------------------------------------------------
# the generator
# ---------------------------------------------------------------------------------------------------------------
def oracle_drafts(want, firsts, T, wrong=0.3, seed=0, chain=False):
    """Drafts out of the tokens that are to come, some of them wrong: a node's children are the right token and another, in either order."""
    r = random.Random(seed)

    def drafts(seen, lens):
        rows, trees = [], []
        for b, n in enumerate(lens.tolist()):
            tokens, parents = [], []
            at = n - firsts[b]
            last, depth = -1, 0
            while len(tokens) < T:
                right = want[b][min(at + depth, len(want[b]) - 1)]
                other = 2 + (right + 7) % 90
                pair = [other, right] if r.random() < 0.5 else [right, other]
                pair = [right] if chain else pair[:T - len(tokens)]
                if r.random() < wrong:
                    pair = [other] * len(pair)
                place = len(tokens) + (pair.index(right) if right in pair else 0)
                tokens += pair
                parents += [last] * len(pair)
                last, depth = place, depth + 1
            rows.append(tokens)
            trees.append(parents)
        drafts.calls += 1
        return torch.tensor(rows, device=DEV), ints(*trees)
    drafts.calls = 0
    return drafts


@pytest.mark.parametrize("record_steps", [False, True])
@pytest.mark.parametrize("T,wrong", [(1, 0.0), (8, 0.3), (8, 1.0), (20, 0.0)])
def test_greedy_tokens_with_drafts_are_those_without(T, wrong, record_steps):
    """Every token is the likeliest one behind those ahead of it, or as near to that as two routes' logits differ (twice the tolerance of ``_close``)."""
    model, prompts, _ = model_and_prompts([3, 40, 21], seed=4)
    gen = generator(model)
    new = 24
    with torch.inference_mode():
        want = gen.generate_ragged(prompts, new).tolist()
        drafts = oracle_drafts(want, [p.numel() for p in prompts], T, wrong)
        got = gen.generate_ragged(prompts, new, record_steps=record_steps, drafts=drafts).tolist()
        if wrong == 0.0 and T == 20:
            assert drafts.calls <= 6
        for b, prompt in enumerate(prompts):
            for i, row in enumerate(alone(model, prompt, [torch.tensor(t, device=DEV) for t in got[b][:-1]])):
                if 1 in got[b][:i]:
                    assert got[b][i] == 1
                else:
                    assert float(row[:96].max() - row[got[b][i]]) <= 2 * 3e-2 * max(float(row.abs().max()), 1.0), (b, i)
        assert gen.generate_ragged(prompts, new).tolist() == want, "drafts change later calls"


def test_drafts_with_a_bias_a_temperature_and_an_end():
    model, prompts, _ = model_and_prompts([3, 40], seed=4)
    firsts = [3, 40]
    # one token for all: a bias that leaves no choice, whatever is drafted
    for kw in (dict(temperature=0.0), dict(temperature=0.7), dict(temperature=1.3, top_k=5), dict(temperature=1.0, top_p=0.8)):
        gen = generator(model, logit_bias={17: 1000.0}, **kw)
        right = oracle_drafts([[17] * 9] * 2, firsts, 6, 0.2)
        assert gen.generate_ragged(prompts, 9, drafts=right).tolist() == [[17] * 9] * 2
    # scores over a temperature beyond fp16's range (the first token is drawn as ever, in the generator's dtype, where several of them are infinite)
    gen = generator(model, dtype=torch.float16, temperature=1e-5, logit_bias={17: 50.0})
    assert gen.generate_ragged(prompts, 9, drafts=oracle_drafts([[17] * 9] * 2, firsts, 4, 0.2))[:, 1:].tolist() == [[17] * 8] * 2
    # the end of the sequence inside an accepted path, and as the first token
    gen = generator(model, logit_bias={1: 1000.0})
    assert gen.generate_ragged(prompts, 5, drafts=oracle_drafts([[1] * 5] * 2, firsts, 3, 0.0)).tolist() == [[1] * 5] * 2
    # every token is one that a filter lets through
    gen = generator(model, temperature=1.0, top_k=1)
    want = generator(model).generate_ragged(prompts, 12)
    got = gen.generate_ragged(prompts, 12, drafts=oracle_drafts(want.tolist(), firsts, 4, 0.5))
    assert got.shape == want.shape and torch.equal(got[:, 0], want[:, 0])
    # more tokens are drafted than are wanted; a single token needs no draft
    gen = generator(model)
    long = oracle_drafts(want.tolist(), firsts, 200, 0.0)
    assert gen.generate_ragged(prompts, 2, drafts=long).shape == (2, 2) and long.calls <= 1
    assert torch.equal(gen.generate_ragged(prompts, 1, drafts=long), want[:, :1]) and long.calls <= 1


def test_what_does_not_combine_with_drafts_is_refused():
    model, prompts, _ = model_and_prompts([3, 40])
    none = lambda seen, lens: (seen[:, :0], ints(*[[]] * 2))      # noqa: E731
    for kw in (dict(repetition_penalty=1.2), dict(presence_penalty=0.1), dict(frequency_penalty=0.1), dict(allowed_tokens=lambda seen, lens: None)):
        with pytest.raises(ValueError, match="drafts do not combine"):
            generator(model, **kw).generate_ragged(prompts, 4, drafts=none)
    gen = generator(model)
    want = gen.generate_ragged(prompts, 4)
    for bad in (lambda seen, lens: (seen[:, 0], ints(-1)), lambda seen, lens: (seen[:1, :2], ints(-1, -1)), lambda seen, lens: (seen[:, :2], ints(-1)),
                lambda seen, lens: (torch.zeros(2, 256, device=DEV, dtype=torch.long), ints(*[-1] * 256)),
                lambda seen, lens: (torch.full((2, 2), 96, device=DEV), ints(-1, -1)), lambda seen, lens: (torch.full((2, 2), -1, device=DEV), ints(-1, -1))):
        with pytest.raises(ValueError, match="drafts must be"):
            gen.generate_ragged(prompts, 4, drafts=bad)
    with pytest.raises(ZeroDivisionError):
        gen.generate_ragged(prompts, 4, drafts=lambda seen, lens: 1 / 0)
    assert torch.equal(gen.generate_ragged(prompts, 4), want), "a call that failed changes later ones"
    empty = lambda seen, lens: (seen[:, :0], torch.empty(0, dtype=torch.int32, device=DEV))      # noqa: E731
    assert gen.generate_ragged(prompts, 4, drafts=empty).shape == want.shape      # (no drafts: a step of one node)


def test_tokens_drawn_with_drafts_have_the_distribution_that_they_have_without():
    """One prompt 512 times, the second token: counts against the model's own probabilities (chi-squared over the bins that expect 8 or more, against its mean plus 5
    standard deviations)."""
    model, prompts, _ = model_and_prompts([6], seed=2)
    B = 512
    gen = generator(model, temperature=1.0, top_k=6, seed=11)
    g = torch.Generator(device=DEV).manual_seed(3)

    def drafts(seen, lens):
        tokens = torch.randint(2, 96, (seen.size(0), 12), generator=g, device=DEV)
        return tokens, ints(*[-1] * 6, *[0, 0, 1, 1, 2, 2])
    table = gen.generate_ragged([prompts[0]] * B, 2, drafts=drafts).cpu()
    with torch.inference_mode():
        follow = torch.zeros(96)
        for t, n in zip(*table[:, 0].unique(return_counts=True)):
            two = alone(model, prompts[0], [t.to(DEV)])[1][:96].float().cpu().bfloat16().float().topk(6)
            follow[two.indices] += n * two.values.softmax(-1)
    seen = torch.bincount(table[:, 1], minlength=96).float()
    big = follow >= 8
    expect, found = [torch.cat([t[big], t[~big].sum()[None]]) for t in (follow, seen)]
    if expect[-1] < 8:
        expect, found = expect[:-1], found[:-1]
    chi, k = float(((found - expect) ** 2 / expect).sum()), expect.numel()
    print(f"chi2 {chi:.1f} over {k} bins")
    assert chi < k + 5 * (2 * k) ** 0.5
