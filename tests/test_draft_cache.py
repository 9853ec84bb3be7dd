"""The bookkeeping of a paged cache whose steps run trees of drafted tokens, and whose sequences fork: pages, lengths and refusals.  No kernel runs here: the one that
moves rows is replaced by a record of its calls."""
import random
import types

import pytest
import torch

from daisy_amd import CausalSelfAttention, PagedKVCache, core, ops


def cpu_cache(**kw):
    return PagedKVCache(**{**dict(L=2, sequences=4, H=2, D=64, pages=20, device="cpu", dtype=torch.bfloat16, page_size=16, max_len=128), **kw})


@pytest.fixture
def moves(monkeypatch):
    calls = []

    def record(k, v, table, starts, counts, *, rows=None, index=None, sources=None, status=None):
        calls.append(types.SimpleNamespace(table=table.clone(), starts=starts.tolist(), counts=counts.tolist(), rows=rows, index=index,
                                           sources=None if sources is None else sources.tolist()))
    monkeypatch.setattr(ops, "paged_move", record)
    return calls


def ints(*values):
    return torch.tensor(values, dtype=torch.int32)


def state(c):
    return (c.page_table.tolist(), sorted(c._free), list(c._users), [dict(o) for o in c._owned], list(c._reach), list(c._length), c.positions.tolist(), c.lens.tolist())


def consistent(c):
    """Every page is free or has as many owners as it counts, and the table says what the host knows."""
    users = [0] * c.pages
    for owned in c._owned:
        for page in owned.values():
            users[page] += 1
    assert users == c._users and sorted(c._free) == [p for p in range(c.pages) if users[p] == 0]
    for slot, owned in enumerate(c._owned):
        assert {e: p for e, p in enumerate(c.page_table[slot].tolist()) if p >= 0} == owned
        n = c.length(slot)
        assert c.positions[slot] == (-1 if n is None else n) and c.lens[slot] == (0 if n is None else n + 1)


def test_a_draft_takes_room_and_its_path_becomes_positions(moves):
    c = cpu_cache()
    assert c.admit([15, 30]) == [0, 1]
    c.begin_draft([5, 40, 7, 9])                            # (free slots have no nodes)
    assert [len(o) for o in c._owned] == [2, 5, 0, 0]
    assert c.accept(torch.zeros(4, 5, dtype=torch.int32), ints(3, 1, 5, 0)) == [3, 1, 0, 0]
    assert moves[0].starts == [15, 30, -1, -1] and moves[0].counts == [3, 1, 5, 0] and moves[0].index is not None
    assert [c.length(s) for s in range(4)] == [18, 31, None, None]
    consistent(c)
    c.begin_step()                                           # the pages are there already
    assert [len(o) for o in c._owned] == [2, 5, 0, 0]
    c.advance()
    consistent(c)
    c.begin_draft([0, 1, 0, 0])
    assert c.accept(torch.zeros(4, 5, dtype=torch.int32), ints(0, 0, 0, 0)) == [0] * 4
    for slot in (0, 1):
        c.release(slot)
    assert c.free_pages == 20
    consistent(c)


def test_what_a_draft_cannot_have_leaves_the_cache_as_it_was(moves):
    c = cpu_cache(pages=5)
    c.admit([30, 30])
    before = state(c)
    for nodes, error, text in (([99, 0, 0, 0], RuntimeError, "128 positions"), ([3, 40, 0, 0], RuntimeError, "full"), ([1, 1], ValueError, "each of the 4"),
                               ([1, -1, 0, 0], ValueError, "each of the 4")):
        with pytest.raises(error, match=text):
            c.begin_draft(nodes)
        assert state(c) == before and c._drafted is None
    with pytest.raises(RuntimeError, match="no draft"):
        c.accept(torch.zeros(4, 3, dtype=torch.int32), ints(0, 0, 0, 0))
    c.begin_draft([2, 2, 0, 0])
    for call in (c.begin_step, lambda: c.begin_draft([1] * 4), lambda: c.fork(0)):
        with pytest.raises(RuntimeError, match="has not had"):
            call()
    for counts in ((3, 0, 0, 0), (-1, 0, 0, 0)):
        with pytest.raises(ValueError, match="cannot be accepted"):
            c.accept(torch.zeros(4, 3, dtype=torch.int32), ints(*counts))
    with pytest.raises(ValueError, match="cannot be accepted"):
        c.accept(torch.zeros(4, 1, dtype=torch.int32), ints(2, 0, 0, 0))
    for path, counts in ((torch.zeros(3, 3, dtype=torch.int32), ints(0, 0, 0, 0)), (torch.zeros(4, dtype=torch.int32), ints(0, 0, 0, 0)), (torch.zeros(4, 3, dtype=torch.int32), ints(0, 0))):
        with pytest.raises(ValueError, match="must be"):
            c.accept(path, counts)
    assert not moves and state(c)[-3:] == before[-3:]
    c.release(0)
    c.admit([3])
    with pytest.raises(ValueError, match="cannot be accepted"):      # another sequence is in the slot now
        c.accept(torch.zeros(4, 3, dtype=torch.int32), ints(1, 1, 0, 0))
    c.forget_draft()
    c.begin_step()
    consistent(c)


@pytest.mark.parametrize("length", [1, 15, 16, 17, 32, 100])
def test_a_fork_shares_full_pages_and_copies_the_last(length, moves):
    c = cpu_cache()
    c.admit([5, length])
    full, rest = divmod(length, 16)
    free = c.free_pages
    assert c.fork(1, 2) == [2, 3]
    assert c.free_pages == free - 2 * (rest > 0)
    for s in (2, 3):
        assert [c._owned[s][e] for e in range(full)] == [c._owned[1][e] for e in range(full)]
        assert c.length(s) == length
    if rest:
        assert len(moves) == 1 and moves[0].starts == [0, 0, 16 * full, 16 * full] and moves[0].counts == [0, 0, rest, rest] and moves[0].sources == [1] * 4 and moves[0].rows == 16
        assert torch.equal(moves[0].table, c.page_table) and len({c._owned[s][full] for s in (1, 2, 3)}) == 3
    else:
        assert not moves
    consistent(c)
    for _ in range(20):                                      # they grow apart
        c.begin_step()
        c.advance()
    pages = [c._owned[s][e] for s in (1, 2, 3) for e in c._owned[s] if e >= full]
    assert len(set(pages)) == len(pages)
    consistent(c)
    for s in (1, 3, 0, 2):                                   # (shared pages stay until the last of them goes)
        c.release(s)
        consistent(c)
    assert c.free_pages == 20


def test_a_fork_that_does_not_fit_leaves_the_cache_as_it_was(moves):
    c = cpu_cache(pages=3)
    c.admit([20])
    before = state(c)
    for call, error, text in ((lambda: c.fork(0, 2), RuntimeError, "full"), (lambda: c.fork(0, 4), RuntimeError, "free slots"), (lambda: c.fork(1), ValueError, "no sequence"),
                              (lambda: c.fork(0, 0), ValueError, "not 0")):
        with pytest.raises(error, match=text):
            call()
        assert state(c) == before and not moves


def test_a_fork_whose_copy_fails_leaves_the_cache_as_it_was():
    c = cpu_cache()
    c.admit([5, 37])
    before = state(c)
    with pytest.raises(RuntimeError, match="no CPU path"):
        c.fork(1, 2)
    after = state(c)
    assert after[0] == before[0] and after[2:] == before[2:] and after[1] == before[1]
    consistent(c)


def test_pages_that_a_window_leaves_go_back_when_the_last_fork_leaves_them(moves):
    c = cpu_cache(sequences=2, pages=6, window=16)
    c.admit([31])
    c.fork(0)
    assert c.free_pages == 3
    for _ in range(2):
        c.begin_step()                                        # position 32 is in another page: 17 to 32 are seen, the first page is neither's any more
        c.advance()
    assert c.free_pages == 2 and [sorted(o) for o in c._owned] == [[1, 2], [1, 2]]
    consistent(c)
    # one leaves a page that the other still has: it is not free for that
    c = cpu_cache(sequences=2, pages=2, window=16)
    c.admit([32])
    c.fork(0)
    before = state(c)
    with pytest.raises(RuntimeError, match="full: 1 pages wanted, 0 of 2 free"):
        c.begin_draft([1, 0])
    assert state(c) == before


def test_drafts_forks_steps_and_releases_in_any_order(moves):
    for seed in range(40):
        r, window = random.Random(seed), (None, 24, 16)[seed % 3]
        c = cpu_cache(sequences=5, pages=24, max_len=90, window=window)
        for _ in range(60):
            live = [s for s in range(5) if c.length(s) is not None]
            what = r.choice(["admit", "release", "fork", "step", "draft", "draft"])
            before = state(c)
            try:
                if what == "admit":
                    c.admit([r.randint(1, 40) for _ in range(r.randint(1, 2))])
                elif what == "release" and live:
                    c.release(r.choice(live))
                elif what == "fork" and live:
                    c.fork(r.choice(live), r.randint(1, 2))
                elif what == "step":
                    c.begin_step()
                    c.advance()
                elif what == "draft":
                    nodes = [r.randint(0, 20) for _ in range(5)]
                    c.begin_draft(nodes)
                    counts = ints(*(r.randint(0, m) for m in nodes))
                    taken = c.accept(torch.zeros(5, 20, dtype=torch.int32), counts)
                    assert taken == [int(n) if c.length(s) is not None else 0 for s, n in enumerate(counts)]
            except RuntimeError:
                assert state(c) == before
            consistent(c)
            for s in range(5):                               # every position that a step sees has a page
                n = c.length(s)
                if n is not None:
                    first = 0 if window is None else max(n + 1 - window, 0)
                    assert all(e in c._owned[s] for e in range(first // 16, (n + 15) // 16))


# ---------------------------------------------------------------------------------------------------------------
# what a step over trees refuses ahead of its first kernel
# ---------------------------------------------------------------------------------------------------------------
def cpu_model(rows=64):
    attn = CausalSelfAttention(128, 2, 64, max_seq_len=rows)
    return types.SimpleNamespace(blocks=[types.SimpleNamespace(attn=attn), types.SimpleNamespace(attn=None)])


@pytest.mark.parametrize("recorded", [False, True])
def test_a_draft_step_refuses_on_the_host(recorded):
    model, c = cpu_model(32), cpu_cache()
    c.admit([5, 28])

    def call(tokens, parents, nodes=None):
        if recorded:
            return core.GraphedDraftStep(model, c, 5)(tokens, parents, nodes)
        return core.draft_step(model, tokens, parents, c, nodes)
    tokens, parents = torch.zeros(4, 5, dtype=torch.long), ints(-1, 0, 0, 1, 1)
    before = state(c)
    for args, error, text in (((tokens, parents), AssertionError, "Rotary buffers too small 32 < 33"), ((tokens, parents, [5, 6, 0, 0]), ValueError, "nodes must be 0 to 5"),
                              ((tokens, parents, [5, 1]), ValueError, "nodes must be"), ((tokens[:3], parents, [1] * 3), AssertionError, "token batch"),
                              ((tokens, parents.long(), [1] * 4), ValueError, "parents must be int32"), ((tokens, parents[:4], [1] * 4), ValueError, "parents must be"),
                              ((tokens[:, :4], parents[:4], [1] * 4), ValueError if recorded else RuntimeError, "recording is of trees of 5" if recorded else "no CPU path")):
        with pytest.raises(error, match=text):
            call(*args)
        assert state(c)[-3:] == before[-3:] and c._drafted is None
    c.begin_step()                                           # and the cache goes on


def test_other_caches_windows_and_sizes_of_a_draft_step():
    model, c = cpu_model(), cpu_cache()
    tokens, parents = torch.zeros(4, 1, dtype=torch.long), ints(-1)
    from daisy_amd import KVCache
    with pytest.raises(AssertionError, match="paged cache"):
        core.draft_step(model, tokens, parents, KVCache(2, 4, 2, 8, 64, "cpu", torch.bfloat16))
    with pytest.raises(ValueError, match="window must be positive"):
        core.draft_step(model, tokens, parents, c, window=0)
    with pytest.raises(ValueError, match="1 to 256 nodes"):
        core.draft_step(model, torch.zeros(4, 257, dtype=torch.long), torch.zeros(257, dtype=torch.int32), c)
    with pytest.raises(ValueError, match="1 to 256 nodes"):
        core.GraphedDraftStep(model, c, 0)
    model.blocks[0].attn = object()
    with pytest.raises(ValueError, match="take its pages"):
        core.draft_step(model, tokens, parents, c)
