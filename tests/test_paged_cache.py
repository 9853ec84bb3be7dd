"""The paged cache's bookkeeping on the host: slots, pages, the table that the device sees, and what it refuses."""
import pytest
import torch

from daisy_amd import PagedKVCache


def cache(**kw):
    args = dict(L=1, sequences=3, H=1, D=64, pages=6, device="cpu", dtype=torch.bfloat16, page_size=16, max_len=80)
    args.update(kw)
    return PagedKVCache(**args)


def owned(c):
    """Every page is free or in one place of the table; returns the table's pages per slot."""
    table = [[p for p in row if p >= 0] for row in c.page_table.tolist()]
    assert sorted([p for row in table for p in row] + c._free) == list(range(c.pages))
    return table


def test_sequences_come_grow_and_go():
    c = cache()
    assert c.admit([17, 16]) == [0, 1] and [len(r) for r in owned(c)] == [2, 1, 0]
    assert c.positions.tolist() == [17, 16, -1] and c.lens.tolist() == [18, 17, 0] and c.free_pages == 3
    c.begin_step()                       # slot 1's 17th position needs a page, slot 0's does not
    assert [len(r) for r in owned(c)] == [2, 2, 0]
    c.advance()
    assert c.positions.tolist() == [18, 17, -1] and (c.length(0), c.length(1), c.length(2)) == (18, 17, None)
    c.release(0)
    assert [len(r) for r in owned(c)] == [0, 2, 0] and c.positions.tolist() == [-1, 17, -1] and c.lens.tolist() == [0, 18, 0]
    assert c.admit([1]) == [0]
    c.begin_step()
    c.advance(on_device=False)           # a recorded step counts by itself
    assert c.positions.tolist() == [1, 17, -1] and c.length(0) == 2


def test_what_does_not_fit_changes_nothing():
    c = cache()
    assert c.admit([]) == []
    c.admit([33, 33])
    before = c.page_table.clone(), list(c._free)
    with pytest.raises(RuntimeError, match="full"):
        c.admit([1])
    with pytest.raises(RuntimeError, match="free slots"):
        c.admit([1, 1])
    assert torch.equal(c.page_table, before[0]) and c._free == before[1] and c.length(2) is None
    for _ in range(15):
        c.begin_step()
        c.advance()
    with pytest.raises(RuntimeError, match="full"):
        c.begin_step()
    assert c.length(0) == 48 and torch.equal(c.page_table, before[0])
    c.release(1)
    c.begin_step()
    assert [len(r) for r in owned(c)] == [4, 0, 0]


def test_a_full_pool_with_a_window_of_one_goes_on_when_there_is_room():
    """The only page of a sequence is behind the window as the next one is wanted: given back and taken again."""
    c = cache(pages=1, sequences=2, window=1)
    c.admit([16])
    c.begin_step()
    assert owned(c) == [[0], []] and c.page_table[0].tolist()[:2] == [-1, 0]
    c = cache(pages=2, sequences=2, window=17)
    c.admit([16, 16])
    for _ in range(3):
        with pytest.raises(RuntimeError, match="full"):
            c.begin_step()
        assert [len(r) for r in owned(c)] == [1, 1]
    c.release(1)
    c.begin_step()
    assert c.page_table[0].tolist()[:3] == [c.page_table[0, 0].item(), c.page_table[0, 1].item(), -1] and [len(r) for r in owned(c)] == [2, 0]


def test_lengths_end_where_the_table_does():
    c = cache(pages=20)
    with pytest.raises(ValueError, match="80 positions"):
        c.admit([81])
    with pytest.raises(ValueError, match="positions"):
        c.admit([0])
    c.admit([80])
    with pytest.raises(RuntimeError, match="reached 80"):
        c.begin_step()
    with pytest.raises(ValueError, match="no sequence"):
        c.release(1)


@pytest.mark.parametrize("window", [1, 15, 16, 17, 32, 40])
def test_pages_behind_a_window_go_back(window):
    c = cache(pages=8, sequences=2, max_len=400, window=window)
    c.admit([50, 3])
    for _ in range(300):
        c.begin_step()
        owned(c)
        for slot, n in ((0, c.length(0)), (1, c.length(1))):
            held = {e for e, p in enumerate(c.page_table[slot].tolist()) if p >= 0}
            seen = set(range(max(0, n + 1 - window) // 16, n // 16 + 1))
            assert seen <= held, "every position that the step sees has its page"
            assert len(held) <= len(seen) + max(4, 1 + 50 // 16), "and not many more"
        c.advance()


def test_refused_arguments():
    for error, kw in [(ValueError, dict(page_size=8)), (ValueError, dict(page_size=0)), (ValueError, dict(page_size=24)), (TypeError, dict(dtype=torch.float32)), (ValueError, dict(pages=0)),
                      (ValueError, dict(window=0)), (ValueError, dict(sequences=0))]:
        with pytest.raises(error):
            cache(**kw)


def test_handles_are_views():
    c = cache(L=2)
    ctx = c.context(1)
    assert ctx.k_pages.data_ptr() == c.k[1].data_ptr() and ctx.positions is c.positions and ctx.lens is c.lens and ctx.rows is None
    pos, rows = torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    ctx = c.context(0, pos, rows)
    assert ctx.positions is pos and ctx.rows is rows and ctx.lens is None and ctx.page_table is c.page_table
