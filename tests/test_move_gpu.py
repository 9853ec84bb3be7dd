"""``ops.paged_move`` against copies row by row: bits, not numbers, so all of it is compared exactly."""
import random

import pytest
import torch

from daisy_amd import _lib, ops
from test_paged_gpu import BF16, DEV, F16, gen, randn
from test_tree_gpu import ints

pytestmark = pytest.mark.gpu


def cache(L, seqs, width, H, page, D, dtype, g):
    order = torch.randperm(seqs * width + 3, generator=g, device=DEV)[:seqs * width]
    k, v = (randn(g, L, seqs * width + 3, H, page, D, dtype=dtype) for _ in range(2))
    return k, v, order.view(seqs, width).int()


def moved(pages, table, starts, counts, index, sources):
    """A copy of the pages with the rows moved, read ahead of all writes."""
    out, page = pages.clone(), pages.size(3)
    t = table.tolist()
    for b, (start, count) in enumerate(zip(starts, counts)):
        for i in range(count if start >= 0 else 0):
            at, to, seq = start + (index[b][i] if index else i), start + i, sources[b] if sources else b
            out[:, t[b][to // page], :, to % page] = pages[:, t[seq][at // page], :, at % page]
    return out


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("L,H,D,page,M", [(1, 1, 64, 16, 1), (3, 2, 128, 16, 5), (2, 5, 256, 48, 17), (4, 12, 128, 64, 64), (2, 3, 64, 32, 65), (1, 2, 128, 16, 256)])
def test_paths_close_up_in_place(dtype, L, H, D, page, M):
    print(f"move L{L} H{H} D{D} page {page} M{M} {dtype}", flush=True)
    g, rng = gen(M), random.Random(M)
    B = 7
    k, v, table = cache(L, B, -(-700 // page), H, page, D, dtype, g)
    starts = [0, 1, page - 1, page, -1, 300, rng.randrange(300)]
    counts = [M, 0, rng.randint(1, M), 1, M, -5, M]
    index = [sorted(rng.sample(range(2 * M), M)) for _ in range(B)]
    index[0] = list(range(M))      # nothing to do
    index[6] = [1 + i for i in range(M)]      # every row onto the one ahead of it
    want = [moved(x, table, starts, [max(c, 0) for c in counts], index, None) for x in (k, v)]
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.paged_move(k, v, table, ints(starts), ints(counts), index=ints(index), status=status)
    assert status.item() == 0 and torch.equal(k, want[0]) and torch.equal(v, want[1])


@pytest.mark.parametrize("L,H,D,page,rows", [(1, 1, 64, 16, 15), (3, 4, 128, 64, 63), (2, 2, 256, 48, 200)])
def test_forks_get_rows_of_their_own(L, H, D, page, rows):
    g, rng = gen(rows), random.Random(rows)
    B = 9
    k, v, table = cache(L, B, -(-500 // page), H, page, D, BF16, g)
    sources = [0, 0, 0, 0, 1, 1, 2, 2, 0]      # sequences 3 to 8 from 0 to 2
    counts = [0, 0, 0] + [rng.randint(1, rows) for _ in range(5)] + [rows]
    starts = [0, 0, 0] + [page * rng.randrange(200 // page) for _ in range(6)]
    want = [moved(x, table, starts, counts, None, sources) for x in (k, v)]
    ops.paged_move(k, v, table, ints(starts), ints([c + 1000 if i == 8 else c for i, c in enumerate(counts)]), rows=rows, sources=ints(sources))      # (no more than `rows`)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_an_index_into_another_sequence_one_layer_and_strides():
    g = gen(1)
    k, v, table = cache(1, 3, 5, 2, 16, 64, F16, g)
    both = torch.stack((k[0], v[0]), 1)      # the pages of k and v beside each other
    starts, counts, index, sources = [2, 30, 7], [3, 2, 0], [[0, 5, 40], [20, 21, 0], [0, 0, 0]], [1, 2, 2]
    index[0] = [0, 5, 40]
    want = [moved(x, table, starts, counts, index, sources)[0] for x in (k, v)]
    wide = torch.full((3, 9), -1, dtype=torch.int32, device=DEV)
    wide[:, 3:8] = table
    longer = torch.full((3, 6), -1, dtype=torch.int32, device=DEV)
    longer[:, :3] = ints(index)
    ops.paged_move(both[:, 0], both[:, 1], wide[:, 3:8], ints(starts), ints(counts), index=longer, sources=ints(sources))
    assert torch.equal(both[:, 0], want[0]) and torch.equal(both[:, 1], want[1])
    layers = torch.empty(2, 2, *k.shape[1:], dtype=F16, device=DEV)      # of k and v in turn
    layers[:, 0], layers[:, 1] = k[0], v[0]
    ops.paged_move(layers[:, 0], layers[:, 1], table, ints(starts), ints(counts), index=ints(index), sources=ints(sources))
    for i in range(2):
        assert torch.equal(layers[i, 0], want[0]) and torch.equal(layers[i, 1], want[1])


def test_what_leads_nowhere_stays_and_says_so():
    g = gen(2)
    k, v, table = cache(2, 6, 4, 2, 16, 64, BF16, g)
    before = k.clone(), v.clone()
    good = table.clone()
    table[1, 1] = -1
    table[2, 2] = 10 ** 6
    starts, counts = [0, 10, 30, 60, 5, 2 ** 31 - 3], [3, 8, 4, 4, 3, 3]
    index = [[0, 2, 1], [1, 2, 3, 4, 5, 6, 7, 9], [3, 4, 5, 6], [1, 2, 3, 4], [1, 2, 4], [0, 5, 2 ** 31 - 1]]      # out of order; over a page that is none; to one; past the table; fine; far out
    width = max(map(len, index))
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.paged_move(k, v, table, ints(starts), ints(counts), index=ints([r + [0] * (width - len(r)) for r in index]), status=status)
    assert status.item() == _lib.STATUS_INDEX_OUT_OF_ORDER | _lib.STATUS_PAGE_OUT_OF_RANGE | _lib.STATUS_LENGTH_PAST_PAGES
    # rows that are there on both sides
    for x, old in zip((k, v), before):
        want = old.clone()
        for b, rows in ((1, [i for i in range(8) if (10 + i) // 16 != 1 and (10 + index[1][i]) // 16 != 1]), (2, [i for i in range(4) if (30 + i) // 16 != 2 and (30 + index[2][i]) // 16 != 2]),
                        (3, [i for i in range(4) if 60 + index[3][i] < 64]), (4, [0, 1, 2])):
            for i in rows:
                at, to = starts[b] + index[b][i], starts[b] + i
                want[:, good[b, to // 16], :, to % 16] = old[:, good[b, at // 16], :, at % 16]
        assert torch.equal(x, want)
    with pytest.raises(RuntimeError, match="past what the page table"):
        ops.raise_for_status(status)
    with pytest.raises(RuntimeError, match="does not rise"):
        ops.raise_for_status(ints([_lib.STATUS_INDEX_OUT_OF_ORDER]))
    status.zero_()
    ops.paged_move(k, v, good, ints([0, 0]), ints([2, 2]), rows=2, sources=ints([7, -1]), status=status)
    assert status.item() == _lib.STATUS_LENGTH_PAST_PAGES


def test_replays_and_streams():
    g = gen(3)
    k, v, table = cache(2, 3, 5, 2, 16, 128, BF16, g)
    starts, counts, index = ints([3, 20, 40]), ints([3, 1, 4]), ints([[1, 3, 8, 9]] * 3)
    mirror = [k.clone(), v.clone()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.paged_move(k, v, table, starts, counts, index=index)
    torch.cuda.current_stream().wait_stream(side)
    mirror = [moved(x, table, starts.tolist(), counts.tolist(), index.tolist(), None) for x in mirror]
    assert torch.equal(k, mirror[0]) and torch.equal(v, mirror[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_move(k, v, table, starts, counts, index=index)
    for n in range(4):
        starts.copy_(ints([n, 30 - n, 50]))
        counts.copy_(ints([n, 4, 2]))
        index.copy_(ints([[n, n + 1, n + 2, n + 6]] * 3))
        graph.replay()
        torch.cuda.synchronize()
        mirror = [moved(x, table, starts.tolist(), counts.tolist(), index.tolist(), None) for x in mirror]
        assert torch.equal(k, mirror[0]) and torch.equal(v, mirror[1]), n


def test_more_rows_than_a_grid_has_workgroups_for():
    rows, page = 16 * 65535 + 40, 4096
    pages = -(-rows // page)
    g = gen(9)
    k, v = (randn(g, 1, 2 * pages, 1, page, 64, dtype=BF16) for _ in range(2))
    table = torch.randperm(2 * pages, generator=g, device=DEV).int().view(2, pages)
    ops.paged_move(k, v, table, ints([0, 3]), ints([0, rows - 3]), rows=rows, sources=ints([0, 0]))
    for x in (k, v):
        from_rows, to_rows = (x[0, table[i].long(), 0].reshape(-1, 64)[:rows] for i in (0, 1))
        assert torch.equal(from_rows[3:], to_rows[3:]) and not torch.equal(from_rows[:3], to_rows[:3])


def test_offsets_past_32_bits():
    L, H, page, D = 2, 2, 16, 64
    pages = 2 ** 31 // (H * page * D) // L + 9
    store = torch.empty(2, L, pages, H, page, D, dtype=BF16, device=DEV)
    table = ints([[pages - 1, 0, pages - 2]])
    g = gen(4)
    for p in (pages - 1, 0, pages - 2):
        store[:, :, p] = randn(g, 2, L, H, page, D, dtype=BF16)
    want = [torch.stack([x[:, p] for p in (0, pages - 2, pages - 1)], 1) for x in store]
    ops.paged_move(store[0], store[1], table, ints([14]), ints([4]), index=ints([[1, 4, 18, 30]]))
    few = ints([[2, 0, 1]])
    for x, w in zip(store, want):
        w = moved(w, few, [14], [4], [[1, 4, 18, 30]], None)
        assert torch.equal(torch.stack([x[:, p] for p in (0, pages - 2, pages - 1)], 1), w)
