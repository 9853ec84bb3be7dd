"""Trees of drafted tokens over a paged cache against their definitions: ``ops.draft_tree`` exactly, ``ops.paged_tree_attention`` in 64 bits, and ``ops.paged_append`` with
``slots``.

Tolerances.  A rounding to a type is off by at most half a step, ``E = finfo.eps / 2`` of the value.  The output is rounded once (E |o|); a probability is held in
two parts, whose second is off by E of the first one's rounding, E^2 <= 2^-16 of p; the scores' sums in fp32 move the exponents by less than 1e-4 (64 to 256 products of values of a few
units, times 0.12 log2 e), which numerator and denominator both feel: 3e-4 of A := sum p |v| / sum p.  Below fp16's normal range a step is 2^-24, half of it 2^-25."""
import math
import random

import pytest
import torch

from daisy_amd import _lib, ops
from test_paged_gpu import BF16, DEV, F16, gen, half_step, randn

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def random_parents(T, rng, shape):
    if shape == "chain":
        return [i - 1 for i in range(T)]
    if shape == "star":
        return [-1] + [0] * (T - 1)
    if shape == "forest":      # several roots, parents that are none
        return [rng.choice([-1, -7, i, i + 3, T + 9, 2 ** 31 - 1, -2 ** 31] + [rng.randrange(i)] * 6) if i else rng.choice([-1, 0, 5]) for i in range(T)]
    return [-1] + [rng.randrange(max(0, i - 6), i) for i in range(1, T)]


def lines_of(parents):
    out = []
    for i, u in enumerate(parents):
        out.append([i] + (out[u] if 0 <= u < i else []))
    return out


def masks_of(parents, W):
    """Bits as the kernel's words."""
    out = []
    for line in lines_of(parents):
        words = [sum(1 << j % 32 for j in line if j // 32 == w) for w in range(W)]
        out.append([w - 2 ** 32 if w >= 2 ** 31 else w for w in words])
    return out


@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 63, 64, 65, 96, 127, 128, 129, 200, 255, 256])
@pytest.mark.parametrize("shape", ["chain", "random", "star", "forest"])
def test_what_nodes_see_and_where_they_lie(T, shape):
    print(f"draft tree T{T} {shape}", flush=True)
    rng = random.Random(T)
    B, W = 5, (T + 31) // 32
    parents = [random_parents(T, rng, shape) for _ in range(B)]
    lens = [0, 7, -1, 100000, 31]
    for nodes in (None, [T, 0, T, rng.randint(0, T), T + 5]):
        tree = ops.draft_tree(ints(parents), ints(lens), nodes=None if nodes is None else ints(nodes))
        assert tree.mask.shape == (B, T, W) and tree.rows.tolist() == [b for b in range(B) for _ in range(T)]
        for b in range(B):
            n = 0 if lens[b] < 0 else T if nodes is None else min(nodes[b], T)
            lines, masks = lines_of(parents[b]), masks_of(parents[b], W)
            at = slice(b * T, (b + 1) * T)
            assert tree.mask[b].tolist() == [masks[i] if i < n else [0] * W for i in range(T)], b
            assert tree.positions[at].tolist() == [lens[b] + len(lines[i]) - 1 if i < n else -1 for i in range(T)]
            assert tree.slots[at].tolist() == [lens[b] + i if i < n else -1 for i in range(T)]
    one = ops.draft_tree(ints(parents[0]), ints(lens))
    each = ops.draft_tree(ints([parents[0]] * B), ints(lens))
    assert all(torch.equal(x, y) for x, y in zip(one, each)), "one tree for all"


def cache_of(extents, H, page, D, dtype, g, junk=float("nan"), extra=2):
    """Shuffled pages of random values for the places [lo, hi) of each sequence; ``junk`` in all other rows, -1 in all other entries.  Returns k, v pages, table, and
    per sequence its places' keys and values, of places before lo zeros."""
    width = max([1] + [-(-hi // page) for _, hi in extents]) + 1
    needed = [range(lo // page, -(-hi // page)) if hi > lo else range(0) for lo, hi in extents]
    total = sum(map(len, needed))
    order = torch.randperm(total + extra, generator=g, device=DEV).tolist()
    k = torch.full((total + extra, H, page, D), junk, device=DEV, dtype=dtype)
    v = torch.full_like(k, junk)
    table = torch.full((len(extents), width), -1, dtype=torch.int32)
    rows, at = [], 0
    for s, (lo, hi) in enumerate(extents):
        kk, vv = randn(g, max(hi, 0), H, D, dtype=dtype), randn(g, max(hi, 0), H, D, dtype=dtype)
        for j in needed[s]:
            table[s, j] = order[at]
            a, b = max(lo, j * page), min(hi, (j + 1) * page)
            k[order[at], :, a - j * page:b - j * page] = kk[a:b].transpose(0, 1)
            v[order[at], :, a - j * page:b - j * page] = vv[a:b].transpose(0, 1)
            at += 1
        rows.append((kk, vv))
    return k, v, table.to(DEV), rows


def seen_by(n, count, masks, window):
    """bool [count, n + count]: which places each node sees."""
    seen = torch.zeros(count, n + count, dtype=torch.bool)
    for i in range(count):
        row = list(range(n)) + [n + j for j in range(count) if j == i or masks[i][j // 32] >> j % 32 & 1]
        seen[i, row[-window:] if window else row] = True
    return seen


def exact(q, rows, lens, nodes, masks, scale, window=None):
    """(o, sum p |v| / sum p) in 64 bits."""
    B, T, Hq, D = q.shape
    o, a = (torch.zeros(B, T, Hq, D, device=DEV, dtype=torch.float64) for _ in range(2))
    for b in range(B):
        n, count = lens[b], nodes[b]
        if n < 0 or count == 0:
            continue
        k, v = (x.double() for x in rows[b])
        H = k.shape[1]
        away = ~seen_by(n, count, masks[b], window).to(DEV)
        for h in range(Hq):
            kh, vh = k[:, h // (Hq // H)], v[:, h // (Hq // H)]
            s = (q[b, :count, h].double() @ kh.T.contiguous() * scale).masked_fill(away, -math.inf)
            p = torch.softmax(s, -1)
            o[b, :count, h], a[b, :count, h] = p @ vh, p @ vh.abs()
    return o, a


def check(o, q, rows, lens, nodes, masks, scale, what, window=None):
    want, a = exact(q, rows, lens, nodes, masks, scale, window)
    E = half_step(o.dtype)
    tol = E * want.abs() + (3e-4 + 2.0 ** -16) * a + 2.0 ** -25
    err = (o.double() - want).abs()
    assert torch.isfinite(o).all(), what
    assert bool((err <= tol).all()), f"{what}: error {err.max().item():.3e}, {(err / tol).max().item():.2f} of what it may be, at {(err / tol).argmax().item()}"
    for b in range(len(lens)):
        n = 0 if lens[b] < 0 else nodes[b]
        assert bool((o[b, n:] == 0).all()), f"{what}: rows of nodes that there are not"


LENS = [0, 1, 15, 16, 31, 32, 33, 40, 63, 64, -1, 65, 100, 127, 200]


def trees(T, B, rng, shape="random"):
    parents = [random_parents(T, rng, shape) for _ in range(B)]
    return parents, [masks_of(p, (T + 31) // 32) for p in parents]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,H,G,T,page", [(64, 2, 1, 1, 16), (64, 1, 3, 5, 48), (128, 2, 1, 8, 16), (128, 3, 2, 8, 32), (128, 1, 1, 17, 64), (128, 2, 4, 8, 16), (128, 1, 8, 33, 32),
                                          (64, 2, 1, 33, 16), (64, 1, 4, 40, 64), (256, 2, 1, 5, 16), (256, 1, 2, 12, 96), (256, 1, 8, 9, 32), (64, 1, 1, 100, 256), (128, 1, 1, 256, 32),
                                          (128, 2, 16, 3, 16), (128, 1, 8, 12, 48), (64, 2, 4, 24, 16), (256, 1, 4, 70, 16)])
def test_attention_over_every_edge_of_blocks_tiles_and_pages(dtype, D, H, G, T, page):
    print(f"tree attention {dtype} D{D} H{H} G{G} T{T} page {page}", flush=True)
    g, rng = gen(D + H + G + T + page), random.Random(T)
    B = len(LENS)
    nodes = [T, T, 1, T] + [rng.randint(0, T) for _ in range(B - 4)]
    _, masks = trees(T, B, rng)
    k, v, table, rows = cache_of([(0, max(n, 0) + (t if n >= 0 else 0)) for n, t in zip(LENS, nodes)], H, page, D, dtype, g)
    q = randn(g, B, T, H * G, D, dtype=dtype)
    o = ops.paged_tree_attention(q, k, v, table, ints(LENS), ints(masks), nodes=ints(nodes), scale=0.12)
    check(o, q, rows, LENS, nodes, masks, 0.12, "all positions")
    assert torch.equal(o, ops.paged_tree_attention(q, k, v, table, ints(LENS), ints(masks), nodes=ints(nodes), scale=0.12)), "twice"
    if dtype == F16:
        wide = ops.paged_tree_attention(q, k, v, table, ints(LENS), ints(masks), nodes=ints(nodes), scale=0.12, out=torch.empty(q.shape, dtype=BF16, device=DEV))
        check(wide, q, rows, LENS, nodes, masks, 0.12, "bf16 results")


@pytest.mark.parametrize("window", [1, 2, 3, 7, 16, 31, 32, 33, 64, 100, 1000])
@pytest.mark.parametrize("D,G,T,page,dtype,shape", [(128, 1, 12, 16, BF16, "random"), (64, 2, 33, 64, F16, "chain"), (128, 4, 40, 32, BF16, "random"), (256, 1, 5, 48, BF16, "chain")])
def test_windows_end_at_each_node_and_see_no_page_that_was_given_back(window, D, G, T, page, dtype, shape):
    print(f"tree attention, window {window}, D{D} T{T} page {page}", flush=True)
    g, rng = gen(window + D), random.Random(window)
    lens = [0, 1, 5, 31, 32, 33, 64, 97, 160, 161, 300, 1023]
    nodes = [T] * 6 + [rng.randint(1, T) for _ in range(6)]
    _, masks = trees(T, len(lens), rng, shape)
    k, v, table, rows = cache_of([(max(0, n + 1 - window), n + t) for n, t in zip(lens, nodes)], 2, page, D, dtype, g)
    q = randn(g, len(lens), T, 2 * G, D, dtype=dtype)
    o = ops.paged_tree_attention(q, k, v, table, ints(lens), ints(masks), nodes=ints(nodes), window=window)
    check(o, q, rows, lens, nodes, masks, ops.ATTN_SCALE, f"window {window}", window)


def test_any_set_of_nodes_and_always_itself():
    """Masks that are no trees: bits of nodes behind, of nodes that there are not, none at all."""
    g, rng = gen(3), random.Random(3)
    T, lens, nodes = 45, [0, 10, 64, 200, 0], [45, 40, 33, 1, 2]
    masks = [[[rng.getrandbits(32) - 2 ** 31 if rng.random() < 0.7 else 0 for _ in range(2)] for _ in range(T)] for _ in lens]
    k, v, table, rows = cache_of([(0, n + t) for n, t in zip(lens, nodes)], 2, 16, 128, BF16, g)
    q = randn(g, len(lens), T, 4, 128, dtype=BF16)
    o = ops.paged_tree_attention(q, k, v, table, ints(lens), ints(masks), nodes=ints(nodes))
    check(o, q, rows, lens, nodes, masks, ops.ATTN_SCALE, "sets")
    for window in (1, 4, 30, 70):
        k, v, table, rows = cache_of([(max(0, n + 1 - window), n + t) for n, t in zip(lens, nodes)], 2, 16, 128, BF16, g)
        o = ops.paged_tree_attention(q, k, v, table, ints(lens), ints(masks), nodes=ints(nodes), window=window)
        check(o, q, rows, lens, nodes, masks, ops.ATTN_SCALE, f"sets, window {window}", window)


@pytest.mark.parametrize("lens,H,G,T", [([5000], 1, 1, 4), ([5000], 1, 1, 64), ([1, 20001, 3], 2, 1, 20), ([9000] + [7] * 70, 1, 4, 8), ([33] * 200, 3, 1, 6), ([4096] * 3, 4, 8, 16),
                                        ([0], 1, 1, 1), ([-1] * 100 + [700] + [-1] * 100, 2, 2, 10), ([50] * 300 + [4000] + [11] * 100, 2, 1, 3), ([17] * 4200 + [900], 1, 1, 2),
                                        ([30000], 2, 8, 32), ([17] * 300 + [900], 1, 8, 20), ([17] * 300 + [900, -1], 1, 2, 20), ([6000, 5, 0], 1, 8, 10)])
def test_work_is_split_over_what_is_there(lens, H, G, T):
    """One long row, long ones among many short, more sequences than a wavefront or a workgroup has lanes, free slots all around."""
    print(f"tree attention of {len(lens)} sequences, the longest {max(lens)}, H{H} G{G} T{T}", flush=True)
    g, rng = gen(len(lens) + T), random.Random(len(lens))
    _, masks = trees(T, len(lens), rng)
    nodes = [T] * len(lens)
    k, v, table, rows = cache_of([(0, n + T if n >= 0 else 0) for n in lens], H, 64, 64, BF16, g)
    q = randn(g, len(lens), T, H * G, 64, dtype=BF16)
    o = ops.paged_tree_attention(q, k, v, table, ints(lens), ints(masks))
    some = sorted({0, len(lens) // 2, len(lens) - 1, *[b for b, n in enumerate(lens) if n > 500][:3]})
    check(o[some], q[some], [rows[b] for b in some], [lens[b] for b in some], [nodes[b] for b in some], [masks[b] for b in some], ops.ATTN_SCALE, "split")
    for b, n in enumerate(lens):
        assert bool((o[b] == 0).all()) == (n < 0)


@pytest.mark.parametrize("D,T,G,length", [(128, 8, 1, 6000), (128, 30, 1, 6000), (128, 16, 4, 6000), (64, 64, 1, 3000), (256, 8, 1, 2500), (256, 20, 2, 2500), (128, 64, 8, 700)])
def test_probabilities_are_not_rounded(D, T, G, length):
    """Values of one sign: a product with probabilities rounded once to bf16 would be off by up to 2^-9 of A; with two parts the output's rounding is what is left."""
    g, rng = gen(D + T), random.Random(T)
    _, masks = trees(T, 1, rng)
    k, v, table, rows = cache_of([(0, length + T)], 1, 32, D, BF16, g)
    v.abs_()
    rows = [(rows[0][0], rows[0][1].abs())]
    q = randn(g, 1, T, G, D, dtype=BF16)
    o = ops.paged_tree_attention(q, k, v, table, ints([length]), ints(masks))
    check(o, q, rows, [length], [T], masks, ops.ATTN_SCALE, "one sign")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("odd", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("T,window", [(20, None), (70, None), (20, 25)])
def test_a_value_that_is_not_finite_reaches_those_who_see_it_alone(dtype, odd, T, window):
    g, rng = gen(5), random.Random(5)
    lens = [0, 37, 90]
    _, masks = trees(T, 3, rng)
    k, v, table, rows = cache_of([(0, n + T) for n in lens], 2, 16, 128, dtype, g, junk=0.0)
    q = randn(g, 3, T, 2, 128, dtype=dtype)
    places = [(b, n + i, h, c) for b, n in enumerate(lens) for i, h, c in ((0, 0, 3), (3, 1, 127), (T // 2, 0, 64), (T - 1, 1, 0))]
    places.append((2, 70, 0, 9))      # of a context: seen by all, or, in a window, by some
    for b, t, h, c in places:
        v[table[b, t // 16], h, t % 16, c] = odd
    o = ops.paged_tree_attention(q, k, v, table, ints(lens), ints(masks), window=window)
    touched = torch.zeros(3, T, 2, 128, dtype=torch.bool)
    for b, t, h, c in places:
        touched[b, seen_by(lens[b], T, masks[b], window)[:, t], h, c] = True
    assert torch.equal(torch.isfinite(o).cpu(), ~touched)
    want, a = exact(q, rows, lens, [T] * 3, masks, ops.ATTN_SCALE, window)
    tol = half_step(dtype) * want.abs() + (3e-4 + 2.0 ** -16) * a + 2.0 ** -25
    assert bool(((o.double() - want).abs() <= tol)[~touched.to(DEV)].all())


def test_keys_that_are_not_finite_and_scores_of_the_lowest():
    """A key that scores NaN spoils who sees it alone; one that scores -inf weighs nothing."""
    g, rng = gen(6), random.Random(6)
    T, n = 20, 40
    parents, masks = trees(T, 1, rng)
    k, v, table, rows = cache_of([(0, n + T)], 1, 16, 64, F16, g)
    q = randn(g, 1, T, 1, 64, dtype=F16).abs() + 0.01
    plain = ops.paged_tree_attention(q, k, v, table, ints([n]), ints(masks))
    at = lambda t: (table[0, t // 16], 0, t % 16)      # noqa: E731
    k[at(n + 4)] = float("nan")
    o = ops.paged_tree_attention(q, k, v, table, ints([n]), ints(masks))
    sees = seen_by(n, T, masks[0], None)[:, n + 4]
    assert torch.equal(torch.isnan(o[0, :, 0]).all(-1).cpu(), sees) and torch.equal(o[0, ~sees], plain[0, ~sees])
    k[at(n + 4)] = -float("inf")
    rows[0][0][n + 4] = -60000.0
    o = ops.paged_tree_attention(q, k, v, table, ints([n]), ints(masks))
    check(o, q, rows, [n], [T], masks, ops.ATTN_SCALE, "-inf")


def test_strides_outputs_and_workspaces():
    g, rng = gen(8), random.Random(8)
    T, H, D, lens = 9, 2, 128, [70, -1, 300]
    _, masks = trees(T, 3, rng)
    k, v, table, rows = cache_of([(0, n + T if n >= 0 else 0) for n in lens], H, 32, D, BF16, g)
    both = torch.stack((k, v), 1)      # pages of k and v beside each other
    wide = torch.full((3, 40), -1, dtype=torch.int32, device=DEV)
    wide[:, 5:5 + table.size(1)] = table
    mask = torch.zeros(3, T + 2, 4, dtype=torch.int32, device=DEV)
    mask[:, 1:1 + T, 2:3] = ints(masks)
    qkv = randn(g, T, 3, 3 * H, D, dtype=BF16).transpose(0, 1)      # nodes outermost, queries a part of the projection
    q = qkv[:, :, H:2 * H]
    out = torch.full((3, T, H + 1, D), 7.0, dtype=BF16, device=DEV)
    need = ops.paged_tree_attention_workspace_bytes(3, T, H, H, D, table.size(1), 32)
    ws = torch.full((need,), 255, dtype=torch.uint8, device=DEV)
    o = ops.paged_tree_attention(q, both[:, 0], both[:, 1], wide[:, 5:5 + table.size(1)], ints(lens), mask[:, 1:1 + T, 2:3], out=out[:, :, 1:], workspace=ws)
    assert o.data_ptr() == out[:, :, 1:].data_ptr() and bool((out[:, :, 0] == 7).all())
    check(o, q, rows, lens, [T] * 3, masks, ops.ATTN_SCALE, "strides")
    want = o.clone()
    inplace = q.contiguous()
    assert torch.equal(ops.paged_tree_attention(inplace, k, v, table, ints(lens), ints(masks), out=inplace), want), "in the queries' place"


def test_bad_pages_and_lengths_spoil_their_own_sequence():
    """What only the device sees: bounds checks of the kernel's own turn it into NaN and a status bit."""
    g, rng = gen(9), random.Random(9)
    T = 6
    lens = [40, 40, 40, 40, 2 ** 31 - 1]
    _, masks = trees(T, 5, rng)
    k, v, table, rows = cache_of([(0, 46)] * 5, 2, 16, 64, BF16, g)
    table[1, 1], table[2, 2] = 10 ** 6, -1
    lens[3] = table.size(1) * 16 - T + 1
    q = randn(g, 5, T, 2, 64, dtype=BF16)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    o = ops.paged_tree_attention(q, k, v, table, ints(lens), ints(masks), status=status)
    assert torch.isnan(o[1:]).all()
    check(o[:1], q[:1], rows[:1], lens[:1], [T], masks[:1], ops.ATTN_SCALE, "its neighbour")
    assert status.item() == _lib.STATUS_PAGE_OUT_OF_RANGE | _lib.STATUS_LENGTH_PAST_PAGES
    with pytest.raises(RuntimeError, match="past what the page table"):
        ops.raise_for_status(status)


def test_streams_and_replays():
    """On another stream, and recorded: replays follow lengths, nodes, masks and the table, with eager work between them."""
    g, rng = gen(10), random.Random(10)
    T, H, D = 11, 2, 128
    k, v, table, rows = cache_of([(0, 500)] * 3, H, 16, D, BF16, g)
    q = randn(g, 3, T, H, D, dtype=BF16)
    parents, lens, nodes = ints([random_parents(T, rng, "random") for _ in range(3)]), ints([100, 20, 3]), ints([T, 4, T])
    side = torch.cuda.Stream()

    def run():
        tree = ops.draft_tree(parents, lens, nodes=nodes)
        return ops.paged_tree_attention(q, k, v, table, lens, tree.mask, nodes=nodes)

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, run())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = run()
    for n in range(4):
        lens.copy_(ints([100 + 77 * n, n - 1, 450]))
        nodes.copy_(ints([T - n, T, n]))
        parents.copy_(ints([random_parents(T, rng, "random") for _ in range(3)]))
        graph.replay()
        torch.cuda.synchronize()
        want = run()
        assert torch.equal(recorded, want), n


def test_offsets_past_32_bits():
    """Pages more than 2^31 elements from the first."""
    g, rng = gen(11), random.Random(11)
    T, H, page, D = 5, 2, 16, 64
    pages = 2 ** 31 // (H * page * D) + 9
    store = torch.empty(pages, H, page, D, dtype=BF16, device=DEV)
    k = v = store
    n = 30
    _, masks = trees(T, 1, rng)
    few_k, _, few, rows = cache_of([(0, n + T)], H, page, D, BF16, g)
    table = few.clone()
    for j in range(3):
        table[0, j] = pages - 1 - 2 * j
        store[pages - 1 - 2 * j] = few_k[few[0, j]]
    q = randn(g, 1, T, H, D, dtype=BF16)
    o = ops.paged_tree_attention(q, k, v, table, ints([n]), ints(masks))
    check(o, q, [(rows[0][0], rows[0][0])], [n], [T], masks, ops.ATTN_SCALE, "far")


@pytest.mark.parametrize("N,T", [(3, 7), (1, 40)])
def test_append_puts_nodes_behind_one_another_and_rotates_them_by_their_lines(N, T):
    """``slots``: the same rows as an append at each node's position, in another place, bit for bit."""
    g, rng = gen(12), random.Random(12)
    H, D, page = 2, 64, 16
    lens = [20, 5, -1][:N] if N > 1 else [33]
    parents = [random_parents(T, rng, "random") for _ in range(N)]
    tree = ops.draft_tree(ints(parents), ints(lens))
    table = torch.arange(N * 6, dtype=torch.int32, device=DEV).view(N, 6)
    theta = torch.outer(torch.arange(200.0), torch.rand(D // 2)).to(DEV)
    cos, sin = theta.cos().contiguous(), theta.sin().contiguous()
    q, k, v = (randn(g, N * T, H, D, dtype=BF16) for _ in range(3))
    pages = [torch.full((N * 6, H, page, D), 3.0, dtype=BF16, device=DEV) for _ in range(2)]
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = ops.paged_append(k, v, *pages, table, tree.positions, rows=tree.rows, q=q, cos=cos, sin=sin, eps=1e-6, slots=tree.slots, status=status)
    assert status.item() == 0
    k_out, v_out = torch.zeros_like(k), torch.zeros_like(v)
    scrap = [torch.empty(N * 6, H, page, D, dtype=BF16, device=DEV) for _ in range(2)]
    want = ops.paged_append(k, v, *scrap, table, tree.positions, rows=tree.rows, q=q, cos=cos, sin=sin, eps=1e-6, k_out=k_out, v_out=v_out)
    assert torch.equal(got, want)
    for x, rows in zip(pages, (k_out, v_out)):
        expect = torch.full((N, 6 * page, H, D), 3.0, dtype=BF16, device=DEV)
        for b, n in enumerate(lens):
            if n >= 0:
                expect[b, n:n + T] = rows[b * T:(b + 1) * T]
        assert torch.equal(x.transpose(1, 2).reshape(N, 6 * page, H, D), expect)
