"""The paged cache's two operators against their definitions in 64 bits: ``ops.paged_append`` and ``ops.paged_attention``.

Tolerances.  A rounding to a type is off by at most half a step, ``E = finfo.eps / 2`` of the value.  Attention: the probabilities are rounded once ahead of
the second product (E of sum p |v| / sum p =: A) and the output once (E |o|); the scores' sums in fp32 move the exponents by less than 1e-4 (128 to 256
products of values of a few units, times 0.12 log2 e), which numerator and denominator both feel: 3e-4 A.  Append: norm, rotation
and mix in fp32 are a dozen roundings of 2^-24 of terms no larger than the sum of the products' magnitudes: 2^-20 of that; the output E |y|, and
half of fp16's smallest step where a value is below its normal range."""
import math

import pytest
import torch

from daisy_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16 = torch.bfloat16, torch.float16


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def make_cache(lens, H, page, D, dtype, g, window=None, extra=2, junk=float("nan")):
    """Pages of random values for sequences of ``lens`` positions, shuffled; ``junk`` in every row that no sequence shows, -1 in every table entry that is
    not needed.  Returns k, v pages, table and, per sequence, its visible positions' keys and values in 64 bits."""
    width = max(1, -(-max(lens + [1]) // page)) + 1
    needed = [range((max(0, n - window) if window else 0) // page, -(-n // page)) for n in lens]
    total = sum(len(r) for r in needed)
    order = torch.randperm(total + extra, generator=g, device=DEV).tolist()
    k = torch.full((total + extra, H, page, D), junk, device=DEV, dtype=dtype)
    v = torch.full_like(k, junk)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    rows, at = [], 0
    for s, n in enumerate(lens):
        lo = max(0, n - window) if window else 0
        kk, vv = randn(g, n - lo, H, D, dtype=dtype), randn(g, n - lo, H, D, dtype=dtype)
        for j in needed[s]:
            p = order[at]
            at += 1
            table[s, j] = p
            a, b = max(lo, j * page), min(n, (j + 1) * page)
            k[p, :, a - j * page:b - j * page] = kk[a - lo:b - lo].transpose(0, 1)
            v[p, :, a - j * page:b - j * page] = vv[a - lo:b - lo].transpose(0, 1)
        rows.append((kk.double(), vv.double()))
    return k, v, table.to(DEV), rows


def attend_exact(q, rows, scale):
    """(o, sum p |v| / sum p) in 64 bits."""
    B, Hq, D = q.shape
    o, a = torch.zeros(B, Hq, D, device=DEV, dtype=torch.float64), torch.zeros(B, Hq, D, device=DEV, dtype=torch.float64)
    for b, (k, v) in enumerate(rows):
        if k.shape[0] == 0:
            continue
        H = k.shape[1]
        for h in range(Hq):
            kh, vh = k[:, h // (Hq // H)], v[:, h // (Hq // H)]
            p = torch.softmax((kh * q[b, h].double()).sum(1) * scale, 0)
            o[b, h], a[b, h] = (p[:, None] * vh).sum(0), (p[:, None] * vh.abs()).sum(0)
    return o, a


def check_attention(o, q, rows, scale, what):
    want, a = attend_exact(q, rows, scale)
    E = half_step(o.dtype)
    err = (o.double() - want).abs()
    tol = (E + 3e-4) * a + E * want.abs() + 1e-7
    assert torch.isfinite(o).all(), what
    assert bool((err <= tol).all()), f"{what}: error {err.max().item():.3e}, {(err / tol).max().item():.2f} of what it may be"


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64, 65, 100, 0, 127, 128, 129, 200]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,H,G,page", [(64, 2, 1, 16), (64, 1, 3, 48), (128, 2, 1, 16), (128, 3, 2, 32), (128, 1, 16, 64), (128, 2, 17, 16), (128, 1, 40, 128),
                                        (256, 2, 1, 16), (256, 1, 8, 96), (64, 5, 4, 256)])
def test_attention_over_every_edge_of_blocks_tiles_and_pages(dtype, D, H, G, page):
    print(f"paged attention {dtype} D{D} H{H} G{G} page {page}", flush=True)
    g = gen(D + H + G + page)
    k, v, table, rows = make_cache(EDGES, H, page, D, dtype, g)
    q = randn(g, len(EDGES), H * G, D, dtype=dtype)
    lens = torch.tensor(EDGES, dtype=torch.int32, device=DEV)
    o = ops.paged_attention(q, k, v, table, lens, scale=0.12)
    check_attention(o, q, rows, 0.12, "all positions")
    assert bool((o[[0, 15]] == 0).all()), "a sequence without positions gives zeros"
    again = ops.paged_attention(q, k, v, table, lens, scale=0.12)
    assert torch.equal(o, again)
    if dtype == F16:
        wide = ops.paged_attention(q, k, v, table, lens, scale=0.12, out=torch.empty(q.shape, dtype=BF16, device=DEV))
        check_attention(wide, q, rows, 0.12, "bf16 results")


@pytest.mark.parametrize("window", [1, 2, 16, 31, 32, 33, 100, 1000])
@pytest.mark.parametrize("D,G,page,dtype", [(128, 1, 16, BF16), (64, 2, 64, F16), (256, 1, 48, BF16)])
def test_windows_see_no_page_that_was_given_back(window, D, G, page, dtype):
    print(f"paged attention, window {window}, D{D} page {page}", flush=True)
    g = gen(window + D)
    lens = [0, 1, 5, 31, 32, 33, 64, 97, 160, 161, 300, 1023]
    k, v, table, rows = make_cache(lens, 2, page, D, dtype, g, window=window)
    q = randn(g, len(lens), 2 * G, D, dtype=dtype)
    o = ops.paged_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=DEV), window=window)
    check_attention(o, q, rows, ops.ATTN_SCALE, f"window {window}")


@pytest.mark.parametrize("lens,H,G", [([5000], 1, 1), ([1, 20001, 3], 2, 1), ([9000] + [7] * 70, 1, 4), ([33] * 200, 3, 1), ([4096] * 3, 4, 8), ([1], 1, 1),
                                      ([0] * 100 + [700] + [0] * 100, 2, 2)])
def test_work_is_split_over_what_is_there(lens, H, G):
    """One long row, long ones among many short, more sequences than a wavefront has lanes, empty ones all around."""
    print(f"paged attention of {len(lens)} sequences, the longest {max(lens)}, H{H} G{G}", flush=True)
    g = gen(len(lens))
    k, v, table, rows = make_cache(lens, H, 32, 128, BF16, g)
    q = randn(g, len(lens), H * G, 128, dtype=BF16)
    o = ops.paged_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=DEV))
    check_attention(o, q, rows, ops.ATTN_SCALE, "split")


@pytest.mark.parametrize("B", [256, 257, 1000, 4096, 4097, 9001])
def test_many_sequences(B):
    print(f"paged attention of {B} sequences", flush=True)
    g = gen(B)
    lens = [(7 * i) % 40 if i % 11 else 0 for i in range(B)]
    lens[B // 2] = 3000
    k, v, table, rows = make_cache(lens, 1, 16, 64, BF16, g)
    q = randn(g, B, 2, 64, dtype=BF16)
    check_attention(ops.paged_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=DEV), scale=0.12), q, rows, 0.12, f"{B} sequences")


@pytest.mark.parametrize("fill", [0, 0x01, 0x7f, 0xff])
def test_what_a_workspace_held_before_means_nothing(fill):
    """One workspace for calls of different shapes, with anything in it."""
    g = gen(17)
    cases = []
    for lens, H, G, D in (([5000, 30, 0], 2, 8, 128), ([100] * 70, 1, 1, 64), ([700, 64, 3], 1, 17, 256)):
        k, v, table, rows = make_cache(lens, H, 32, D, BF16, g)
        q = randn(g, len(lens), H * G, D, dtype=BF16)
        cases.append((q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=DEV)))
    need = max(ops.paged_attention_workspace_bytes(q.shape[0], q.shape[1], k.shape[1], q.shape[2], table.shape[1], 32) for q, k, v, table, _ in cases)
    space = torch.full((need,), fill, dtype=torch.uint8, device=DEV)
    for args in cases + cases:
        assert torch.equal(ops.paged_attention(*args, workspace=space), ops.paged_attention(*args))


def test_every_sequence_empty():
    g = gen(1)
    k, v, table, _ = make_cache([0, 0, 0], 2, 16, 128, BF16, g)
    out = torch.full((3, 2, 128), 7.0, dtype=BF16, device=DEV)
    o = ops.paged_attention(randn(g, 3, 2, 128, dtype=BF16), k, v, table, torch.tensor([0, -5, 0], dtype=torch.int32, device=DEV), out=out)
    assert o is out and bool((o == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("direction", [1, -1])
def test_scores_that_rise_and_fall_by_hundreds(dtype, direction):
    """The reference of the exponentials moves from tile to tile, or stands while everything behind it vanishes."""
    g = gen(3)
    n, D = 700, 128
    k, v, table, _ = make_cache([n], 1, 16, D, dtype, g)
    q = torch.ones(1, 1, D, device=DEV, dtype=dtype)
    ramp = torch.linspace(-1.0, 1.0, n, device=DEV) * direction
    keys = (ramp[:, None] * 20 / 16 + 0.01 * randn(g, n, D)).to(dtype)
    values = randn(g, n, D, dtype=dtype)
    for t in range(n):
        p = int(table[0, t // 16])
        k[p, 0, t % 16], v[p, 0, t % 16] = keys[t], values[t]
    rows = [(keys.double()[:, None], values.double()[:, None])]
    o = ops.paged_attention(q, k, v, table, torch.tensor([n], dtype=torch.int32, device=DEV), scale=1.0)
    # the scores reach 160, sums of 128 products of one sign: their error is up to 128 * 2^-24 * 160 = 1.2e-3 in the exponent
    want, a = attend_exact(q, rows, 1.0)
    E = half_step(dtype)
    err = (o.double() - want).abs()
    assert bool((err <= (E + 3e-3) * a + E * want.abs() + 1e-7).all()), (err / a).max()


def test_many_small_probabilities_beside_a_large_one():
    """A first key far above 20000 others that share a quarter of the weight: none of them may vanish in fp16."""
    g = gen(4)
    n, D = 20000, 64
    k, v, table, _ = make_cache([n], 1, 64, D, F16, g)
    q = torch.zeros(1, 1, D, device=DEV, dtype=F16)
    q[..., 0] = 1
    k.zero_()
    v.zero_()
    k[int(table[0, 0]), 0, 0, 0] = math.log(3.0 * (n - 1))
    seen = torch.zeros_like(v)
    for j in range(-(-n // 64)):
        seen[int(table[0, j]), 0, :min(64, n - 64 * j)] = 1
    seen[int(table[0, 0]), 0, 0] = 0
    v.copy_(seen)
    o = ops.paged_attention(q, k, v, table, torch.tensor([n], dtype=torch.int32, device=DEV), scale=1.0)
    top = math.exp(float(torch.tensor(math.log(3.0 * (n - 1)), dtype=F16)))
    want = (n - 1) / (n - 1 + top)
    # every probability is rounded alike here: half a step of each, and of the output
    assert abs(float(o[0, 0, 0]) - want) <= (2 * half_step(F16) + 1e-4) * want


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("B", [1, 40])
def test_keys_that_score_minus_infinity_weigh_nothing(dtype, B):
    """In single places, a whole tile at the beginning, several in a run and parts of a long sequence: as if they were not there.  A sequence of
    nothing else has no softmax: NaN."""
    g = gen(5)
    n, H, page, D = 5000, 2, 64, 128
    k, v, table, _ = make_cache([n] * B, H, page, D, dtype, g)
    q = randn(g, B, H, D, dtype=dtype)
    q[..., 0] = 1.0
    off = torch.zeros(n, dtype=torch.bool, device=DEV)
    for a, b in ((0, 70), (100, 101), (500, 1700), (4990, 5000)):
        off[a:b] = True
    lens = torch.full((B,), n, dtype=torch.int32, device=DEV)
    at = torch.arange(n, device=DEV)
    for b in range(B):
        k[table[b, at // page].long()[off], :, (at % page)[off], 0] = -math.inf
    rows = []
    for b in range(B):
        pages = table[b, at // page].long()
        rows.append((k[pages, :, at % page][~off].double(), v[pages, :, at % page][~off].double()))
    check_attention(ops.paged_attention(q, k, v, table, lens, scale=0.12), q, rows, 0.12, f"{B} sequences")
    nothing = ops.paged_attention(q, k, v, table, torch.full_like(lens, 65), scale=0.12)
    assert bool(torch.isnan(nothing).all())


def test_strides_of_every_tensor():
    """Views: queries of one projection, pages that lie [page, row, head, D] or between others, a slice of a wider table, a slice of the output."""
    g = gen(5)
    lens, H, D, page = [70, 1, 300], 3, 128, 16
    k, v, table, rows = make_cache(lens, H, page, D, BF16, g)
    lt = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = randn(g, 3, 4 * H, D, dtype=BF16)[:, H:3 * H]
    base = ops.paged_attention(q.contiguous(), k, v, table, lt)
    check_attention(base, q, rows, ops.ATTN_SCALE, "contiguous")
    k2 = k.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    v2 = torch.zeros(v.shape[0], 2, H + 1, page, D + 8, dtype=BF16, device=DEV)[:, 1, 1:, :, 8:]
    v2.copy_(v)
    wide = torch.full((5, table.shape[1] + 7), 9999, dtype=torch.int32, device=DEV)
    wide[:3, 3:3 + table.shape[1]] = table
    room = torch.full((3, 2, 2 * H + 2, D), 5.0, dtype=BF16, device=DEV)
    out = room[:, 1, 1:-1]
    got = ops.paged_attention(q, k2, v2, wide[:3, 3:3 + table.shape[1]], lt, out=out)
    assert got is out and torch.equal(got, base)
    assert bool((room[:, 0] == 5).all() and (room[:, 1, 0] == 5).all() and (room[:, 1, -1] == 5).all())


def test_strides_of_dims_of_one_say_nothing():
    g = gen(15)
    k, v, table, rows = make_cache([40], 1, 16, 64, BF16, g)
    odd = lambda t: torch.as_strided(t, t.shape, (3, 5) + t.stride()[2:])      # noqa: E731
    q = odd(randn(g, 1, 1, 64, dtype=BF16))
    assert q.stride() == (3, 5, 1)
    o = ops.paged_attention(q, k, v, table, torch.tensor([40], dtype=torch.int32, device=DEV), out=odd(torch.empty(1, 1, 64, dtype=BF16, device=DEV)))
    check_attention(o, q, rows, ops.ATTN_SCALE, "one row")
    x, pos = odd(randn(g, 1, 1, 64, dtype=BF16)), torch.tensor([5], dtype=torch.int32, device=DEV)
    ops.paged_append(x, x, k, v, table, pos, q=x)
    assert torch.equal(k[int(table[0, 0]), 0, 5], x[0, 0])


def test_rows_of_the_table_behind_the_last_sequence_are_not_read():
    g = gen(6)
    k, v, table, rows = make_cache([40, 50], 1, 16, 64, BF16, g)
    more = torch.cat([table, torch.full((3, table.shape[1]), 1 << 30, dtype=torch.int32, device=DEV)])
    q = randn(g, 2, 1, 64, dtype=BF16)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    o = ops.paged_attention(q, k, v, more, torch.tensor([40, 50], dtype=torch.int32, device=DEV), status=status)
    check_attention(o, q, rows, ops.ATTN_SCALE, "first rows")
    assert int(status) == 0


@pytest.mark.parametrize("bad", [-1, 10 ** 6, -2 ** 31, 2 ** 31 - 1])
def test_a_page_that_is_none_is_reported_and_touches_nothing_else(bad):
    g = gen(7)
    lens, H = [40, 3000, 50], 2
    k, v, table, rows = make_cache(lens, H, 16, 128, BF16, g)
    table[1, 100] = bad
    q = randn(g, 3, H, 128, dtype=BF16)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    o = ops.paged_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=DEV), status=status)
    assert int(status) == _lib.STATUS_PAGE_OUT_OF_RANGE
    assert bool(torch.isnan(o[1]).all())
    check_attention(o[[0, 2]], q[[0, 2]], [rows[0], rows[2]], ops.ATTN_SCALE, "the other sequences")
    with pytest.raises(RuntimeError, match="no page of the pool"):
        ops.raise_for_status(status)


def test_a_length_past_the_table_is_reported():
    g = gen(8)
    k, v, table, rows = make_cache([40, 64], 1, 16, 64, BF16, g)
    q = randn(g, 2, 1, 64, dtype=BF16)
    table = table[:, :4].contiguous()
    table[0] = table[1]
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    o = ops.paged_attention(q, k, v, table, torch.tensor([2 ** 31 - 1, 64], dtype=torch.int32, device=DEV), status=status)
    assert int(status) == _lib.STATUS_LENGTH_PAST_PAGES and bool(torch.isnan(o[0]).all())
    check_attention(o[1:], q[1:], rows[1:], ops.ATTN_SCALE, "the other sequence")
    with pytest.raises(RuntimeError, match="past what the page table has room for"):
        ops.raise_for_status(status)


def test_offsets_past_32_bits():
    """A pool of more than 2^31 elements: the last pages are reached with 64-bit offsets, for reading and for writing."""
    H, page, D = 1, 256, 256
    pages = (1 << 31) // (H * page * D) + 4
    k = torch.empty(pages, H, page, D, dtype=BF16, device=DEV)
    v = torch.empty_like(k)
    g = gen(9)
    n = 300
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device=DEV)
    kk, vv = randn(g, n, H, D, dtype=BF16), randn(g, n, H, D, dtype=BF16)
    ops.paged_append(kk, vv, k, v, table, torch.arange(n, dtype=torch.int32, device=DEV), rows=torch.zeros(n, dtype=torch.int32, device=DEV))
    assert torch.equal(k[pages - 1, 0], kk[:256, 0]) and torch.equal(v[pages - 3, 0, :44], vv[256:, 0])
    q = randn(g, 1, 2, D, dtype=BF16)
    o = ops.paged_attention(q, k, v, table, torch.tensor([n], dtype=torch.int32, device=DEV))
    check_attention(o, q, [(kk.double(), vv.double())], ops.ATTN_SCALE, "far pages")


# ---------------------------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------------------------
def prepared(x, pos, cos, sin, eps):
    """Norm and rotation in 64 bits, and the magnitude that their roundings are relative to."""
    x = x.double()
    if eps is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    if cos is None:
        return x, x.abs()
    c, s = cos.double()[pos.clamp(min=0).long()][:, None], sin.double()[pos.clamp(min=0).long()][:, None]
    a, b = x.chunk(2, -1)
    size = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], -1)
    return torch.cat([a * c + b * s, b * c - a * s], -1), size


def near(got, want, size, what):
    E, least = half_step(got.dtype), torch.finfo(got.dtype).smallest_normal * half_step(got.dtype)
    err = (got.double() - want).abs()
    tol = E * want.abs() + 2 ** -20 * size + least
    assert bool((err <= tol).all()), f"{what}: {err.max().item():.3e}, {(err / tol).max().item():.2f} of what it may be"


def tables(D, rows, g):
    theta = torch.rand(rows, D // 2, generator=g, device=DEV) * 6.3
    return theta.cos().contiguous(), theta.sin().contiguous()


@pytest.mark.parametrize("source,cache", [(BF16, BF16), (BF16, F16), (F16, F16), (F16, BF16)])
@pytest.mark.parametrize("D,Hq,H,page", [(64, 4, 4, 16), (128, 3, 3, 48), (128, 8, 1, 64), (256, 2, 2, 16), (64, 0, 5, 32)])
@pytest.mark.parametrize("norm,rotate,mix", [(True, True, True), (False, True, False), (True, False, False), (False, False, True)])
def test_append_of_packed_prompts(source, cache, D, Hq, H, page, norm, rotate, mix):
    print(f"paged append {source}->{cache} D{D} Hq{Hq} H{H} page {page} norm {norm} rotation {rotate} mix {mix}", flush=True)
    g = gen(D + H)
    lens, start = [1, 70, 5, 33], [0, 3, 95, 16]
    width = -(-130 // page)
    table = torch.randperm(4 * width + 2, generator=g, device=DEV)[:4 * width].view(4, width).to(torch.int32)
    k_pages, v_pages = randn(g, 4 * width + 2, H, page, D, dtype=cache), randn(g, 4 * width + 2, H, page, D, dtype=cache)
    rows = torch.tensor([s for s, n in enumerate(lens) for _ in range(n)], dtype=torch.int32, device=DEV)
    pos = torch.tensor([a + t for a, n in zip(start, lens) for t in range(n)], dtype=torch.int32, device=DEV)
    N = pos.numel()
    pos[[4, 40]] = -1
    qkv = randn(g, N, Hq + 2 * H, D, dtype=source)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
    cos, sin = tables(D, 200, g) if rotate else (None, None)
    eps = 1e-6 if norm else None
    ve, gate = (randn(g, N, H, D, dtype=source), torch.tensor([0.3], device=DEV)) if mix else (None, None)
    before = k_pages.clone(), v_pages.clone()
    k_out, v_out = torch.full((N, H, D), 3.0, dtype=source, device=DEV), torch.full((N, H, D), 3.0, dtype=source, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = ops.paged_append(k, v, k_pages, v_pages, table, pos, rows=rows, q=q if Hq else None, cos=cos, sin=sin, eps=eps, ve=ve, gate=gate,
                           k_out=k_out, v_out=v_out, status=status)
    live = pos >= 0
    if Hq:
        other = ops.paged_append(k, v, k_pages, v_pages, table, pos, rows=rows, q=q, cos=cos, sin=sin, eps=eps, ve=ve, gate=gate, q_out=torch.empty(N, Hq, D, dtype=source, device=DEV))
        near(other[live], *(t[live] for t in prepared(q, pos, cos, sin, eps)), "q in the inputs' type")
        assert got.dtype == cache and bool((got[~live] == 0).all())
        want, size = prepared(q, pos, cos, sin, eps)
        near(got[live], want[live], size[live], "q")
    else:
        assert got is None
    vw, vs = prepared(v, pos, None, None, eps)
    if mix:
        vw, vs = 0.3 * vw + 0.7 * ve.double(), vs + ve.double().abs()
    for pages, old, (want, size), copy, name in ((k_pages, before[0], prepared(k, pos, cos, sin, eps), k_out, "k"), (v_pages, before[1], (vw, vs), v_out, "v")):
        p = table[rows.long(), (pos.clamp(min=0) // page).long()].long()[live]
        slot = (pos % page).long()[live]
        near(pages[p, :, slot], want[live], size[live], name)
        rest = pages.clone()
        rest[p, :, slot] = old[p, :, slot]
        assert torch.equal(rest, old), f"{name}: rows that no token has stay as they were"
        near(copy[live], want[live], size[live], name + " copy")
        assert bool((copy[~live] == 3).all()), "a skipped token's row of a caller's buffer stays as it was"
    assert int(status) == 0


@pytest.mark.parametrize("N", [1, 2, 63, 64, 65, 300])
def test_append_of_one_token_per_sequence(N):
    g = gen(N)
    H, D, page = 3, 128, 16
    pos = torch.randint(0, 100, (N,), generator=g, device=DEV).to(torch.int32)
    table = torch.full((N + 2, 7), -1, dtype=torch.int32, device=DEV)
    table[torch.arange(N, device=DEV), (pos // page).long()] = torch.randperm(N, generator=g, device=DEV).to(torch.int32)
    k_pages, v_pages = randn(g, N, H, page, D, dtype=BF16), randn(g, N, H, page, D, dtype=BF16)
    k, v, q = (randn(g, N, H, D, dtype=BF16) for _ in range(3))
    cos, sin = tables(D, 100, g)
    q_out = torch.empty(N, 2 * H, D, dtype=BF16, device=DEV)[:, H:]
    got = ops.paged_append(k, v, k_pages, v_pages, table, pos, q=q, cos=cos, sin=sin, q_out=q_out)
    assert got is q_out
    want, size = prepared(q, pos, cos, sin, None)
    near(got, want, size, "q")
    at = table[torch.arange(N, device=DEV), (pos // page).long()].long(), (pos % page).long()
    want, size = prepared(k, pos, cos, sin, None)
    near(k_pages[at[0], :, at[1]], want, size, "k")
    assert torch.equal(v_pages[at[0], :, at[1]], v)


def test_rows_of_the_callers_queries_stay_where_a_token_is_skipped():
    g = gen(2)
    k_pages, v_pages = randn(g, 3, 1, 16, 64, dtype=BF16), randn(g, 3, 1, 16, 64, dtype=BF16)
    before = k_pages.clone(), v_pages.clone()
    q_out = torch.full((3, 1, 64), 3.0, dtype=BF16, device=DEV)
    x = randn(g, 3, 1, 64, dtype=BF16)
    ops.paged_append(x, x, k_pages, v_pages, torch.zeros(3, 1, dtype=torch.int32, device=DEV), torch.full((3,), -1, dtype=torch.int32, device=DEV), q=x, q_out=q_out)
    assert bool((q_out == 3).all()) and torch.equal(k_pages, before[0]) and torch.equal(v_pages, before[1])


@pytest.mark.parametrize("what,bits", [("page", 4), ("page below", 4), ("row", 2), ("row below", 2), ("position", 2), ("table", 1)])
def test_append_to_nowhere_is_reported_and_writes_nothing(what, bits):
    g = gen(11)
    H, D, page = 2, 128, 16
    k_pages, v_pages = randn(g, 4, H, page, D, dtype=BF16), randn(g, 4, H, page, D, dtype=BF16)
    before = k_pages.clone(), v_pages.clone()
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV)
    pos = torch.tensor([5, 20], dtype=torch.int32, device=DEV)
    rows = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    cos, sin = tables(D, 32, g)
    if what == "page":
        table[1, 1] = 4
    elif what == "page below":
        table[1, 1] = -1
    elif what == "row":
        rows[1] = 2
    elif what == "row below":
        rows[1] = -1
    elif what == "position":
        pos[1] = 2 ** 31 - 1
        cos = sin = None
    else:
        cos, sin = cos[:20].contiguous(), sin[:20].contiguous()
    k, v, q = (randn(g, 2, H, D, dtype=BF16) for _ in range(3))
    copy = torch.zeros(2, H, D, dtype=BF16, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = ops.paged_append(k, v, k_pages, v_pages, table, pos, rows=rows, q=q, cos=cos, sin=sin, k_out=copy, status=status)
    assert int(status) == bits
    assert bool(torch.isnan(got[1]).all() and torch.isnan(copy[1]).all()) and bool(torch.isfinite(got[0]).all())
    for pages, old in ((k_pages, before[0]), (v_pages, before[1])):
        changed = (pages != old).flatten(1).any(1)
        assert changed.tolist() == [True, False, False, False]
    with pytest.raises(RuntimeError):
        ops.raise_for_status(status)


# ---------------------------------------------------------------------------------------------------------------
# the two of them as a decode step has them
# ---------------------------------------------------------------------------------------------------------------
class Steps:
    """A few sequences whose positions and lengths count up on the device."""

    def __init__(self, seed, dtype=BF16):
        self.g = gen(seed)
        self.B, self.H, self.D, self.page = 5, 2, 128, 16
        g = self.g
        self.k, self.v = randn(g, 40, self.H, self.page, self.D, dtype=dtype), randn(g, 40, self.H, self.page, self.D, dtype=dtype)
        self.table = torch.randperm(40, generator=g, device=DEV).view(5, 8).to(torch.int32)
        self.pos = torch.tensor([0, 14, 31, 100, -1], dtype=torch.int32, device=DEV)
        self.cos, self.sin = tables(self.D, 128, g)
        self.x = randn(g, 5, 3 * self.H, self.D, dtype=BF16)
        self.lens = torch.zeros(5, dtype=torch.int32, device=DEV)

    def step(self):
        H = self.H
        torch.add(self.pos, 1, out=self.lens)
        q = ops.paged_append(self.x[:, H:2 * H], self.x[:, 2 * H:], self.k, self.v, self.table, self.pos, q=self.x[:, :H], cos=self.cos, sin=self.sin, eps=1e-6)
        return ops.paged_attention(q, self.k, self.v, self.table, self.lens)

    def exact(self):
        rows = []
        for b, n in enumerate(self.lens.tolist()):
            t = torch.arange(n, device=DEV)
            p = self.table[b, t // self.page].long()
            rows.append((self.k[p, :, t % self.page].double(), self.v[p, :, t % self.page].double()))
        return rows


def test_steps_recorded_once_and_replayed_while_sequences_grow():
    s, ref = Steps(1), Steps(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = s.step()
    for it in range(6):
        print(f"replay {it}", flush=True)
        x = randn(s.g, 5, 6, 128, dtype=BF16)
        s.x.copy_(x)
        ref.x.copy_(x)
        graph.replay()
        want = ref.step()
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(s.k, ref.k) and torch.equal(s.v, ref.v), it
        q = prepared(x[:, :2], s.pos, s.cos, s.sin, 1e-6)[0].to(BF16)
        check_attention(o[:4], q[:4], ref.exact()[:4], ops.ATTN_SCALE, f"replay {it}")
        for t in (s, ref):
            t.pos[:4] += 1
            if it == 2:          # a sequence comes, another one goes
                t.pos[4], t.pos[0] = 7, -1


def test_calls_on_two_streams_at_once():
    a, b = Steps(2), Steps(3, dtype=F16)
    want = [Steps(2).step(), Steps(3, dtype=F16).step()]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for it in range(10):
        for i, (s, x) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                got[i].append(x.step())
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(o, want[i]) for o in got[i])


@pytest.mark.parametrize("lens", [[1, 40, 0, 7], [3000, 5, 900]])
def test_results_in_the_place_of_the_inputs(lens):
    g = gen(19)
    B, H, G, D = len(lens), 2, 4, 128
    k, v, table, _ = make_cache(lens, H, 32, D, BF16, g, junk=0.0)
    cos, sin = tables(D, 4000, g)
    pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device=DEV)
    seen = torch.tensor(lens, dtype=torch.int32, device=DEV)
    x = randn(g, B, H * G + 2 * H, D, dtype=BF16)
    y, kc, vc = x.clone(), k.clone(), v.clone()
    part = lambda t: (t[:, :H * G], t[:, H * G:H * G + H], t[:, H * G + H:])      # noqa: E731
    (q, kk, vv), (q2, k2, v2) = part(x), part(y)
    want = [torch.full_like(t, 0.0) for t in (q, kk, vv)]
    for t, s in zip(want, (q, kk, vv)):
        t.copy_(s)                                   # (skipped tokens stay as they are)
    ops.paged_append(kk, vv, k, v, table, pos, q=q, cos=cos, sin=sin, eps=1e-6, q_out=want[0], k_out=want[1], v_out=want[2])
    ops.paged_append(k2, v2, kc, vc, table, pos, q=q2, cos=cos, sin=sin, eps=1e-6, q_out=q2, k_out=k2, v_out=v2)
    assert all(torch.equal(a, b) for a, b in zip(want, (q2, k2, v2))) and torch.equal(k, kc) and torch.equal(v, vc)
    o = ops.paged_attention(want[0], k, v, table, seen)
    assert torch.equal(ops.paged_attention(q2, k, v, table, seen, out=q2), o)


def test_prefixes_shared_by_sequences():
    """Two sequences whose tables name the same first pages, as a shared prompt has them."""
    g = gen(12)
    k, v, table, rows = make_cache([100, 50], 2, 16, 64, BF16, g)
    table[1, :3] = table[0, :3]
    shared = (torch.cat([rows[0][0][:48], rows[1][0][48:]]), torch.cat([rows[0][1][:48], rows[1][1][48:]]))
    q = randn(g, 2, 2, 64, dtype=BF16)
    o = ops.paged_attention(q, k, v, table, torch.tensor([100, 50], dtype=torch.int32, device=DEV))
    check_attention(o, q, [rows[0], shared], ops.ATTN_SCALE, "shared prefix")


def test_refusals_name_what_is_wrong():
    g = gen(13)
    k, v, table, _ = make_cache([40], 2, 16, 64, BF16, g)
    q, lens = randn(g, 1, 2, 64, dtype=BF16), torch.tensor([40], dtype=torch.int32, device=DEV)
    call = lambda **kw: ops.paged_attention(*[kw.pop(n, d) for n, d in (("q", q), ("k", k), ("v", v), ("table", table), ("lens", lens))], **kw)      # noqa: E731
    call()
    for error, kw in [(TypeError, dict(q=q.half())), (TypeError, dict(q=q.float())), (TypeError, dict(v=v.half())), (ValueError, dict(q=q[:, :1])),
                      (ValueError, dict(q=randn(g, 1, 3, 64, dtype=BF16))), (ValueError, dict(q=randn(g, 2, 2, 64, dtype=BF16))), (ValueError, dict(v=v[:-1])),
                      (ValueError, dict(table=table.long())), (ValueError, dict(table=table[:, :0])), (ValueError, dict(lens=lens.long())),
                      (ValueError, dict(lens=lens.repeat(2))), (ValueError, dict(window=0)), (ValueError, dict(window=-3)), (ValueError, dict(out=q[..., :32])),
                      (TypeError, dict(out=q.float())), (TypeError, dict(out=q.half())), (RuntimeError, dict(lens=lens.cpu())), (ValueError, dict(status=torch.zeros(2, dtype=torch.int32, device=DEV))),
                      (RuntimeError, dict(k=k[:, :, :8], v=v[:, :, :8])), (RuntimeError, dict(k=k[..., :32], v=v[..., :32], q=q[..., :32])),
                      (RuntimeError, dict(q=q.clone().requires_grad_()))]:
        with pytest.raises(error):
            call(**kw)
    assert ops.paged_attention(q[:0], k, v, table, lens[:0]).shape == (0, 2, 64)
    x, pos = randn(g, 1, 2, 64, dtype=BF16), torch.tensor([3], dtype=torch.int32, device=DEV)
    cos, sin = tables(64, 50, g)
    call = lambda **kw: ops.paged_append(*[kw.pop(n, d) for n, d in (("k", x), ("v", x), ("k_pages", k), ("v_pages", v), ("table", table), ("pos", pos))], **kw)      # noqa: E731
    call()
    for error, kw in [(TypeError, dict(k=x.float())), (TypeError, dict(v=x.half())), (ValueError, dict(k=x[:, :1])), (ValueError, dict(pos=pos.long())),
                      (ValueError, dict(rows=pos.repeat(2))), (ValueError, dict(cos=cos)), (ValueError, dict(cos=cos, sin=sin[:40])), (ValueError, dict(cos=cos.bfloat16(), sin=sin.bfloat16())),
                      (ValueError, dict(eps=-1.0)), (ValueError, dict(ve=x)), (ValueError, dict(ve=x[..., :32], gate=cos[0, :1])), (ValueError, dict(q_out=x)), (TypeError, dict(q=x.float())),
                      (ValueError, dict(q=x[:, :0])), (ValueError, dict(q=x, q_out=x[:0])), (ValueError, dict(k_out=x[:0])), (TypeError, dict(v_out=x.half())),
                      (ValueError, dict(table=table[:0])), (RuntimeError, dict(pos=pos.cpu())), (RuntimeError, dict(k=x.clone().requires_grad_())),
                      (RuntimeError, dict(k_pages=k.clone().requires_grad_()))]:
        with pytest.raises(error):
            call(**kw)
    with torch.no_grad():
        call(k=x.clone().requires_grad_())
    assert ops.paged_append(x[:0], x[:0], k, v, table, pos[:0], q=x[:0]).shape == (0, 2, 64)
