"""Results of the paged cache's operators in memory that they share with other tensors, row beside row: what they are in memory of their own."""
import pytest
import torch

from daisy_amd import ops
from test_paged_gpu import BF16, DEV, gen, make_cache, randn, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,Hq,H", [(1, 2, 2), (5, 4, 2), (70, 6, 3)])
def test_appends_into_one_buffer_of_everything(N, Hq, H):
    """Queries in place, keys and values into rows beside them, pages of k and v in turn in one pool."""
    g = gen(N)
    D, page, pages = 128, 16, 8
    room = randn(g, N, Hq + 4 * H, D, dtype=BF16)
    q, k, v, k_out, v_out = room[:, :Hq], room[:, Hq:Hq + H], room[:, Hq + H:Hq + 2 * H], room[:, Hq + 2 * H:Hq + 3 * H], room[:, Hq + 3 * H:]
    own = [t.clone() for t in (q, k, v)]
    pool = torch.zeros(pages, 2, H, page, D, dtype=BF16, device=DEV)
    k_pages, v_pages = torch.zeros(pages, H, page, D, dtype=BF16, device=DEV), torch.zeros(pages, H, page, D, dtype=BF16, device=DEV)
    table = torch.randperm(pages, generator=g, device=DEV).view(1, pages).to(torch.int32)
    rows, pos = torch.zeros(N, dtype=torch.int32, device=DEV), torch.arange(N, dtype=torch.int32, device=DEV)
    cos, sin = tables(D, 128, g)
    kw = dict(rows=rows, cos=cos, sin=sin, eps=1e-6)
    want = [torch.empty_like(t) for t in own]
    ops.paged_append(own[1], own[2], k_pages, v_pages, table, pos, q=own[0], q_out=want[0], k_out=want[1], v_out=want[2], **kw)
    ops.paged_append(k, v, pool[:, 0], pool[:, 1], table, pos, q=q, q_out=q, k_out=k_out, v_out=v_out, **kw)
    assert torch.equal(q, want[0]) and torch.equal(k_out, want[1]) and torch.equal(v_out, want[2])
    assert torch.equal(k, own[1]) and torch.equal(v, own[2])
    assert torch.equal(pool[:, 0], k_pages) and torch.equal(pool[:, 1], v_pages)


def test_appends_over_what_others_read_are_refused():
    g = gen(1)
    x = randn(g, 3, 6, 64, dtype=BF16)
    q, k, v = x[:, :2], x[:, 2:4], x[:, 4:]
    pages = randn(g, 2, 4, 2, 16, 64, dtype=BF16)
    table, pos = torch.zeros(3, 1, dtype=torch.int32, device=DEV), torch.arange(3, dtype=torch.int32, device=DEV)
    gate = torch.ones(1, device=DEV)
    before = x.clone(), pages.clone()
    for kw in (dict(q_out=k), dict(k_out=v), dict(v_out=k), dict(k_out=x[:, 3:5]), dict(k_out=k, v_out=k), dict(v_out=pages[0, 0].transpose(0, 1)[:3]),
               dict(ve=v.clone(), gate=gate, k_out=q), dict(k_pages=pages[1])):
        kp = kw.pop("k_pages", pages[0])
        with pytest.raises(RuntimeError, match="share no memory"):
            ops.paged_append(k, v, kp, pages[1], table, pos, q=q, **kw)
    assert torch.equal(x, before[0]) and torch.equal(pages, before[1])


@pytest.mark.parametrize("lens,G", [([40, 0, 7], 1), ([3000, 5, 900], 4)])
def test_attention_into_the_buffer_of_its_queries(lens, G):
    """Beside the queries, over them, and refused across them."""
    g = gen(G)
    H, D = 2, 128
    k, v, table, _ = make_cache(lens, H, 32, D, BF16, g)
    lt = torch.tensor(lens, dtype=torch.int32, device=DEV)
    room = randn(g, len(lens), 3 * H * G, D, dtype=BF16)
    q = room[:, :H * G]
    want = ops.paged_attention(q.clone(), k, v, table, lt)
    assert torch.equal(ops.paged_attention(q, k, v, table, lt, out=room[:, H * G:2 * H * G]), want)
    before = room.clone()
    for out in (room[:, 1:1 + H * G], room.flatten(1)[:, 8:8 + H * G * D].unflatten(1, (H * G, D)), k[0, 0, :H * G].expand(len(lens), H * G, D), k.flatten()[:q.numel()].view(q.shape)):
        with pytest.raises(RuntimeError, match="share no memory|must not overlap"):
            ops.paged_attention(q, k, v, table, lt, out=out)
    assert torch.equal(room, before)
    assert torch.equal(ops.paged_attention(q, k, v, table, lt, out=q), want)
