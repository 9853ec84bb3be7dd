"""What the entry points of drafted trees, their attention, their verification and the moves of rows refuse before they touch a GPU, and the sizes of their
workspaces."""
import ctypes

import pytest
import torch

from daisy_amd import _lib, ops
from test_paged_abi import P, S2, S3, error

Q3, S4 = (ctypes.c_int64 * 3)(1024, 256, 128), (ctypes.c_int64 * 4)(1 << 16, 4096, 2048, 128)
OTHER = P + (1 << 14)


def strides(*s):
    return (ctypes.c_int64 * len(s))(*s)


def tree(parents=P, stride=4, lens=P, nodes=None, mask=P, positions=P, slots=P, rows=P, B=1, T=4):
    return _lib.load().daisy_draft_tree_fwd(parents, stride, lens, nodes, mask, positions, slots, rows, B, T, None)


def attend(q=P, qs=Q3, k=P, ks=S3, v=P, kind=0, table=P, stride=4, max_pages=4, num_pages=8, page=16, lens=P, mask=P, ms=S2, o=OTHER, os=Q3, o_kind=0, B=1, T=4, Hq=2, H=2, D=128, ws=P,
           ws_bytes=1 << 15):
    return _lib.load().daisy_paged_tree_attn_fwd(q, qs, k, ks, v, ks, kind, table, stride, max_pages, num_pages, page, lens, None, mask, ms, o, os, o_kind, B, T, Hq, H, D, 0, 0.12, None,
                                                 ws, ws_bytes, None)


def verify(logits=P, ls=S2, kind=0, tokens=P, ts=4, parents=P, ps=4, temps=None, t=0.0, accept=None, acs=0, noise=None, ns=0, draft=None, ds=None, path=P, counts=P, following=P, B=1, T=4,
           V=32, ws=P, ws_bytes=1 << 15):
    return _lib.load().daisy_verify_fwd(logits, ls, kind, tokens, ts, 1, parents, ps, None, temps, t, accept, acs, noise, ns, draft, ds, path, counts, following, B, T, V, ws, ws_bytes, None)


def move(k=P, ks=S4, v=P + (1 << 24), vs=S4, table=P, stride=4, n_seq=2, max_pages=4, num_pages=8, page=16, starts=P, counts=P, index=P, index_stride=4, sources=None, B=2, rows=4, L=2, H=2, D=128):
    return _lib.load().daisy_paged_move_fwd(k, ks, v, vs, table, stride, n_seq, max_pages, num_pages, page, starts, counts, index, index_stride, sources, B, rows, L, H, D, None, None)


@pytest.mark.parametrize("kw,rc,text", [
    *[({name: None}, -1, "non-NULL") for name in ("parents", "lens", "mask", "positions", "slots", "rows")],
    (dict(B=0), -1, "B=0"), (dict(T=0), -1, "T=0"), (dict(stride=-1), -1, "positive"), (dict(T=257), -2, "at most 256")])
def test_tree_argument_errors(kw, rc, text):
    assert tree(**kw) == rc and text in error(), error()


@pytest.mark.parametrize("kw,rc,text", [
    *[({name: None}, -1, "non-NULL") for name in ("q", "qs", "o", "os", "lens", "mask", "ms", "k", "v", "table")],
    (dict(B=0), -1, "B=0"), (dict(T=0), -1, "T=0"), (dict(Hq=3), -1, "Hq=3"), (dict(H=0), -1, "H=0"), (dict(T=257), -2, "at most 256"), (dict(Hq=1 << 17), -2, "65536"), (dict(D=96), -2, "head_dim 96"),
    (dict(page=8), -2, "page_size 8"), (dict(page=24), -2, "page_size"), (dict(num_pages=0), -1, "num_pages"), (dict(max_pages=0), -1, "max_pages"), (dict(max_pages=1 << 27), -1, "too long"),
    (dict(max_pages=1 << 20, B=1 << 15), -1, "too many"), (dict(q=P + 2), -1, "aligned"), (dict(o=OTHER + 8), -1, "aligned"), (dict(k=P + 8), -1, "aligned"), (dict(qs=strides(1024, 256, 12)), -1, "multiples of 8"),
    (dict(os=strides(1024, 260, 128)), -1, "multiples of 8"), (dict(ks=strides(4096, 2048, 129)), -1, "multiples of 8"), (dict(ks=strides(4096, 2048, -128)), -1, "strides"),
    (dict(ms=strides(-4, 1), B=2), -1, "mask"), (dict(ms=strides(4, -1)), -1, "mask"), (dict(o_kind=1), -2, "fp16 cache"), (dict(qs=strides(1024, 1 << 36, 128)), -2, "too long"),
    (dict(os=strides(1 << 36, 256, 128), B=2), -2, "too long"), (dict(ks=strides(1 << 36, 2048, 128)), -2, "too long"), (dict(stride=1 << 32, B=2), -2, "too long"),
    (dict(os=strides(1024, 256, 64)), -1, "overlap"), (dict(os=strides(1024, 128, 128)), -1, "overlap"), (dict(os=strides(512, 256, 128), B=2), -1, "overlap"),
    (dict(ws=None), -3, "workspace"), (dict(ws_bytes=64), -3, "workspace"), (dict(ws=P + 8), -3, "workspace"),
    (dict(o=P + 256), -1, "share no memory"), (dict(o=P, os=strides(1024, 384, 128)), -1, "share no memory"), (dict(q=P + (1 << 20), o=P + 4096), -1, "share no memory"),
    (dict(q=P + (1 << 20), k=P + (1 << 21), v=P), -1, None)])
def test_attention_argument_errors(kw, rc, text):
    if text is None:
        kw, text = {**kw, "o": P + 8192}, "share no memory"
    assert attend(**kw) == rc and text in error(), error()


@pytest.mark.parametrize("kw,rc,text", [
    *[({name: None}, -1, "non-NULL") for name in ("logits", "ls", "tokens", "parents", "path", "counts", "following")],
    (dict(B=0), -1, "B=0"), (dict(T=0), -1, "T=0"), (dict(V=0), -1, "V=0"), (dict(T=257), -2, "at most 256"), (dict(B=65536), -2, "65535"), (dict(kind=3), -2, "type 3"), (dict(kind=-1), -2, "type -1"),
    (dict(ls=strides(-1, 32)), -1, "negative"), (dict(ls=strides(128, -32)), -1, "negative"), (dict(ts=-1), -1, "negative"), (dict(ps=-1), -1, "negative"), (dict(t=-0.5), -1, "temperature"),
    (dict(t=float("nan")), -1, "temperature"), (dict(t=float("inf")), -1, "temperature"), (dict(t=1.0), -1, "needs"), (dict(t=1.0, accept=P), -1, "needs"), (dict(temps=P, noise=P), -1, "needs"),
    (dict(t=1.0, accept=P, noise=P, draft=P), -1, "strides"), (dict(draft=P, ds=strides(128, -32)), -1, "strides"), (dict(acs=-1), -1, "negative"), (dict(logits=P + 2), -1, "aligned"),
    (dict(ws=None), -3, "workspace"), (dict(ws_bytes=16), -3, "workspace"), (dict(ws=P + 8), -3, "workspace")])
def test_verification_argument_errors(kw, rc, text):
    assert verify(**kw) == rc and text in error(), error()


@pytest.mark.parametrize("kw,rc,text", [
    (dict(starts=None), -1, "non-NULL"), (dict(counts=None), -1, "non-NULL"), (dict(index=None), -1, "an index or sources"), (dict(k=None), -1, "non-NULL"), (dict(vs=None), -1, "non-NULL"),
    (dict(table=None), -1, "page table"), (dict(B=0), -1, "B=0"), (dict(B=3), -1, "at most the table's 2"), (dict(rows=0), -1, "rows=0"), (dict(L=0), -1, "L=0"), (dict(H=0), -1, "H=0"),
    (dict(B=65536, n_seq=65536), -2, "65535"), (dict(index_stride=-1), -1, "stride"), (dict(D=96), -2, "head_dim 96"), (dict(page=20), -2, "page_size"),
    (dict(num_pages=0), -1, "num_pages"), (dict(max_pages=1 << 27), -1, "too long"), (dict(k=P + 2), -1, "aligned"), (dict(ks=strides(1 << 16, 4096, 2048, 130)), -1, "multiples of 8"),
    (dict(ks=strides((1 << 16) + 4, 4096, 2048, 128)), -1, "multiples of 8"), (dict(ks=strides(1 << 16, 4096, 2048, 64)), -1, "overlap"), (dict(ks=strides(1 << 14, 4096, 2048, 128)), -1, "overlap"),
    (dict(v=P + 256), -1, "share no memory"), (dict(v=P), -1, "share no memory"), (dict(v=P + (1 << 17)), -1, "share no memory"), (dict(v=P + (1 << 17) + (1 << 16) - 256), -1, "share no memory"),
    (dict(L=1 << 20, H=1 << 12, ks=strides(1 << 40, 4096 << 12, 2048, 128), vs=strides(1 << 40, 4096 << 12, 2048, 128), v=P + (1 << 38)), -1, "too many")])
def test_move_argument_errors(kw, rc, text):
    assert move(**kw) == rc and text in error(), error()


@pytest.mark.skipif(torch.cuda.device_count() > 0, reason="host addresses are no GPU's")
def test_layers_in_any_order_of_the_dims_can_be_moved():
    """These end at the launch, for want of a GPU: layers of each page beside one another, k and v of each layer, and v in what the layers of k leave free."""
    inside = strides(4096, 3 * 4096, 2048, 128)
    for kw in (dict(ks=inside, vs=inside, L=3), dict(ks=inside, vs=inside, L=1, v=P + 2 * 4096), dict(ks=strides(2 * 4096, 6 * 4096, 2048, 128), vs=strides(2 * 4096, 6 * 4096, 2048, 128), L=3, v=P + 2 * 4096),
               dict(v=P + (1 << 16))):
        assert move(**kw) == -4, error()
    for kw in (dict(ks=inside, vs=inside, L=4), dict(ks=inside, vs=inside, L=3, v=P + 2 * 4096), dict(ks=inside, vs=inside, L=2, v=P + 2 * 4096)):
        assert move(**kw) == -1 and ("overlap" in error() or "share" in error()), error()


def test_workspaces():
    size = ops.verify_drafts_workspace_bytes
    assert size(0, 4, 32) == size(1, 0, 32) == size(1, 4, 0) == size(1, 257, 32) == size(65536, 4, 32) == 0
    assert 0 < size(1, 1, 1) <= size(1, 1, 50000) <= size(64, 8, 50000) <= size(65535, 256, 50000)
    size = ops.paged_tree_attention_workspace_bytes
    assert size(0, 1, 1, 1, 128, 1, 16) == size(1, 257, 1, 1, 128, 1, 16) == size(1, 1, 3, 2, 128, 1, 16) == size(1, 1, 1, 1, 80, 1, 16) == size(1, 1, 1, 1, 128, 1 << 27, 16) == 0
    # two partial results of D + 2 floats for every column of a workgroup, and 32 bytes: columns are the queries of a key head, 256 of them at most
    assert size(1, 1, 1, 1, 128, 1, 16) % (32 + 2 * 130 * 4) == 0
    assert size(1, 64, 8, 1, 128, 4096, 64) % (32 + 2 * 256 * 130 * 4) == 0
    assert size(1000, 64, 64, 8, 128, 4096, 64) < 1 << 28      # (bounded by what the chip holds)


def test_cpu_tensors_and_shapes_are_refused():
    ints = lambda *shape: torch.zeros(*shape, dtype=torch.int32)      # noqa: E731
    half = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16)      # noqa: E731
    k = half(2, 1, 16, 64)
    for call in (lambda: ops.draft_tree(ints(1, 4), ints(1)), lambda: ops.paged_tree_attention(half(1, 4, 1, 64), k, k, ints(1, 2), ints(1), ints(1, 4, 1)),
                 lambda: ops.verify_drafts(torch.zeros(1, 4, 32), torch.zeros(1, 4, dtype=torch.long), ints(1, 4)),
                 lambda: ops.paged_move(k, k.clone(), ints(1, 2), ints(1), ints(1), index=ints(1, 4)),
                 lambda: ops.paged_append(half(1, 1, 64), half(1, 1, 64), k, k.clone(), ints(1, 2), ints(1), slots=ints(1))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(ValueError, match="window must be positive"):
        ops.paged_tree_attention(half(1, 4, 1, 64), k, k, ints(1, 2), ints(1), ints(1, 4, 1), window=0)
    with pytest.raises(RuntimeError, match="does not rise"):
        ops.raise_for_status(torch.tensor([8], dtype=torch.int32))


@pytest.mark.gpu
def test_what_the_python_entry_points_refuse():
    dev = "cuda:0"
    ints = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=dev)      # noqa: E731
    half = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16, device=dev)      # noqa: E731
    k, v, table, lens, mask, parents = half(3, 2, 16, 64), half(3, 2, 16, 64), ints(2, 3), ints(2), ints(2, 4, 1), ints(2, 4)
    q, logits, tokens = half(2, 4, 4, 64), torch.zeros(2, 4, 30, device=dev), torch.zeros(2, 4, dtype=torch.long, device=dev)
    rand, noise = torch.rand(2, 4, device=dev), torch.zeros(2, 30, device=dev)

    def attend(q=q, k=k, v=v, table=table, lens=lens, mask=mask, **kw):
        return ops.paged_tree_attention(q, k, v, table, lens, mask, **kw)

    def verify(logits=logits, tokens=tokens, parents=parents, **kw):
        return ops.verify_drafts(logits, tokens, parents, **kw)

    def move(k=k, v=v, table=table, starts=lens, counts=lens, **kw):
        return ops.paged_move(k, v, table, starts, counts, **kw)
    index = ints(2, 4)
    for call, error, text in (
            (lambda: ops.draft_tree(parents.long(), lens), ValueError, "parents must be"), (lambda: ops.draft_tree(parents[:1], lens), ValueError, "parents must be"),
            (lambda: ops.draft_tree(parents.t().contiguous().t(), lens), ValueError, "contiguous"), (lambda: ops.draft_tree(parents, lens.long()), ValueError, "lens must be"),
            (lambda: ops.draft_tree(parents, lens, nodes=ints(3)), ValueError, "nodes"), (lambda: ops.draft_tree(ints(2, 257), lens), ValueError, "1 to 256"),
            (lambda: ops.draft_tree(ints(2, 0), lens), ValueError, "1 to 256"),
            (lambda: attend(q=q.float()), (TypeError, ValueError), "q"), (lambda: attend(q=q.half()), (TypeError, ValueError), "q"), (lambda: attend(q=q[:, :, :3]), ValueError, "multiple of 2"),
            (lambda: attend(q=q[0]), ValueError, "q"), (lambda: attend(mask=mask[:, :3]), ValueError, "mask must be"), (lambda: attend(mask=mask.long()), ValueError, "mask must be"),
            (lambda: attend(lens=lens.long()), ValueError, "lens"), (lambda: attend(lens=ints(1)), ValueError, "lens"), (lambda: attend(table=table[:1]), ValueError, "rows for 2"),
            (lambda: attend(nodes=ints(2).float()), ValueError, "nodes"), (lambda: attend(out=half(2, 4, 4, 32)), ValueError, "out"), (lambda: attend(out=torch.zeros_like(q).half()), (TypeError, ValueError), "out"),
            (lambda: attend(out=q.clone().requires_grad_()), RuntimeError, "no backward"), (lambda: attend(q=q.clone().requires_grad_()), RuntimeError, "no backward"),
            (lambda: attend(out=q[:, :, :1].expand(2, 4, 4, 64)), RuntimeError, "overlap"), (lambda: attend(status=ints(2)), ValueError, "status"),
            (lambda: verify(logits=logits.double()), TypeError, "float32"), (lambda: verify(logits=logits[0]), ValueError, "logits must be"),
            (lambda: verify(logits=logits.transpose(1, 2).contiguous().transpose(1, 2)), ValueError, "contiguous"), (lambda: verify(tokens=tokens[:, :3]), ValueError, "tokens must be"),
            (lambda: verify(tokens=tokens.float()), ValueError, "tokens must be"), (lambda: verify(parents=parents[:, :3]), ValueError, "parents must be"), (lambda: verify(temperature=1.0), ValueError, "needs accept"),
            (lambda: verify(temperature=-1.0), ValueError, "not be negative"), (lambda: verify(temperature=torch.ones(3, device=dev), accept=rand, noise=noise), ValueError, "temperature"),
            (lambda: verify(temperature=1.0, accept=rand[:, :3], noise=noise), ValueError, "accept must be"), (lambda: verify(temperature=1.0, accept=rand, noise=noise[:1]), ValueError, "noise must be"),
            (lambda: verify(temperature=1.0, accept=rand, noise=noise, draft=logits.bfloat16()), ValueError, "draft must be"), (lambda: verify(nodes=ints(1)), ValueError, "nodes"),
            (lambda: verify(logits=logits.clone().requires_grad_()), RuntimeError, "no backward"), (lambda: verify(temperature=1.0, accept=rand, noise=noise, draft=logits.clone().requires_grad_()), RuntimeError, "no backward"),
            (lambda: move(), ValueError, "index"), (lambda: move(sources=lens), ValueError, "rows"), (lambda: move(index=index.long()), ValueError, "index"), (lambda: move(index=index[:1]), ValueError, "index"),
            (lambda: move(index=index, starts=lens[:1]), ValueError, "counts|starts"), (lambda: move(index=index, counts=lens.long()), ValueError, "counts"), (lambda: move(index=index, k=k.float(), v=v.float()), (TypeError, ValueError), "pages"),
            (lambda: move(index=index, v=k), RuntimeError, "share no memory"), (lambda: move(index=index, k=k.clone().requires_grad_()), RuntimeError, "no backward"),
            (lambda: move(rows=4, sources=ints(3)), ValueError, "sources")):
        with pytest.raises(error, match=text):
            call()
    # the same calls, made right
    ops.draft_tree(parents, lens), attend(), verify(), verify(temperature=1.0, accept=rand, noise=noise, draft=logits), move(index=index), move(rows=4, sources=lens)
    torch.cuda.synchronize()
