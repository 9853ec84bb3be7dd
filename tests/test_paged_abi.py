"""What the entry points of the paged cache and of the logits refuse before they touch a GPU, and the sizes of their workspaces."""
import ctypes

import pytest
import torch

from daisy_amd import _lib, ops

BUF = ctypes.create_string_buffer(1 << 16)
P = (ctypes.addressof(BUF) + 255) & ~255
S2, S3 = (ctypes.c_int64 * 2)(128, 128), (ctypes.c_int64 * 3)(4096, 2048, 128)


def error():
    return _lib.load().daisy_last_error().decode()


def attend(q=P, qs=S2, k=P, ks=S3, v=P, table=P, stride=4, max_pages=4, num_pages=8, page=16, lens=P, o=P, os=S2, B=1, Hq=2, H=2, D=128, ws=P, ws_bytes=1 << 15):
    return _lib.load().daisy_paged_attn_fwd(q, qs, k, ks, v, ks, 0, table, stride, max_pages, num_pages, page, lens, o, os, 0, B, Hq, H, D, 0, 0.12, None, ws, ws_bytes, None)


def append(q=P, k=P, v=P, table=P, stride=4, n_seq=1, max_pages=4, num_pages=8, page=16, positions=P, rows=None, q_out=P, N=1, Hq=2, H=2, D=128, ve=None, gate=None,
           cos=None, sin=None, table_rows=0, k_out=None, k_out_strides=None, ss=S2):
    return _lib.load().daisy_paged_append_fwd(q, S2, k, ss, v, S2, 0, ve, S2, gate, cos, sin, table_rows, P, S3, P, S3, 0, table, stride, n_seq, max_pages, num_pages, page,
                                              positions, rows, q_out, S2, 0, k_out, k_out_strides, None, None, 0, N, Hq, H, D, 1e-6, None, None)


@pytest.mark.parametrize("kw,rc,text", [
    (dict(q=None), -1, "non-NULL"), (dict(lens=None), -1, "non-NULL"), (dict(k=None), -1, "pages"), (dict(table=None), -1, "page table"), (dict(B=0), -1, "B=0"),
    (dict(Hq=3), -1, "Hq=3"), (dict(H=0), -1, "H=0"), (dict(D=96), -2, "head_dim 96"), (dict(D=512), -2, "head_dim"), (dict(page=8), -2, "page_size 8"),
    (dict(page=24), -2, "page_size"), (dict(page=0), -2, "page_size"), (dict(num_pages=0), -1, "num_pages"), (dict(max_pages=0), -1, "max_pages"),
    (dict(max_pages=1 << 27, page=16), -1, "too long"), (dict(max_pages=(1 << 27) - 63, page=16), -1, "too long"), (dict(max_pages=1 << 20, B=1 << 15), -1, "too many"),
    (dict(q=P + 2), -1, "aligned"), (dict(k=P + 8), -1, "aligned"), (dict(ks=(ctypes.c_int64 * 3)(4096, 2048, 129)), -1, "multiples of 8"),
    (dict(ks=(ctypes.c_int64 * 3)(4096, 2048, -128)), -1, "strides"), (dict(ks=(ctypes.c_int64 * 3)(4096, 2048, 1 << 23)), -1, "2^23"),
    (dict(qs=(ctypes.c_int64 * 2)(256, 1 << 35)), -2, "too long"), (dict(os=(ctypes.c_int64 * 2)(1 << 35, 128), B=2), -2, "too long"),
    (dict(ks=(ctypes.c_int64 * 3)(1 << 35, 2048, 128)), -2, "too long"), (dict(ks=(ctypes.c_int64 * 3)(4096, 1 << 36, 128)), -2, "too long"), (dict(stride=1 << 32, B=2), -2, "too long"),
    (dict(qs=(ctypes.c_int64 * 2)(128, 4)), -1, "multiples of 8"), (dict(os=(ctypes.c_int64 * 2)(256, 0)), -1, "overlap"), (dict(os=(ctypes.c_int64 * 2)(0, 128), B=2), -1, "overlap"),
    (dict(B=1 << 30, Hq=1 << 20, H=1 << 20, max_pages=1 << 20), -1, "too many"), (dict(ws=None), -3, "workspace"), (dict(ws_bytes=16), -3, "workspace"), (dict(ws=P + 4), -3, "workspace")])
def test_attention_argument_errors(kw, rc, text):
    assert attend(**kw) == rc and text in error(), error()


@pytest.mark.parametrize("kw,rc,text", [
    (dict(k=None), -1, "non-NULL"), (dict(positions=None), -1, "non-NULL"), (dict(q=None), -1, "go together"), (dict(q_out=None), -1, "go together"), (dict(Hq=0), -1, "go together"),
    (dict(N=0), -1, "N=0"), (dict(H=0), -1, "H=0"), (dict(n_seq=0), -1, "n_seq"), (dict(N=2), -1, "token i belongs"), (dict(cos=P), -1, "cos and sin"),
    (dict(cos=P, sin=P), -1, "cos and sin"), (dict(ve=P), -1, "gate"), (dict(gate=P), -1, "gate"), (dict(k_out=P), -1, "strides"), (dict(D=32), -2, "head_dim 32"),
    (dict(page=17), -2, "page_size"), (dict(k=P + 2), -1, "aligned"), (dict(ss=(ctypes.c_int64 * 2)(128, 12)), -1, "multiples of 8"),
    (dict(N=1 << 30, rows=P, Hq=1 << 20), -1, "too many rows"), (dict(k_out=P, k_out_strides=(ctypes.c_int64 * 2)(0, 0)), -1, "overlap")])
def test_append_argument_errors(kw, rc, text):
    assert append(**kw) == rc and text in error(), error()


def process(x=P, y=P, xs=100, ys=100, kind=0, history=P, T=10, lookback=10, repetition=1.0, half_life=0.0, cap=1.0, B=2, V=100):
    return _lib.load().daisy_logits_process_fwd(x, xs, y, ys, kind, history, 10, 1, None, T, lookback, None, repetition, None, 0.0, None, 0.0, half_life, cap, None, 0, None, 0, B, V, None)


@pytest.mark.parametrize("kw,rc,text", [
    (dict(x=None), -1, "non-NULL"), (dict(B=0), -1, "B=0"), (dict(B=1 << 17), -1, "65535"), (dict(V=0), -1, "V=0"), (dict(kind=3), -2, "type 3"), (dict(ys=99), -1, "overlap"),
    (dict(T=-1), -1, "T=-1"), (dict(lookback=-1), -1, "lookback=-1"), (dict(half_life=-1.0), -1, "half_life"), (dict(cap=-1.0), -1, "cap"), (dict(repetition=0.0), -1, "repetition"),
    (dict(repetition=float("nan")), -1, "repetition"), (dict(repetition=float("inf")), -1, "repetition"), (dict(T=1 << 30), -2, "too long"), (dict(T=1 << 20, lookback=1 << 17), -2, "131072"), (dict(x=P + 2), -1, "aligned"),
    (dict(y=P + 4), -1, "apart"), (dict(y=P + 4, B=1), -1, "apart"), (dict(ys=200), -1, "apart"), (dict(y=P + 400), -1, "apart"), (dict(xs=0), -1, "apart"),
    (dict(x=P + 396, xs=200, ys=200), -1, "apart"), (dict(y=P + 404, xs=200, ys=200), -1, "apart")])
def test_logits_argument_errors(kw, rc, text):
    assert process(**kw) == rc and text in error(), error()


def test_workspaces_of_the_paged_attention():
    size = ops.paged_attention_workspace_bytes
    # 16 bytes and two partial results of D + 2 floats for every query head of a unit, for each workgroup of four wavefronts with a tile of 32 positions each
    assert size(1, 1, 1, 128, 1, 16) == 16 + 2 * 130 * 4
    assert size(1, 12, 12, 128, 128, 64) == (256 * 12 // 4) * (16 + 2 * 130 * 4)
    assert size(1000, 16, 16, 128, 128, 64) == 768 * (16 + 2 * 130 * 4)               # as many workgroups as the chip holds
    assert size(1000, 64, 1, 128, 128, 64) == 512 * (16 + 2 * 16 * 130 * 4)           # at most 16 heads to a unit; their sums fill the LDS
    assert size(1 << 30, 1 << 20, 1 << 20, 128, 1 << 20, 64) == 0
    assert size(0, 1, 1, 128, 1, 16) == size(1, 3, 2, 128, 1, 16) == size(1, 1, 1, 80, 1, 16) == size(1, 1, 1, 128, 1 << 27, 16) == 0


def test_cpu_tensors_are_refused():
    k = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    table, one = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.paged_attention(torch.zeros(1, 1, 64, dtype=torch.bfloat16), k, k, table, one)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.paged_append(torch.zeros(1, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 1, 64, dtype=torch.bfloat16), k, k, table, one)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.process_logits(torch.zeros(1, 10))


def test_pages_the_device_reports():
    for bits, text in ((1, "rotary tables"), (2, "room for"), (4, "no page of the pool"), (6, "room for")):
        with pytest.raises(RuntimeError, match=text):
            ops.raise_for_status(torch.tensor([bits], dtype=torch.int32))
    ops.raise_for_status(torch.tensor([0], dtype=torch.int32))
