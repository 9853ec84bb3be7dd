"""Memory that the paged cache's entry points must not share, refused on the host ahead of any launch.  Calls that pass end at the launch, for want of a
GPU: with one, these are left out."""
import ctypes
import random

import pytest
import torch

from test_paged_abi import P, S2, S3, append, attend, error

pytestmark = pytest.mark.skipif(torch.cuda.device_count() > 0, reason="host addresses are no GPU's")


def strides(*s):
    return (ctypes.c_int64 * len(s))(*s)


def append_into(pages=S3, q_out=S2, k_out=None, v_out=None, N=1, num_pages=8, page=16, H=2):
    """``daisy_paged_append_fwd`` with strides of its own for everything that it writes."""
    from daisy_amd import _lib
    return _lib.load().daisy_paged_append_fwd(P, S2, P, S2, P, S2, 0, None, None, None, None, None, 0, P, pages, P, pages, 0, P, 4, 8, 4, num_pages, page, P, None,
                                              P, q_out, 0, P if k_out else None, k_out, P if v_out else None, v_out, 0, N, H, H, 128, 1e-6, None, None)


@pytest.mark.parametrize("kw", [
    dict(q_out=strides(256, 8)), dict(q_out=strides(256, 120)), dict(q_out=strides(8, 1024), N=2), dict(q_out=strides(128, 128), N=2), dict(q_out=strides(256, 128), N=3, H=4),
    dict(k_out=strides(256, 120)), dict(v_out=strides(136, 128), N=2), dict(pages=strides(4096, 2048, 8)), dict(pages=strides(4096, 2048, 120)), dict(pages=strides(4096, 2040, 128)),
    dict(pages=strides(4088, 2048, 128)), dict(pages=strides(2048, 2048, 128)), dict(pages=strides(4096, 128, 128)), dict(pages=strides(256, 128, 2040)),
    dict(pages=strides(128, 1 << 20, 1016))])
def test_written_rows_that_reach_into_each_other(kw):
    """Strides above zero, too: a row is 128 elements wide."""
    assert append_into(**kw) == -1 and "rows that are written must not overlap" in error(), error()


@pytest.mark.parametrize("os,B", [((256, 8), 1), ((256, 120), 1), ((128, 128), 2), ((248, 128), 2), ((120, 1 << 20), 2)])
def test_results_of_the_attention_that_reach_into_each_other(os, B):
    assert attend(os=strides(*os), B=B) == -1 and "rows of o must not overlap" in error(), error()


def test_nested_rows_in_any_order_of_the_dims():
    """Refused for the missing workspace, which is looked at behind the rows: these pass."""
    for os, B in (((256, 128), 2), ((128, 1 << 20), 2), ((8, 128), 1), ((264, 128), 5), ((136, 680), 5)):
        assert attend(os=strides(*os), B=B, ws=None) == -3, error()


# ---------------------------------------------------------------------------------------------------------------
# what shares memory with what
# ---------------------------------------------------------------------------------------------------------------
MEMORY = "share no memory"


def appended(N=2, Hq=2, H=2, D=128, q=(0, 128), k=(256, 128), v=(512, 128), token=768, ve=None, q_out=None, k_out=None, v_out=None, k_pages=20000, v_pages=60000, page_strides=(4096, 2048, 128)):
    """Everything in one buffer, at element offsets: (offset, head stride[, token stride]); pools of 8 pages."""
    from daisy_amd import _lib
    at = lambda t: None if t is None else P + 2 * t[0]      # noqa: E731
    st = lambda t: None if t is None else strides(t[2] if len(t) > 2 else token, t[1])      # noqa: E731
    q_out = (10000, 128, 256) if q_out is None else q_out
    return _lib.load().daisy_paged_append_fwd(at(q), st(q), at(k), st(k), at(v), st(v), 0, at(ve), st(ve), P if ve else None, None, None, 0, P + 2 * k_pages, strides(*page_strides),
                                              P + 2 * v_pages, strides(*page_strides), 0, P, 4, 8, 4, 8, 16, P, None, at(q_out), st(q_out), 0, at(k_out), st(k_out), at(v_out), st(v_out), 0,
                                              N, Hq, H, D, 1e-6, None, None)


@pytest.mark.parametrize("kw", [
    dict(q_out=(256, 128)), dict(q_out=(512, 128)), dict(k_out=(0, 128)), dict(k_out=(512, 128)), dict(v_out=(256, 128)), dict(v_out=(0, 128)),      # another one of the projection's parts
    dict(q_out=(8, 128)), dict(q_out=(128, 128)), dict(q_out=(768, 128)), dict(k_out=(256 - 8, 128)), dict(k_out=(256 + 768, 128)), dict(v_out=(512 + 120, 128)),      # its own, shifted
    dict(q_out=(0, 128, 256)), dict(q_out=(0, 256, 768)), dict(q_out=(0, 128, 768), Hq=3),                                                          # its own, other strides
    dict(ve=(9000, 128, 256), k_out=(9000, 128, 256)), dict(ve=(512, 128), v_out=(512, 128)), dict(ve=(9000, 128, 256), v_out=(9120, 128, 256)),
    dict(k_out=(10000, 128, 256)), dict(k_out=(9000, 128, 256), v_out=(9000, 128, 256)), dict(k_out=(9000, 128, 256), v_out=(9128, 128, 256)),
    dict(q_out=(20000, 128, 256)), dict(v_out=(60000 + 4096 * 8 - 512, 128, 256)), dict(k_out=(20000 - 120, 256, 128)),                            # a pool
    dict(v_pages=20000), dict(v_pages=20000 + 120), dict(v_pages=20000 + 4096), dict(v_pages=20000 + 2048 * 3 + 128 * 5),                          # the two pools
    dict(v_pages=20000 + 4096 + 8, page_strides=(8192, 2048, 128)), dict(v_pages=20000 + 4096 - 8, page_strides=(8192, 2048, 128))])
def test_appends_that_write_what_they_read(kw):
    assert appended(**kw) == -1 and MEMORY in error(), error()


@pytest.mark.parametrize("kw", [
    dict(), dict(q_out=(0, 128)), dict(q_out=(0, 128), k_out=(256, 128), v_out=(512, 128)), dict(k_out=(256, 128)), dict(ve=(9000, 128, 256), k_out=(11000, 128, 256)),
    dict(q_out=(0, 128), token=904, k_out=(64, 128), D=64), dict(N=1, q_out=(0, 128, 8)), dict(N=1, q_out=(128 * 2, 128, 8), k=(9000, 128), v=(9000, 128)),
    dict(v_pages=20000 + 4096, page_strides=(8192, 2048, 128)), dict(v_pages=20000 + 128, page_strides=(8192, 4096, 256)), dict(v_pages=20000 - 2048, page_strides=(8192, 4096, 128)),
    dict(k=(256, 128), v=(256, 128))])
def test_appends_whose_memory_is_their_own(kw):
    assert appended(**kw) == -4 and "launch failed" in error(), error()


def test_random_layouts_against_their_elements():
    """Layouts of one buffer that share an element are refused; what is refused without one lies in ranges that meet, with strides that differ or are no nest."""
    rng = random.Random(1)
    D, seen = 64, {-1: 0, -4: 0}
    for _ in range(4000):
        N, H = rng.randrange(1, 5), rng.randrange(1, 4)
        shape = rng.choice([(D * H, D), (D * H + 64, D), (D, D * N), (D, D * N + 32), (2 * D * H, 2 * D), (3 * D * H, D), (D * H, D + 8)])
        other = shape if rng.random() < 0.8 else rng.choice([(D * H, D), (D, D * N)])
        a = rng.randrange(0, 60) * 8 if rng.random() < 0.7 else 8 * rng.randrange(0, 250)
        b = 8 * rng.randrange(0, 250) if rng.random() < 0.7 else a
        of = lambda at, st: {at + i * st[0] + j * st[1] + d for i in range(N) for j in range(H) for d in range(D)}      # noqa: E731
        k, out = of(a, shape), of(b, other)
        rc = appended(N=N, Hq=1, H=H, D=D, q=(15000, 64, 64), q_out=(16000, 64, 64), k=(a, shape[1], shape[0]), v=(17000, 64, 256), k_out=(b, other[1], other[0]), page_strides=(4096, 1024, 64))
        seen[rc] += 1
        nest = len(out) == N * H * D
        norm = lambda st: (0 if N == 1 else st[0], 0 if H == 1 else st[1])      # noqa: E731
        if not nest:
            assert rc == -1 and "rows that are written" in error()
        elif a == b and norm(shape) == norm(other):
            assert rc == -4, error()
        elif k & out:
            assert rc == -1 and MEMORY in error(), (N, H, a, b, shape, other)
        elif norm(shape) == norm(other) or max(k) < min(out) or max(out) < min(k):
            assert rc == -4, (error(), N, H, a, b, shape, other)
    assert min(seen.values()) > 500, seen


def attended(q=(0, 256, 128), o=(4096, 256, 128), k=8192, v=24576, B=3, Hq=2, num_pages=4):
    """Everything in one buffer, at element offsets."""
    return attend(q=P + 2 * q[0], qs=strides(*q[1:]), o=P + 2 * o[0], os=strides(*o[1:]), k=P + 2 * k, v=P + 2 * v, B=B, Hq=Hq, num_pages=num_pages, ws=P + 100000)


@pytest.mark.parametrize("kw", [
    dict(o=(8, 256, 128)), dict(o=(128, 256, 128)), dict(o=(256, 256, 128)), dict(o=(0, 128, 384)), dict(q=(4096 + 760, 256, 128)), dict(o=(8192, 256, 128)), dict(o=(8192 + 16384 - 8, 256, 128)),
    dict(o=(24576 + 16384 - 128, 256, 128)), dict(o=(8192 - 760, 256, 128)), dict(q=(0, 512, 128), o=(128, 512, 128)), dict(q=(0, 512, 128), o=(0, 512, 256))])
def test_attention_over_what_it_reads(kw):
    assert attended(**kw) == -1 and MEMORY in error(), error()


@pytest.mark.parametrize("kw", [dict(), dict(o=(0, 256, 128)), dict(q=(0, 512, 128), o=(256, 512, 128)), dict(q=(0, 128, 128), o=(0, 128, 128), B=1), dict(o=(8192 - 768, 256, 128)),
                                dict(q=(0, 8, 128), o=(0, 16, 128), B=1), dict(v=8192)])
def test_attention_beside_what_it_reads(kw):
    """One pool for k and v is read only, and fine."""
    assert attended(**kw) == -4 and "launch failed" in error(), error()
