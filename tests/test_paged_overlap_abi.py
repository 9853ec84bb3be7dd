"""Memory that the paged cache's entry points must not share, refused on the host ahead of any launch."""
import ctypes

import pytest

from test_paged_abi import P, S2, S3, append, attend, error


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
