"""Results of the logits' operator over what its other workgroups read, refused on the host.  Calls that pass end at the launch, for want of a GPU: with one,
these are left out."""
import ctypes

import pytest
import torch

from daisy_amd import _lib

pytestmark = pytest.mark.skipif(torch.cuda.device_count() > 0, reason="host addresses are no GPU's")
BUF = ctypes.create_string_buffer(1 << 16)
P = (ctypes.addressof(BUF) + 255) & ~255
B, V, T = 3, 100, 10


def process(x=(0, 100), y=(2000, 100), kind=0, history=(8000, 10), int64=1, lens=9000, repetition=9100, presence=9200, frequency=9300, bias=(10000, 100), allowed=(12000, 4), rows=B):
    """Byte offsets in one buffer, strides in elements."""
    at = lambda o: None if o is None else P + o      # noqa: E731
    rc = _lib.load().daisy_logits_process_fwd(at(x[0]), x[1], at(y[0]), y[1], kind, at(history[0]), history[1], int64, at(lens), T, T, at(repetition), 1.0, at(presence), 0.0, at(frequency), 0.0,
                                              0.0, 1.0, at(bias[0]), bias[1], at(allowed[0]), allowed[1], rows, V, None)
    return rc, _lib.load().daisy_last_error().decode()


@pytest.mark.parametrize("kw", [
    dict(history=(2000, 10)), dict(history=(2000 + 1196, 10)), dict(history=(2000 - 236, 10)), dict(history=(2000 - 72, 100)), dict(history=(1196, 300), y=(1200, 600)),
    dict(int64=0, history=(2000 - 116, 10)), dict(lens=2000), dict(lens=2000 + 1196), dict(lens=1992), dict(repetition=2100), dict(presence=2800), dict(frequency=3196),
    dict(bias=(2000, 100)), dict(bias=(2000, 0)), dict(bias=(1604, 0)), dict(bias=(3196, 0)), dict(bias=(2396, 200), y=(2000, 200)), dict(bias=(2000, 101)),
    dict(allowed=(2000, 4)), dict(allowed=(3196, 0)), dict(allowed=(1988, 0)), dict(allowed=(1960, 4)), dict(y=(0, 100), bias=(0, 100)), dict(rows=1, bias=(2396, 100))])
def test_results_over_what_is_read(kw):
    rc, text = process(**kw)
    assert rc == -1 and "must lie apart from the history" in text, text


@pytest.mark.parametrize("kw", [
    dict(), dict(y=(0, 100)), dict(y=(2000, 200), bias=(2400, 200)), dict(y=(2400, 200), bias=(2000, 200)), dict(y=(2000, 200), bias=(2400, 0)), dict(bias=(3200, 0)), dict(bias=(1600, 0)),
    dict(y=(2000, 120), allowed=(2400, 120)), dict(y=(2000, 120), history=(2400, 60)), dict(lens=1988), dict(lens=3200), dict(history=(3200, 10)), dict(history=(2000 - 240, 10)),
    dict(bias=(None, 0), allowed=(None, 0), lens=None, repetition=None, presence=None, frequency=None), dict(rows=1, bias=(2400, 100)), dict(kind=1, y=(2000, 100), bias=(2600, 0))])
def test_results_beside_what_is_read(kw):
    rc, text = process(**kw)
    assert rc == -4 and "launch failed" in text, text
