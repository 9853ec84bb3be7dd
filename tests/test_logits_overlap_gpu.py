"""Logits, biases and results as parts of one buffer's rows, and results over what the call reads."""
import pytest
import torch

from daisy_amd import ops
from test_logits_gpu import DEV, check, gen, history, logits

pytestmark = pytest.mark.gpu


def test_results_in_rows_shared_with_logits_and_biases():
    g = gen(2)
    B, V = 5, 1301
    room = logits(g, B, 3 * V)
    x, bias, out = room[:, :V], room[:, V:2 * V], room[:, 2 * V:]
    h, lens = history(g, B, 40, V), torch.tensor([0, 1, 40, 7, 33], dtype=torch.int32, device=DEV)
    kw = dict(repetition=torch.linspace(0.9, 1.4, B, device=DEV), frequency=0.25, bias=bias)
    want = ops.process_logits(x.clone(), h, lens, **kw)
    check(want, x, h, lens, **kw)
    assert torch.equal(ops.process_logits(x, h, lens, out=out, **kw), want) and torch.equal(out, want)
    before = room.clone()
    whole = torch.empty(B, V, device=DEV)
    for refused in (dict(out=bias), dict(out=room[:, V + 1:2 * V + 1]), dict(out=whole, bias=whole), dict(out=whole, bias=whole[3]), dict(out=whole, presence=whole[0, :B]),
                    dict(out=whole, allowed=whole.view(torch.int32)[:, :41])):
        with pytest.raises(RuntimeError, match="apart"):
            ops.process_logits(x, h, lens, **{**kw, **refused})
    with pytest.raises(RuntimeError, match="apart"):
        ops.process_logits(x, whole.view(torch.int32)[:, :40], lens, out=whole)
    assert torch.equal(room, before)
    assert torch.equal(ops.process_logits(x, h, lens, out=x, **kw), want)
