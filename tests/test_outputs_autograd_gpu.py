"""Results that a caller gives and that want gradients are refused, as torch refuses them for ``out=``: nothing could follow what is written there."""
import pytest
import torch

from daisy_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_results_that_want_gradients_are_refused():
    half = lambda *shape: torch.randn(*shape, device=DEV).bfloat16()      # noqa: E731
    k, v, table = half(3, 2, 16, 64), half(3, 2, 16, 64), torch.tensor([[1, 2]], dtype=torch.int32, device=DEV)
    x, pos = half(1, 2, 64), torch.tensor([3], dtype=torch.int32, device=DEV)
    for name in ("q_out", "k_out", "v_out"):
        out = half(1, 2, 64).requires_grad_()
        before = out.detach().clone()
        with pytest.raises(RuntimeError, match="no backward"):
            ops.paged_append(x, x, k, v, table, pos, q=x, **{name: out})
        assert torch.equal(out, before)
        with torch.no_grad():
            ops.paged_append(x, x, k, v, table, pos, q=x, **{name: out})
    out = half(1, 2, 64).requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        ops.paged_attention(x, k, v, table, pos, out=out)
    logits = torch.randn(2, 30, device=DEV)
    with pytest.raises(RuntimeError, match="no backward"):
        ops.process_logits(logits, out=torch.empty_like(logits).requires_grad_())
