"""A recorded step over a paged cache takes a token for every slot."""
import pytest
import torch

from daisy_amd import core
from test_core_gpu import DEV, _Core
from test_paged_model_gpu import paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("recorded", [False, True])
def test_one_token_is_not_every_slots(recorded):
    model = _Core(window=48).to(DEV).eval()
    cache = paged(model, 3)
    step = core.GraphedPagedStep(model, cache) if recorded else lambda tokens: core.step(model, tokens, cache)
    with torch.inference_mode():
        core.admit(model, [torch.arange(2, 2 + n, device=DEV) for n in (16, 9)], cache)
        for n in (1, 2, 4):
            with pytest.raises(AssertionError, match="does not match the cache"):
                step(torch.zeros(n, dtype=torch.long, device=DEV))
        assert cache.length(0) == 16 and cache.free_pages == 38, "nothing was taken for a step that was refused"
        step(torch.zeros(3, dtype=torch.long, device=DEV))
        with pytest.raises(AssertionError, match="does not match the cache"):
            step(torch.zeros(1, dtype=torch.long, device=DEV))
        assert cache.length(0) == 17
