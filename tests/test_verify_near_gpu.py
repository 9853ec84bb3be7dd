"""``ops.verify_drafts`` where what a rejection leaves, ``max(p - q, 0)``, is a small part of ``p``: drafts whose probabilities are next to the target's.

The definition's walk (``test_verify_gpu.walk``, 64 bits) says how near the nearest of its decisions is, and cases nearer than 1e-5 of what is compared are left out; what the subtraction
leaves of ``p`` is no reason to be off by more: 64 bits hold ``p - q`` to 2^-53 of ``p``, 1e-9 of differences of 1e-7."""
import pytest
import torch

from daisy_amd import ops
from test_paged_gpu import BF16, DEV, F16, gen
from test_tree_gpu import ints
from test_verify_gpu import F32, check

pytestmark = pytest.mark.gpu


def near(B, T, V, eps, dtype=F32, temperature=0.8, kept=0, seed=0):
    """Stars whose first children (all but the last two) are tokens that the draft finds three times as likely as the target and that are rejected; the last ones are drawn from the draft.
    All other probabilities differ by about ``eps`` of themselves."""
    g = gen(seed)
    x = (torch.randn(B, T, V, generator=g, device=DEV) * 3).to(dtype)
    if kept:
        x = x.masked_fill(x < x.topk(kept, -1).values[..., -1:], -float("inf"))
    q = torch.softmax(x.double() / temperature + eps * torch.randn(B, T, V, generator=g, device=DEV, dtype=torch.float64), -1).float()
    accept = torch.rand(B, T, generator=g, device=DEV)
    tokens = torch.randint(V, (B, T), generator=g, device=DEV)
    for i in range(1, T):
        tokens[:, i] = (q[:, 0] / torch.empty(B, V, device=DEV).exponential_(generator=g)).argmax(-1)
    for i in range(1, max(2, T - 2)):
        at = tokens[:, i:i + 1]
        q[:, 0].scatter_(1, at, 3 * torch.softmax(x[:, 0].double() / temperature, -1).float().gather(1, at))
        accept[:, i] = 0.5 + 0.5 * accept[:, i]
    u = torch.rand(B, V, generator=g, device=DEV).clamp_(min=1e-6)
    return dict(logits=x, tokens=tokens, parents=ints([-1] + [0] * (T - 1)), nodes=None, temperature=temperature, accept=accept, noise=-torch.log(-torch.log(u)), draft=q)


@pytest.mark.parametrize("eps", [1e-7, 1e-6, 1e-5, 1e-4, 1e-2])
@pytest.mark.parametrize("T", [2, 4, 7])
@pytest.mark.parametrize("dtype,V", [(F32, 8192), (BF16, 5001), (F16, 50257)])
def test_what_is_left_of_a_draft_next_to_the_target(eps, T, dtype, V):
    print(f"verify near eps {eps} T{T} {dtype} V{V}", flush=True)
    B = 200 if V < 10000 else 40
    got = check(near(B, T, V, eps, dtype, seed=T), f"near, {eps}")
    assert bool((got[1] == 1).any())
    if T > 2:
        assert bool((got[1] == 2).any())


@pytest.mark.parametrize("eps", [1e-6, 1e-3])
@pytest.mark.parametrize("kept", [3, 40])
def test_what_is_left_behind_a_filter(eps, kept):
    print(f"verify near eps {eps} kept {kept}", flush=True)
    check(near(100, 4, 3001, eps, kept=kept, temperature=0.5, seed=kept), f"near, {kept} kept")
