"""Temperatures of ``ops.verify_drafts``: a number counts as it is given, rows in fp32; rows that are not finite, which a number may not be, leave node 0 alone with nothing behind it.

A child that is 68 below the likeliest token has p = exp(-68 / t).  At t = 0.8 that is exp(-85); with t rounded to fp32 (0.8 (1 + 1.49e-8)) it is 85 * 1.49e-8 = 1.27e-6 of itself more.  The
kernel's own rounding is that of one fp32 exponential, 2^-23 = 1.2e-7 (the other token's is 1 exactly), and accept's is 2^-24: numbers 5e-7 of p below and above it decide for sure."""
import math

import pytest
import torch

from daisy_amd import ops
from test_paged_gpu import BF16, DEV, F16
from test_tree_gpu import ints
from test_verify_gpu import F32, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("t", [0.8, 0.85, 1.1, 1.3])
def test_a_temperature_counts_as_it_is_given(t, draft):
    print(f"verify temperature {t} draft {draft}", flush=True)
    below = round(85 * t)
    p = math.exp(-below / t)
    p /= 1 + p
    logits = torch.tensor([0.0, -float(below)], device=DEV).expand(2, 2, 2).contiguous()
    accept = torch.tensor([[0.0, p * (1 - 5e-7)], [0.0, p * (1 + 5e-7)]], dtype=torch.float64).to(F32).to(DEV)
    noise = torch.zeros(2, 2, device=DEV)
    one = torch.ones(2, 2, 2, device=DEV) if draft else None      # (accepted where accept * 1 < p)
    call = lambda temperature: ops.verify_drafts(logits, ints([[0, 1], [0, 1]]), ints([-1, 0]), temperature=temperature, accept=accept, noise=noise, draft=one)      # noqa: E731
    assert call(t)[1].tolist() == [2, 1]
    # rows have fp32's: p moves as the rounding does, by more than the margin for each of these
    moved = below / t * (float(torch.tensor(t, dtype=F32)) / t - 1)
    assert abs(moved) > 1e-6
    assert call(torch.full((2,), t, device=DEV))[1].tolist() == ([2, 2] if moved > 0 else [1, 1])


def test_numbers_that_fp32_rounds_to_zero_are_temperatures():
    logits = torch.tensor([0.0, 0.0, -1e-30], device=DEV).expand(1, 2, 3).contiguous()
    args = (logits, ints([[0, 2]]), ints([-1, 0]))
    for t in (1e-50, 1e-310):
        path, counts, token = ops.verify_drafts(*args, temperature=t, accept=torch.zeros(1, 2, device=DEV), noise=torch.tensor([[0.0, 1.0, 9.0]], device=DEV))
        assert counts[0] == 1 and token[0] == 1, t      # (the two likeliest are alike, and the noise tells them apart)
    assert ops.verify_drafts(*args, temperature=0.0)[2][0] == 0
    with pytest.raises(RuntimeError, match="finite in fp32"):
        ops.verify_drafts(*args, temperature=1e39, accept=torch.zeros(1, 2, device=DEV), noise=torch.zeros(1, 3, device=DEV))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("V", [7, 3000])
def test_rows_whose_temperature_is_not_finite_have_no_followers(dtype, draft, V):
    print(f"verify temperatures {dtype} draft {draft} V{V}", flush=True)
    odd = {1: float("inf"), 4: float("nan"), 6: -float("nan"), 7: float("inf")}
    s = make(10, 6, V, dtype, shape="star", draft=draft, seed=V)
    t = torch.full((10,), 0.8, device=DEV)
    t[0], t[2], t[9] = 0.0, -1.0, -float("inf")
    want = check(dict(s, temperature=t), "finite")
    for row, x in odd.items():
        t[row] = x
    path, counts, token = ops.verify_drafts(s["logits"], s["tokens"], s["parents"], temperature=t, accept=s["accept"], noise=s["noise"], draft=s["draft"])
    for b in range(10):
        if b in odd:
            assert path[b].tolist() == [0, -1, -1, -1, -1, -1] and counts[b] == 1 and token[b] == -1, b
        else:
            assert torch.equal(path[b], want[0][b]) and counts[b] == want[1][b] and token[b] == want[2][b], b


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("kept", [0, 5])
def test_the_smallest_and_largest_temperatures(dtype, draft, kept):
    """3e38: all that a filter has left is alike; 1e-40: nothing but the likeliest counts."""
    s = make(12, 5, 900, dtype, draft=draft, kept=kept, seed=3)
    t = torch.tensor([3e38, 1e-40, 1e30, 1e-30, 1.0, 2e-38] * 2, device=DEV)
    check(dict(s, temperature=t), "extremes")
