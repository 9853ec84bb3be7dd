"""The precision of ``ops.paged_attention``: its probabilities reach the matrix cores in two parts, so that a result is off by its own rounding and by fp32 sums;
and its joins, each of their forms, against the definition in 64 bits.

Tolerances.  E is half a step of a type.  The second part of a probability is rounded to E of itself, E^2 of the probability; the result to E |o|, or half of fp16's smallest step.  Sums of fp32 in a
chain of n terms: n 2^-24 of the terms' magnitudes, in numerator and denominator each; A is sum p |v| / sum p."""
import math

import pytest
import torch

from daisy_amd import ops
from test_paged_gpu import BF16, DEV, F16, attend_exact, gen, half_step, make_cache, randn

pytestmark = pytest.mark.gpu


def paged_from(keys, values, page, g):
    """Pages and table of one sequence per row of ``keys``, ``values`` [B, n, H, D], all of one length."""
    B, n, H, D = keys.shape
    width = -(-n // page)
    table = torch.randperm(B * width, generator=g, device=DEV).view(B, width).to(torch.int32)
    k = torch.full((B * width, H, page, D), float("nan"), dtype=keys.dtype, device=DEV)
    v = torch.full_like(k, float("nan"))
    t = torch.arange(n, device=DEV)
    for b in range(B):
        k[table[b, t // page].long(), :, t % page], v[table[b, t // page].long(), :, t % page] = keys[b], values[b]
    return k, v, table


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,n", [(64, 2), (64, 20), (128, 3), (128, 32), (128, 150), (256, 5), (256, 64)])
def test_probabilities_are_not_rounded_to_the_caches_type(dtype, D, n):
    """A query with one channel: scores are single products, exact, below 3 in magnitude, so that an exponent is off by fp32's rounding of
    numbers below 2^4 twice and by exp2's own 2^-22, less than 2e-6 together.  Tolerance E |o| + (E^2 + 2 (2e-6 + 2 n 2^-24)) A + half of the smallest step.  With
    probabilities in one part the same formula, on the CPU, leaves it."""
    g = gen(D + n)
    B, H = 8, 4
    keys, values = randn(g, B, n, H, D, dtype=dtype), randn(g, B, n, H, D, dtype=dtype)
    keys[..., 0] = (torch.rand(B, n, H, generator=g, device=DEV) * 6 - 3).to(dtype)
    q = torch.zeros(B, H, D, dtype=dtype, device=DEV)
    q[..., 0] = 1
    k, v, table = paged_from(keys, values, 16, g)
    o = ops.paged_attention(q, k, v, table, torch.full((B,), n, dtype=torch.int32, device=DEV), scale=1.0).double().cpu()
    s, vals, E = keys[..., 0].double().cpu(), values.double().cpu(), half_step(dtype)
    top, head = s.amax(1, keepdim=True), 9.0 if dtype == F16 else 0.0      # the reference of the exponentials: the largest probability is 2^head
    p = torch.exp2((s - top) / math.log(2.0) + head)
    total = p.sum(1)[..., None]
    want, A = (p[..., None] * vals).sum(1) / total, (p[..., None] * vals.abs()).sum(1) / total
    tol = E * want.abs() + (E * E + 2 * (2e-6 + 2 * n * 2.0 ** -24)) * A + torch.finfo(dtype).smallest_normal * E
    err = (o - want).abs()
    assert bool((err <= tol).all()), f"{err.max().item():.3e}, {(err / tol).max().item():.2f} of what it may be"
    one_part = (p.to(dtype).double()[..., None] * vals).sum(1) / total
    assert not bool(((one_part.to(dtype).double() - want).abs() <= tol).all()), "this case would not show probabilities in one part"


def check_two_parts(o, q, rows, scale, what):
    """E |o| + (E^2 + 5e-4) A: scores of up to 256 products of normal numbers move an exponent by less than 256 * 2^-24 * 96 * 0.12 = 1.8e-4, which numerator and
    denominator feel; chains of sums are a thousand terms at most, 6e-5 each."""
    want, A = attend_exact(q, rows, scale)
    E = half_step(o.dtype)
    err, tol = (o.double() - want).abs(), E * want.abs() + (E * E + 5e-4) * A + 1e-7
    assert torch.isfinite(o).all(), what
    assert bool((err <= tol).all()), f"{what}: {err.max().item():.3e}, {(err / tol).max().item():.2f} of what it may be"


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lens,H,G,D", [
    ([5000], 1, 8, 128),              # 40 parts, 32 channels at a time: fewer helpers than 16 would make pieces
    ([10000], 1, 16, 128),            # 79 parts of 16 heads: 64 < parts <= 128
    ([5000, 30, 0], 2, 8, 128), ([700, 64, 3], 1, 17, 256), ([3000, 5, 900], 2, 4, 128),
    ([9000], 1, 16, 256), ([9000, 17], 1, 17, 256), ([2000, 1], 2, 16, 256),      # the widest sums of a workgroup
    ([4096] * 3, 4, 8, 128), ([20001, 3], 2, 1, 64), ([400] * 9, 3, 2, 128), ([100] * 70, 1, 1, 64)])
def test_every_form_of_the_join(dtype, lens, H, G, D):
    print(f"paged attention {dtype} {lens[:4]} H{H} G{G} D{D}", flush=True)
    g = gen(len(lens) + D + G)
    k, v, table, rows = make_cache(lens, H, 32, D, dtype, g)
    q = randn(g, len(lens), H * G, D, dtype=dtype)
    lt = torch.tensor(lens, dtype=torch.int32, device=DEV)
    o = ops.paged_attention(q, k, v, table, lt, scale=0.12)
    check_two_parts(o, q, rows, 0.12, f"{lens[:4]} H{H} G{G} D{D}")
    space = torch.full((ops.paged_attention_workspace_bytes(len(lens), H * G, H, D, table.shape[1], 32),), 0x7f, dtype=torch.uint8, device=DEV)
    for _ in range(3):
        assert torch.equal(ops.paged_attention(q, k, v, table, lt, scale=0.12, workspace=space), o)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_a_value_that_is_not_finite_spoils_its_own_channel_only(dtype, value):
    g = gen(21)
    lens, H, G, D = [300, 2000, 9], 2, 2, 128
    k, v, table, rows = make_cache(lens, H, 16, D, dtype, g)
    q = randn(g, 3, H * G, D, dtype=dtype)
    lt = torch.tensor(lens, dtype=torch.int32, device=DEV)
    want = ops.paged_attention(q, k, v, table, lt, scale=0.12)
    for b, t, h, d in ((1, 700, 1, 77), (2, 8, 0, 0)):
        v[int(table[b, t // 16]), h, t % 16, d] = value
    got = ops.paged_attention(q, k, v, table, lt, scale=0.12)
    spoiled = torch.zeros_like(got, dtype=torch.bool)
    spoiled[1, G:, 77] = True
    spoiled[2, :G, 0] = True
    assert not bool(torch.isfinite(got[spoiled]).any()) and torch.equal(got[~spoiled], want[~spoiled])
