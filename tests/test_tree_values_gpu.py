"""Values that are not finite in the tiles of a long context that every node sees whole: their channel is not finite for the nodes and the heads that share them, whatever kernel has
the columns, and nobody else's results change."""
import random

import pytest
import torch

from daisy_amd import ops
from test_paged_gpu import BF16, DEV, F16, gen, randn
from test_tree_gpu import cache_of, check, ints, trees

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("odd", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype,D,G,T", [(BF16, 128, 1, 7), (F16, 64, 4, 8), (BF16, 128, 8, 12), (F16, 64, 8, 40), (BF16, 256, 8, 8)])
@pytest.mark.parametrize("window", [None, 600])
def test_a_value_that_is_not_finite_deep_in_a_context(odd, dtype, D, G, T, window):
    print(f"tree value {odd} {dtype} D{D} G{G} T{T} window {window}", flush=True)
    rng, g = random.Random(T), gen(T)
    lens, H, page = [700, 650], 2, 32
    parents, masks = trees(T, 2, rng)
    k, v, table, rows = cache_of([(0, n + T) for n in lens], H, page, D, dtype, g)
    q = randn(g, 2, T, G * H, D, dtype=dtype)
    call = lambda: ops.paged_tree_attention(q, k, v, table, ints(lens), ints(masks), window=window)      # noqa: E731
    plain = call()
    check(plain, q, rows, lens, [T, T], masks, ops.ATTN_SCALE, "as it is", window)
    spot, channel, head = 400, 5, 1                      # (far from the context's end and from the window's edge)
    page_of = int(table[0, spot // page])
    v[page_of, head, spot % page, channel] = odd
    got = call()
    felt = torch.zeros_like(got, dtype=torch.bool)
    felt[0, :, head * G:(head + 1) * G, channel] = True
    assert not bool(torch.isfinite(got[felt]).any())
    assert torch.equal(got[~felt], plain[~felt])
