"""The pool that the generator's ragged loop takes is enough for it, to the last step, and little more."""
import random

import torch

from daisy_amd import PagedKVCache
from daisy_amd.generate import _ragged_pages


def test_the_ragged_loops_pool_is_enough():
    rng = random.Random(0)
    for _ in range(150):
        size, new, window = 16, rng.randrange(1, 120), rng.choice([1, 2, 15, 16, 17, 18, 33, 40, 64, 200, 10 ** 6])
        lengths = [rng.randrange(1, 90) for _ in range(rng.randrange(1, 5))]
        pages = _ragged_pages(lengths, new, window, size)
        cache = PagedKVCache(L=1, sequences=len(lengths), H=1, D=16, pages=pages, device="cpu", dtype=torch.bfloat16, page_size=size, max_len=max(lengths) + new,
                             window=window)
        cache.admit(lengths)
        for _ in range(new - 1):
            cache.begin_step()
            cache.advance()
    assert _ragged_pages([10, 1], 150, 21, 64) == 4 and _ragged_pages([1000], 8, 21, 64) == 16 and _ragged_pages([10, 1], 3, 10 ** 6, 64) == 2
