"""What a window's sequences hold of the pool: a prompt all of its positions, until the sequence crosses into another page; then what a step sees."""
import pytest
import torch

from daisy_amd import PagedKVCache


def test_a_prompt_takes_all_of_its_pages_and_gives_them_back_at_the_next_page():
    c = PagedKVCache(L=1, sequences=2, H=1, D=64, pages=7, device="cpu", dtype=torch.bfloat16, page_size=16, max_len=400, window=20)
    assert c.admit([100]) == [0] and c.free_pages == 0
    with pytest.raises(RuntimeError, match="full"):
        c.admit([1])
    for n in range(100, 112):
        c.begin_step()
        assert c.free_pages == 0
        c.advance()
    c.begin_step()                       # position 112 is in another page: 93 to 112 are seen
    assert c.free_pages == 4 and [e for e, p in enumerate(c.page_table[0].tolist()) if p >= 0] == [5, 6, 7]
    assert c.admit([1]) == [1]
