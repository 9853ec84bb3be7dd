"""``Generator(window=W)`` bounds what the steps of ``generate_ragged`` see as it bounds those of ``generate_batch``: a ring of W rows beside the new
token where the model's window is wider, W positions where the model names none."""
import pytest
import torch

from daisy_amd import core
from daisy_amd.generate import Generator
from test_core_gpu import DEV, _close, _Core
from test_paged_model_gpu import paged

pytestmark = pytest.mark.gpu


def forced(model, window, prompt, tokens, ragged, **kw):
    """The scores that a generator draws from, one row a step, where ``tokens`` are what it draws."""
    gen = Generator(model, window=window, seed=3, device=DEV, dtype=torch.bfloat16, temperature=0.0)
    scores, left = [], list(tokens)

    def sample(x, *settings):
        scores.append(x[-1].float().clone())
        return left.pop(0).view(1)

    gen.sample = sample
    out = gen.generate_ragged([prompt], len(tokens), **kw) if ragged else gen.generate_batch(prompt[None], len(tokens), **kw)
    assert torch.equal(out[0], tokens)
    return torch.stack(scores), gen


@pytest.mark.parametrize("record_steps", [False, True])
@pytest.mark.parametrize("window,named", [(12, True), (20, True), (47, True), (48, True), (90, True), (12, False), (48, False)])
def test_a_window_below_the_models_bounds_the_ragged_loop_too(window, named, record_steps):
    model = _Core(window=48).to(DEV).eval()
    if not named:
        del model.attn_window_size
    g = torch.Generator(device=DEV).manual_seed(1)
    prompt = torch.randint(2, 96, (10,), generator=g, device=DEV)
    tokens = torch.randint(2, 96, (75,), generator=g, device=DEV)
    want, _ = forced(model, window, prompt, tokens, False)
    got, gen = forced(model, window, prompt, tokens, True, record_steps=record_steps)
    _close(got, want, f"window {window}")
    if window <= 20:
        wide, _ = forced(model, 48 if named else 90, prompt, tokens, False)
        assert float((wide - want).abs().max()) > 6e-2 * max(float(want.abs().max()), 1.0), "the window makes no difference here"
    seen = (min(window + 1, 48) if named else window) if window < 90 else 48
    assert gen._paged_cache.window == seen


def test_pages_behind_the_generators_window_go_back():
    """160 positions in a window of 20, pages of 64: two at a time."""
    model = _Core(window=48).to(DEV).eval()
    gen = Generator(model, window=20, seed=3, device=DEV, dtype=torch.bfloat16, temperature=0.0)
    prompts = [torch.arange(2, 2 + n, device=DEV) for n in (10, 1)]
    with torch.inference_mode():
        out = gen.generate_ragged(prompts, 150)
        assert gen._paged_cache.pages == 4
        assert torch.equal(gen.generate_ragged(prompts, 150, record_steps=True), out)
        # a pool that holds everything gives the same
        cache = paged(model, 2, pages=20, page_size=64, window=21)
        logits, _ = core.admit(model, prompts, cache)
        for n in range(149):
            assert torch.equal(gen._trim(logits)[:, :96].argmax(-1)[out[:, n] != 1], out[:, n][out[:, n] != 1])
            logits = core.step(model, out[:, n], cache, window=21)


def test_a_replaced_pool_is_given_up_first():
    model = _Core(window=48).to(DEV).eval()
    gen = Generator(model, window=48, seed=3, device=DEV, dtype=torch.bfloat16, temperature=0.0)
    gen.generate_ragged([torch.arange(2, 12, device=DEV)], 3, record_steps=True)
    import weakref
    import daisy_amd.generate as generate
    old, made = weakref.ref(gen._paged_cache), []
    real = generate.PagedKVCache

    def make(*args, **kw):
        made.append(old() is None and gen._paged_step is None)
        return real(*args, **kw)

    generate.PagedKVCache = make
    try:
        gen.generate_ragged([torch.arange(2, 12, device=DEV)] * 2, 3)
    finally:
        generate.PagedKVCache = real
    assert made == [True]


def test_a_window_of_a_call_is_for_paged_caches():
    from daisy_amd import KVCache
    model = _Core(window=48).to(DEV).eval()
    ring = KVCache(4, 1, 2, 48, 128, DEV, torch.bfloat16)
    with pytest.raises(ValueError, match="paged"):
        core.step(model, torch.zeros(1, dtype=torch.long, device=DEV), ring, window=20)
    cache = paged(model, 1, window=32)
    core.admit(model, [torch.arange(2, 12, device=DEV)], cache)
    with pytest.raises(ValueError, match="window must be positive"):
        core.step(model, torch.zeros(1, dtype=torch.long, device=DEV), cache, window=0)
    core.step(model, torch.zeros(1, dtype=torch.long, device=DEV), cache, window=32)      # the model's is 48
