"""Where the steps of a paged cache end: at the rows of the rotary tables, which the host knows, with the cache as it was; and what the cache's
status word says once it has been read."""
import types

import pytest
import torch

from daisy_amd import CausalSelfAttention, PagedKVCache, core


def cpu_model(rows):
    """As much of a model as a step looks at ahead of its first kernel."""
    attn = CausalSelfAttention(128, 2, 64, max_seq_len=rows)
    return types.SimpleNamespace(blocks=[types.SimpleNamespace(attn=attn), types.SimpleNamespace(attn=None)])


def cpu_cache(**kw):
    return PagedKVCache(**{**dict(L=2, sequences=3, H=2, D=64, pages=12, device="cpu", dtype=torch.bfloat16, page_size=16, max_len=64), **kw})


@pytest.mark.parametrize("recorded", [False, True])
def test_a_step_past_the_rotary_tables_is_refused_on_the_host(recorded):
    model, cache = cpu_model(32), cpu_cache()
    step = core.GraphedPagedStep(model, cache) if recorded else lambda tokens: core.step(model, tokens, cache)
    cache.admit([5, 32])
    before = cache.page_table.clone(), cache.free_pages, cache.positions.clone()
    with pytest.raises(AssertionError, match="Rotary buffers too small 32 < 33"):
        step(torch.zeros(3, dtype=torch.long))
    assert torch.equal(cache.page_table, before[0]) and cache.free_pages == before[1] and torch.equal(cache.positions, before[2])
    assert (cache.length(0), cache.length(1)) == (5, 32)


def test_a_status_word_that_was_reported_is_clear():
    cache = cpu_cache()
    cache.check()
    cache.status.fill_(1)
    with pytest.raises(RuntimeError, match="rotary tables"):
        cache.check()
    cache.check()
    assert cache.status.tolist() == [0]


@pytest.mark.gpu
@pytest.mark.parametrize("recorded", [False, True])
def test_the_other_sequences_go_on_when_the_one_at_the_end_is_released(recorded):
    from test_core_gpu import DEV, _Core
    from test_paged_model_gpu import paged
    model = _Core(window=48, max_seq_len=32).to(DEV).eval()
    g = torch.Generator(device=DEV).manual_seed(0)
    prompts = [torch.randint(2, 96, (n,), generator=g, device=DEV) for n in (30, 4)]
    cache = paged(model, 2)
    step = core.GraphedPagedStep(model, cache) if recorded else lambda tokens: core.step(model, tokens, cache)
    tokens = torch.tensor([5, 7], device=DEV)
    with torch.inference_mode():
        core.admit(model, prompts, cache)
        for _ in range(2):
            assert bool(torch.isfinite(step(tokens)).all())
        with pytest.raises(AssertionError, match="Rotary buffers too small 32 < 33"):
            step(tokens)
        assert (cache.length(0), cache.length(1)) == (32, 6) and cache.positions.tolist() == [32, 6]
        cache.release(0)
        for _ in range(3):
            assert bool(torch.isfinite(step(tokens)[1]).all())
        cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("record_steps", [False, True])
def test_the_generator_refuses_to_run_past_the_rotary_tables(record_steps):
    """The last token that is drawn is not run through the model: 30 + 3 tokens need positions 0 to 31."""
    from daisy_amd.generate import Generator
    from test_core_gpu import DEV, _Core
    model = _Core(window=48, max_seq_len=32).to(DEV).eval()
    gen = Generator(model, window=48, seed=3, device=DEV, dtype=torch.bfloat16, temperature=0.0)
    g = torch.Generator(device=DEV).manual_seed(0)
    prompts = [torch.randint(2, 96, (n,), generator=g, device=DEV) for n in (30, 4)]
    assert gen.generate_ragged(prompts, 3, record_steps=record_steps).shape == (2, 3)
    with pytest.raises(AssertionError, match="Rotary buffers too small 32 < 33"):
        gen.generate_ragged(prompts, 4, record_steps=record_steps)
    assert gen.generate_ragged(prompts[1:], 29, record_steps=record_steps).shape == (1, 29)


@pytest.mark.gpu
def test_the_generator_reads_the_status_word(monkeypatch):
    """A page that is lost on the device while the ragged loop runs is an error of that call, and of no later one."""
    from daisy_amd.generate import Generator
    from test_core_gpu import DEV, _Core
    model = _Core(window=48).to(DEV).eval()
    gen = Generator(model, window=48, seed=3, device=DEV, dtype=torch.bfloat16, temperature=0.0)
    prompts = [torch.arange(2, 2 + n, device=DEV) for n in (30, 4)]
    want = gen.generate_ragged(prompts, 4)
    real = core.step

    def step(model, tokens, cache, **kw):
        cache.page_table[1, 0] = -1
        return real(model, tokens, cache, **kw)

    with monkeypatch.context() as m:
        m.setattr(core, "step", step)
        with pytest.raises(RuntimeError, match="no page of the pool"):
            gen.generate_ragged(prompts, 4)
    assert torch.equal(gen.generate_ragged(prompts, 4), want)
