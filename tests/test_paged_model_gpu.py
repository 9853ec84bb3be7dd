"""Sequences of unequal length through a small model: ``core.admit``, ``core.step`` and ``core.GraphedPagedStep`` over a ``PagedKVCache``, the generator's
ragged batches, and its penalties, biases and masks.  The model is that of the cache-aware glue's tests; what each sequence gives alone through the ring cache is
the reference (bf16 activations rounded along two routes: the tolerance of those tests)."""
import pytest
import torch

from daisy_amd import PagedKVCache, core, ops
from daisy_amd.generate import Generator
from test_core_gpu import DEV, _close, _Core

pytestmark = pytest.mark.gpu


def model_and_prompts(lengths, window=48, D=128, seed=0):
    model = _Core(window=window, D=D, H=256 // D).to(DEV).eval()
    g = torch.Generator(device=DEV).manual_seed(seed)
    return model, [torch.randint(2, 96, (n,), generator=g, device=DEV) for n in lengths], g


def paged(model, sequences, pages=40, page_size=16, max_len=300, dtype=torch.bfloat16, window=None):
    return PagedKVCache(L=4, sequences=sequences, H=model.attn_num_heads, D=model.attn_head_dim, pages=pages, device=DEV, dtype=dtype, page_size=page_size,
                        max_len=max_len, window=window)


def alone(model, prompt, tokens):
    """Logits of the prompt and of every step, one sequence through the ring cache."""
    from daisy_amd import KVCache
    ring = KVCache(4, 1, model.attn_num_heads, model.attn_window_size, model.attn_head_dim, DEV, torch.bfloat16)
    out = [core.prefill(model, prompt[None], ring)[0][0]]
    return out + [core.step(model, t[None], ring)[0] for t in tokens]


@pytest.mark.parametrize("D,dtype,window,keep", [(128, torch.bfloat16, 48, None), (64, torch.bfloat16, 48, 48), (128, torch.float16, 20, 32)])
def test_unequal_sequences_give_what_each_gives_alone(D, dtype, window, keep):
    lengths = [1, 70, 17, 48]
    model, prompts, g = model_and_prompts(lengths, window, D)
    cache = paged(model, 5, dtype=dtype, window=keep)
    with torch.inference_mode():
        logits, slots = core.admit(model, prompts, cache)
        assert slots == [0, 1, 2, 3]
        got = [[row] for row in logits]
        tokens = torch.randint(2, 96, (20, 5), generator=g, device=DEV)
        for t in tokens:
            for i, row in enumerate(core.step(model, t, cache)[:4]):
                got[i].append(row)
        cache.check()
        for i, prompt in enumerate(prompts):
            for n, (a, b) in enumerate(zip(got[i], alone(model, prompt, tokens[:, i]))):
                _close(a, b, f"sequence {i}, step {n}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_step_in_one_call_and_kernel_by_kernel_are_the_same(dtype, monkeypatch):
    from daisy_amd import _lib
    model, prompts, g = model_and_prompts([9, 40, 3])
    a, b = paged(model, 4, dtype=dtype), paged(model, 4, dtype=dtype)
    native = _lib.native()

    class WithoutTheCall:
        def __getattr__(self, name):
            return (lambda *args: None) if name == "paged_layer_step" else getattr(native, name)

    with torch.inference_mode():
        for c in (a, b):
            core.admit(model, prompts, c)
        for _ in range(4):
            tokens = torch.randint(2, 96, (4,), generator=g, device=DEV)
            one = core.step(model, tokens, a)
            with monkeypatch.context() as m:
                m.setattr(_lib, "native", lambda: WithoutTheCall())
                other = core.step(model, tokens, b)
            assert torch.equal(one[:3], other[:3])


def test_sequences_come_and_go_between_recorded_steps():
    """The recorded step follows admissions and releases, bit for bit as the eager one, and slots that are free disturb nobody."""
    model, prompts, g = model_and_prompts([5, 33, 12, 20, 7])
    a, b = paged(model, 3), paged(model, 3)
    with torch.inference_mode():
        recorded = core.GraphedPagedStep(model, a)
        for c in (a, b):
            core.admit(model, prompts[:2], c)
        for n in range(12):
            print(f"recorded step {n}", flush=True)
            tokens = torch.randint(2, 96, (3,), generator=g, device=DEV)
            x, y = recorded(tokens), core.step(model, tokens, b)
            live = [s for s in range(3) if b.length(s) is not None]
            torch.cuda.synchronize()
            assert torch.equal(x[live], y[live]), n
            for c in (a, b):
                if n == 2:
                    core.admit(model, prompts[2:3], c)
                if n == 5:
                    c.release(0)
                if n == 7:
                    core.admit(model, prompts[3:4], c)
        recorded.check()
        assert a.positions.tolist() == b.positions.tolist() and a._length == b._length
        # a sequence that came late gives what it gives alone
        late = paged(model, 3)
        want = core.admit(model, prompts[4:], late)[0]
        b.release(1)
        _close(core.admit(model, prompts[4:], b)[0], want, "a late prompt")


def test_a_failed_admission_leaves_the_cache_as_it_was():
    model, prompts, _ = model_and_prompts([5, 600])
    cache = paged(model, 2, pages=60, max_len=800)
    with pytest.raises(AssertionError, match="Rotary buffers too small"):
        core.admit(model, prompts, cache)
    assert cache.free_pages == 60 and cache.length(0) is None
    blocks = list(model.blocks)
    del blocks[1].attn
    blocks[1].attn = object()      # an attention layer of another kind
    with pytest.raises(ValueError, match="take its pages"):
        core.admit(model, prompts[:1], cache)
    with pytest.raises(ValueError, match="take its pages"):
        core.step(model, torch.zeros(2, dtype=torch.long, device=DEV), cache)


def test_a_window_wider_than_the_cache_keeps_is_refused():
    model, prompts, _ = model_and_prompts([5])
    cache = paged(model, 1, window=32)
    with torch.inference_mode():
        core.admit(model, prompts, cache)
        with pytest.raises(ValueError, match="keeps 32 positions"):
            core.step(model, prompts[0][:1], cache)


# ---------------------------------------------------------------------------------------------------------------
# the generator
# ---------------------------------------------------------------------------------------------------------------
def generator(model, **kw):
    args = dict(window=48, seed=3, device=DEV, dtype=torch.bfloat16, temperature=0.0)
    args.update(kw)
    return Generator(model, **args)


def test_ragged_prompts_follow_the_loop_written_out():
    model, prompts, _ = model_and_prompts([3, 40, 21])
    gen = generator(model, repetition_penalty=1.3)
    with torch.inference_mode():
        out = gen.generate_ragged(prompts, 12)
        assert out.shape == (3, 12)
        assert torch.equal(gen.generate_ragged(prompts, 12, record_steps=True), out), "recorded steps change the tokens"
        assert torch.equal(gen.generate_ragged(prompts, 12), out), "a cache that is used again changes the tokens"
        cache = paged(model, 3)
        logits, _ = core.admit(model, prompts, cache)
        seen = [p.tolist() for p in prompts]
        done = [False] * 3
        for _ in range(12):
            token = []
            for i in range(3):
                told = torch.tensor(seen[i][-128:], device=DEV)[None]
                scores = ops.process_logits(logits[i:i + 1].bfloat16()[:, :96], told, repetition=1.3, half_life=140.0, cap=3.0)
                t = 1 if done[i] else int(scores.argmax())
                done[i] |= t == 1
                seen[i].append(t)
                token.append(t)
            logits = core.step(model, torch.tensor(token, device=DEV), cache)
        assert out.tolist() == [s[-12:] for s in seen]
        short = gen.generate_ragged(prompts[:1], 1)
        assert short.tolist() == [[seen[0][3]]]


def test_presence_and_frequency_penalties_biases_and_masks_reach_every_loop():
    model, prompts, _ = model_and_prompts([9, 9])
    both = torch.stack(prompts)
    with torch.inference_mode():
        # a bias that decides
        gen = generator(model, logit_bias={17: 1e4})
        assert gen.generate_batch(both, 3).tolist() == [[17] * 3] * 2 and gen.generate_ragged(prompts, 3).tolist() == [[17] * 3] * 2
        assert [int(t) for t in gen.generate(prompts[0], 3)] == [17] * 3
        # a frequency penalty above every difference of the logits: no token twice
        gen = generator(model, frequency_penalty=1e3, logit_bias=torch.zeros(96))
        for row in (*gen.generate_batch(both, 8).tolist(), *gen.generate_ragged(prompts, 8).tolist(), [int(t) for t in gen.generate(prompts[0], 8)]):
            row = row[:row.index(1)] if 1 in row else row
            assert len(set(row)) == len(row)
        # a mask that counts: after n tokens only token 2 + n may follow
        def next_in_line(seen, lens):
            keep = torch.zeros(seen.size(0), 96, dtype=torch.bool, device=DEV)
            return keep.scatter_(1, lens.long()[:, None] % 90 + 2, True)
        gen = generator(model, allowed_tokens=next_in_line, temperature=1.0, presence_penalty=0.5)
        want = [11, 12, 13, 14]
        assert gen.generate_batch(both, 4).tolist() == [want] * 2 and gen.generate_ragged(prompts, 4).tolist() == [want] * 2
        assert [int(t) for t in gen.generate(prompts[0], 4)] == want
        # bits, and None for no mask
        bits = ops.pack_allowed(torch.arange(96, device=DEV) == 33)
        assert generator(model, allowed_tokens=lambda seen, lens: bits).generate_batch(both, 2).tolist() == [[33] * 2] * 2
        plain, none = generator(model, presence_penalty=0.0), generator(model, allowed_tokens=lambda seen, lens: None)
        assert torch.equal(none.generate_batch(both, 4), plain.generate_batch(both, 4))
        # nothing may follow after the second token of the first row: it ends, the other goes on
        def two(seen, lens):
            keep = torch.ones(seen.size(0), 96, dtype=torch.bool, device=DEV)
            keep[:, 1] = False
            keep[:1] &= (lens[:1, None] < 11)
            return keep
        for temperature, top_p in ((0.0, None), (1.0, 0.9)):
            gen = generator(model, allowed_tokens=two, temperature=temperature, top_p=top_p)
            for out in (gen.generate_batch(both, 5), gen.generate_ragged(prompts, 5)):
                assert (out[0] == 1).tolist() == [False, False, True, True, True] and not bool((out[1] == 1).any())
            assert len([t for t in gen.generate(prompts[0], 5)]) == 2
    with pytest.raises(ValueError, match="token 96"):
        generator(model, logit_bias={96: 1.0})
    gen = generator(model, presence_penalty=1.0)
    gen.apply_repetition_penalty = lambda logits, recent, strength, one: logits
    with pytest.raises(ValueError, match="does not combine"):
        gen.generate_batch(both, 2)
