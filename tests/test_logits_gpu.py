"""``ops.process_logits`` against its definition in 64 bits.

Tolerances.  A weight is one exp2 (2^-22 of it) and a rounding to 2^-31; their sum is exact, the power ``min(w, cap) log2 r`` is off by 2^-21 of itself and by
2^-30 n, the exp2 of it by 2^-22: together 2^-21 (1 + |power|) of ``x s``.  Each of the three sums rounds to 2^-24 of its terms' magnitudes, the store to half a
step of the value, or, below the type's normal numbers, to half of its smallest step: eps / 2 of the smallest normal number (fp16: 2^-25)."""
import math

import pytest
import torch

from daisy_amd import ops
from daisy_amd.generate import penalise_repeats

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def exact(x, history=None, lens=None, repetition=1.0, half_life=None, cap=None, presence=0.0, frequency=0.0, lookback=None, bias=None, allowed=None):
    """(y, tolerance) by loops over the tokens of the history, fp64 on the CPU."""
    E, least = torch.finfo(x.dtype).eps / 2, torch.finfo(x.dtype).smallest_normal
    x = x.double().cpu()
    B, V = x.shape
    of = lambda t, b: float(t[b]) if isinstance(t, torch.Tensor) else float(t)      # noqa: E731
    y, tol = x.clone(), torch.zeros_like(x)
    for b in range(B):
        if history is not None:
            n = history.shape[1] if lens is None else max(0, min(int(lens[b]), history.shape[1]))
            told = history[b, :n].tolist()
            told = told[max(0, n - (lookback if lookback is not None else n)):]
            count, weight = {}, {}
            for age, v in zip(range(len(told), 0, -1), told):
                if 0 <= v < V:
                    count[v] = count.get(v, 0) + 1
                    weight[v] = weight.get(v, 0.0) + (2.0 ** (-age / half_life) if half_life else 1.0)
            for v, c in count.items():
                power = min(weight[v], cap if cap is not None else math.inf) * math.log2(of(repetition, b))
                z = float(x[b, v]) * 2.0 ** (-power if x[b, v] > 0 else power)
                off = of(frequency, b) * c + of(presence, b)
                y[b, v] = z - off
                tol[b, v] = 2 ** -21 * (1 + abs(power)) * abs(z) + 2 ** -23 * (abs(z) + abs(off))
        if bias is not None:
            row = (bias if bias.dim() == 1 else bias[b]).double().cpu()
            tol[b] += 2 ** -23 * (y[b].abs() + row.abs())
            y[b] += row
        if allowed is not None:
            words = (allowed if allowed.dim() == 1 else allowed[b]).cpu().long()
            bits = (words[:, None] >> torch.arange(32)) & 1
            y[b, bits.flatten()[:V] == 0] = -math.inf
    return y, tol + E * y.abs().nan_to_num(posinf=0.0, neginf=0.0) + E * float(least) + 1e-30


def check(got, x, *args, **kw):
    want, tol = exact(x, *args, **kw)
    got = got.double().cpu()
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    err = (got - want).abs()[~inf]
    assert bool((err <= tol[~inf]).all()), f"{err.max().item():.3e}, {(err / tol[~inf]).max().item():.2f} of what it may be"


def logits(g, B, V, dtype=F32):
    return (torch.randn(B, V, generator=g, device=DEV) * 4).to(dtype)


def history(g, B, T, V, dtype=torch.int64):
    return (torch.rand(B, T, generator=g, device=DEV).pow(3) * V).to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,V,T", [(1, 1, 1), (1, 3, 5), (2, 31, 7), (3, 32, 0), (3, 33, 40), (2, 1023, 200), (1, 1024, 128), (2, 1025, 3), (5, 4099, 1000), (1, 50257, 128),
                                   (300, 2049, 17), (70, 8191, 33)])
@pytest.mark.parametrize("tokens", [torch.int64, torch.int32])
def test_everything_at_once(dtype, B, V, T, tokens):
    print(f"logits {dtype} B{B} V{V} T{T} {tokens}", flush=True)
    g = gen(B + V + T)
    x, h = logits(g, B, V, dtype), history(g, B, T, V, tokens)
    lens = torch.randint(0, T + 1, (B,), generator=g, device=DEV).to(torch.int32)
    lens[0] = T
    rows = lambda lo, hi: lo + (hi - lo) * torch.rand(B, generator=g, device=DEV)      # noqa: E731
    kw = dict(repetition=rows(0.8, 1.5), cap=2.0, presence=rows(-0.5, 0.5), frequency=rows(-0.1, 0.1), bias=torch.randn(V, generator=g, device=DEV),
              allowed=torch.randint(-2 ** 31, 2 ** 31, (B, -(-V // 32)), generator=g, device=DEV).to(torch.int32))
    got = ops.process_logits(x, h, lens, **kw)
    assert got.dtype == dtype and got.shape == x.shape
    check(got, x, h, lens, **kw)
    assert torch.equal(got, ops.process_logits(x, h, lens, **kw))


@pytest.mark.parametrize("half_life,cap,lookback", [(140.0, 3.0, 128), (None, 1.0, None), (None, None, None), (5.0, None, 40), (1000.0, 0.5, None), (None, 0.0, 3), (20.0, 2.0, 0)])
def test_repetition_decay_cap_and_lookback(half_life, cap, lookback):
    g = gen(7)
    x, h = logits(g, 3, 700), history(g, 3, 300, 60)
    kw = dict(repetition=1.3, half_life=half_life, cap=cap, lookback=lookback)
    check(ops.process_logits(x, h, **kw), x, h, **kw)


def test_the_generators_penalty():
    """``penalise_repeats`` in fp32 computes weights, powers and quotients in as many roundings: twice the tolerance of one side."""
    g = gen(8)
    x, h = logits(g, 4, 5000), history(g, 4, 128, 300)
    want = penalise_repeats(x, h, torch.tensor(1.2, device=DEV))
    got = ops.process_logits(x, h, repetition=1.2, half_life=140.0, cap=3.0, lookback=128)
    _, tol = exact(x, h, repetition=1.2, half_life=140.0, cap=3.0, lookback=128)
    assert bool(((got - want).abs().cpu() <= 2 * tol.float() + 2 ** -20 * want.abs().cpu()).all())


def test_one_row_settings_as_numbers_and_single_parts():
    g = gen(9)
    x, h = logits(g, 1, 3001)[0], history(g, 1, 50, 3001)[0]
    for kw in (dict(presence=0.7), dict(frequency=-0.3), dict(repetition=2.0, cap=1.0)):
        got = ops.process_logits(x, h, **kw)
        assert got.shape == x.shape
        check(got[None], x[None], h[None], **kw)
    b = torch.randn(3001, generator=g, device=DEV)
    assert torch.equal(ops.process_logits(x, bias=b), x + b)
    keep = torch.rand(3001, generator=g, device=DEV) < 0.3
    assert torch.equal(ops.process_logits(x, allowed=ops.pack_allowed(keep)), torch.where(keep, x, -math.inf))
    assert torch.equal(ops.process_logits(x), x)


def test_masked_places_may_hold_anything():
    """NaN and infinities under a clear bit become -inf; the rest follows the arithmetic; a row without a set bit is -inf throughout."""
    x = torch.tensor([[math.nan, math.inf, -math.inf, 1.0, math.nan, math.inf, -math.inf, -1.0]], device=DEV).repeat(2, 1)
    h = torch.tensor([[0, 1, 2, 3, 4, 5, 6, 7]], device=DEV).repeat(2, 1)
    keep = torch.tensor([[0, 0, 0, 0, 1, 1, 1, 1], [0] * 8], device=DEV).bool()
    got = ops.process_logits(x, h, repetition=2.0, allowed=ops.pack_allowed(keep))
    assert bool((got[0, :4] == -math.inf).all() and (got[1] == -math.inf).all())
    assert math.isnan(got[0, 4]) and got[0, 5] == math.inf and got[0, 6] == -math.inf and got[0, 7] == -2.0


@pytest.mark.parametrize("repetition", [1.3, 0.7, 1.0])
def test_powers_beyond_the_range_of_32_bits(repetition):
    """A token that came hundreds of times has a power of hundreds: zero stays zero, -inf stays -inf, the others end at zero or an infinity."""
    values = torch.tensor([[0.0, -math.inf, math.inf, 5.0, -5.0, 1e-20, -1e-20, 1e30, -1e30]], device=DEV)
    n = values.shape[1]
    for times in (100, 300, 400, 1000, 14000):
        h = torch.arange(n, device=DEV).repeat(times)[None]
        got = ops.process_logits(values, h, repetition=repetition)[0].tolist()
        for y, x in zip(got, values[0].tolist()):
            power = times * math.log2(repetition) * (-1 if x > 0 else 1)
            want = x if x == 0 or math.isinf(x) else math.copysign(2.0 ** min(max(math.log2(abs(x)) + power, -1000), 1000), x)
            if abs(want) >= 2.0 ** 128:
                assert y == math.copysign(math.inf, want), (times, x)
            else:
                # (a result below the normal numbers may be zero)
                assert y == want or abs(y - want) <= 2 ** -21 * (1 + abs(power)) * abs(want) + 2 ** -126, (times, x, y, want)


def test_lowest_values_of_a_type():
    for dtype in (F32, BF16, F16):
        low = torch.finfo(dtype).min
        x = torch.tensor([[low, -low, 0.0, -0.0]], device=DEV, dtype=dtype)
        h = torch.tensor([[0, 1, 2, 3]], device=DEV)
        got = ops.process_logits(x, h, repetition=2.0, cap=1.0)
        assert got[0].tolist() == [-math.inf, -low / 2, 0.0, 0.0]


def test_ids_that_are_no_tokens_and_what_lies_behind_a_history():
    g = gen(10)
    x = logits(g, 2, 100)
    h = torch.tensor([[5, -1, 100, 5, 2 ** 40, -2 ** 40, 7, 7], [1, 2, 3, 4, 5, 6, 7, 8]], device=DEV)
    lens = torch.tensor([6, -3], dtype=torch.int32, device=DEV)
    got = ops.process_logits(x, h, lens, frequency=1.0, repetition=1.5)
    check(got, x, h, lens, frequency=1.0, repetition=1.5)
    assert torch.equal(got[1], x[1]) and float(got[0, 7]) == float(x[0, 7])
    lens = torch.tensor([100, 8], dtype=torch.int32, device=DEV)      # past the tensor: all of it
    check(ops.process_logits(x, h, lens, frequency=1.0), x, h, lens, frequency=1.0)


@pytest.mark.parametrize("T", [40000, 131071])
def test_one_token_all_over_a_long_history(T):
    """Counts and weights of the longest history stay apart and exact."""
    g = gen(11)
    x = logits(g, 1, 2000)
    h = torch.full((1, T), 1999, device=DEV)
    h[0, ::3] = 0
    kw = dict(repetition=1.0001, frequency=0.001, presence=0.25)
    check(ops.process_logits(x, h, **kw), x, h, **kw)
    kw = dict(repetition=1.01, half_life=300.0, frequency=0.001)
    check(ops.process_logits(x, h, **kw), x, h, **kw)
    with pytest.raises(ValueError, match="too long"):
        ops.process_logits(x, torch.zeros(1, 131072, dtype=torch.int64, device=DEV))
    long = torch.zeros(1, 140000, dtype=torch.int64, device=DEV)
    check(ops.process_logits(x, long, lookback=10, frequency=1.0), x, long, lookback=10, frequency=1.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_in_place(dtype):
    g = gen(12)
    B, V = 3, 1501
    room = logits(g, B, 2 * V + 3, dtype)
    x = room[:, 3:3 + V]
    h = history(g, B, 90, V)[:, 1:71]
    bias = torch.randn(B, V + 1, generator=g, device=DEV)[:, 1:]
    allowed = torch.randint(-2 ** 31, 2 ** 31, (B, 60), generator=g, device=DEV).to(torch.int32)[:, 5:5 + 47]
    kw = dict(repetition=1.2, frequency=0.1, bias=bias, allowed=allowed)
    want = ops.process_logits(x.contiguous(), h.contiguous(), repetition=1.2, frequency=0.1, bias=bias.contiguous(), allowed=allowed.contiguous())
    check(want, x, h, **kw)
    assert torch.equal(ops.process_logits(x, h, **kw), want)
    one = bias[:1].expand(B, V)
    assert torch.equal(ops.process_logits(x, h, bias=one), ops.process_logits(x, h, bias=bias[0]))
    half = room[:, 3 + V:]
    assert torch.equal(ops.process_logits(x, h, out=half, **kw), want) and torch.equal(half, want)      # the other half of each row
    for out in (room[:, 2:2 + V], room[:, 2 + V:2 + 2 * V]):
        with pytest.raises(RuntimeError, match="apart"):
            ops.process_logits(x, h, out=out, **kw)
    before = room.clone()
    got = ops.process_logits(x, h, out=x, **kw)
    assert got is x and torch.equal(x, want)
    assert torch.equal(room[:, :3], before[:, :3]) and torch.equal(room[:, 3 + V:], before[:, 3 + V:])


def test_recorded_once_and_replayed():
    g = gen(13)
    x, h = logits(g, 2, 9000), history(g, 2, 64, 9000)
    lens = torch.tensor([3, 60], dtype=torch.int32, device=DEV)
    allowed = ops.pack_allowed(torch.rand(2, 9000, generator=g, device=DEV) < 0.5)
    call = lambda: ops.process_logits(x, h, lens, repetition=1.2, half_life=10.0, allowed=allowed)      # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for it in range(4):
        x.copy_(logits(g, 2, 9000))
        h[:, int(lens[0]) % 64] = it
        lens += 1
        allowed.bitwise_xor_(1 << it)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, call()), it


def test_pack_allowed():
    for device in ("cpu", DEV):
        for V in (1, 31, 32, 33, 100):
            keep = torch.rand(3, V, generator=torch.Generator().manual_seed(V)).to(device) < 0.5
            words = ops.pack_allowed(keep)
            assert words.dtype == torch.int32 and words.shape == (3, -(-V // 32)) and words.device == keep.device
            for b in range(3):
                for v in range(V):
                    assert bool((int(words[b, v // 32]) >> (v % 32)) & 1) == bool(keep[b, v])


def test_refusals():
    g = gen(14)
    x, h = logits(g, 2, 64), history(g, 2, 5, 64)
    lens = torch.tensor([1, 2], dtype=torch.int32, device=DEV)
    bits = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    for error, args, kw in [(TypeError, (x.double(),), {}), (ValueError, (x[None],), {}), (ValueError, (x.t(),), {}), (ValueError, (x, h[:1]), {}), (ValueError, (x, h.float()), {}),
                            (ValueError, (x, None, lens), {}), (ValueError, (x, h, lens.long()), {}), (ValueError, (x, h, lens[:1]), {}), (ValueError, (x, h), dict(half_life=0.0)),
                            (ValueError, (x, h), dict(cap=-1.0)), (ValueError, (x, h), dict(repetition=0.0)), (ValueError, (x, h), dict(repetition=math.nan)), (ValueError, (x, h), dict(repetition=math.inf)),
                            (ValueError, (x, h), dict(repetition=lens.float()[:1])), (ValueError, (x, h), dict(presence=lens)), (ValueError, (x, h), dict(lookback=-1)),
                            (ValueError, (x,), dict(bias=x.bfloat16())), (ValueError, (x,), dict(bias=x[:, :32])), (ValueError, (x,), dict(allowed=bits[:, :1])),
                            (ValueError, (x,), dict(allowed=bits.bool())), (ValueError, (x,), dict(out=x[:1])), (ValueError, (x,), dict(out=x.half())), (RuntimeError, (x.cpu(),), {}),
                            (RuntimeError, (x, h.cpu()), {}), (RuntimeError, (x.clone().requires_grad_(),), {})]:
        with pytest.raises(error):
            ops.process_logits(*args, **kw)
    with pytest.raises(TypeError):
        ops.pack_allowed(bits)
    assert ops.process_logits(x[:0]).shape == (0, 64)
