"""``ops.process_logits`` at settings that fp32 does not hold."""
import pytest
import torch

from daisy_amd import ops
from test_logits_gpu import DEV, check, gen, history, logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("half_life", [1e-300, 1e-50, 1e-45, 1e-39, 1e-38, 1e-3])
def test_half_lives_below_the_normal_numbers_forget_everything(half_life):
    """2 ** (-age / half_life) is zero from the first token on: the repetition penalty leaves every logit, presence and frequency count as ever."""
    g = gen(3)
    x, h = logits(g, 2, 300), history(g, 2, 50, 300)
    kw = dict(repetition=1.7, half_life=half_life, presence=0.25, frequency=0.5)
    check(ops.process_logits(x, h, **kw), x, h, **kw)


@pytest.mark.parametrize("half_life", [1e39, 1e300, float("inf")])
def test_half_lives_past_the_largest_number_forget_nothing(half_life):
    g = gen(4)
    x, h = logits(g, 2, 300), history(g, 2, 50, 300)
    kw = dict(repetition=1.7, presence=0.25, frequency=0.5)
    check(ops.process_logits(x, h, half_life=half_life, **kw), x, h, **kw)


def test_the_way_through_python_is_the_same(monkeypatch):
    """What the call in front of it does not take."""
    from daisy_amd import _lib
    g = gen(5)
    x, h = logits(g, 2, 300), history(g, 2, 50, 300)
    native = _lib.native()

    class WithoutTheCall:
        def __getattr__(self, name):
            return (lambda *args: None) if name == "process_logits" else getattr(native, name)

    monkeypatch.setattr(_lib, "native", lambda: WithoutTheCall())
    for half_life in (1e-300, 1e-39, 140.0, 1e39):
        kw = dict(repetition=1.7, half_life=half_life, presence=0.25, frequency=0.5)
        check(ops.process_logits(x, h, **kw), x, h, **kw)
