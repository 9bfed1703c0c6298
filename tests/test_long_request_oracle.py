"""The plain forms of the recurrence's gradients against differences and against automatic ones, and the rotary frequencies."""
import math

import pytest
import torch

import long_request_oracle as oracle


def test_recurrence_gradients_against_automatic_ones_and_differences():
    g = torch.Generator().manual_seed(1)
    lengths, channels = [7, 0, 1, 12], 3
    tokens = sum(lengths)
    make = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).float()
    x, l, dout = make(tokens, channels), -make(tokens, channels).abs(), make(tokens, channels)
    initial, dfinal = make(4, channels), make(4, channels)
    got = oracle.recurrence(x, l, lengths, initial, dout, dfinal)

    def loss(x, l, initial):
        total, at = 0.0, 0
        for b, n in enumerate(lengths):
            h = initial[b]
            for t in range(at, at + n):
                h = l[t].exp() * h + x[t]
                total = total + (h * dout[t].double()).sum()
            total = total + (h * dfinal[b].double()).sum()
            at += n
        return total

    inputs = [t.double().requires_grad_() for t in (x, l, initial)]
    for name, grad in zip(("dx", "dlog_decay", "dinitial"), torch.autograd.grad(loss(*inputs), inputs)):
        assert torch.allclose(got[name][0], grad, rtol=1e-12, atol=1e-12), name
    for which, name in enumerate(("dx", "dlog_decay", "dinitial")):
        v = make(*inputs[which].shape).double()
        step = 1e-5
        moved = lambda s: [t.detach() + (s * v if i == which else 0.0) for i, t in enumerate(inputs)]
        difference = (loss(*moved(step)) - loss(*moved(-step))) / (2 * step)
        # Rounding 1e-16 of a loss of some hundred over 1e-5, and 1e-10 times the third derivative.
        assert abs(float(difference - (got[name][0] * v).sum())) < 1e-7, name


def test_frequencies(hip):
    make = lambda *a, **k: hip.rotary_frequencies(*a, device="cpu", **k)
    i = torch.arange(64, dtype=torch.float64)
    plain = 10000.0 ** (-i / 64)
    close = lambda a, b: torch.allclose(a, b, rtol=1e-14, atol=0.0)
    assert close(make(128), plain)
    assert close(make(128, base=500.0), 500.0 ** (-i / 64))
    assert close(make(128, scaling="linear", scale=4.0), plain / 4)
    stretched = make(128, scaling="base", scale=8.0)
    assert close(stretched[0], plain[0]) and close(stretched[-1], plain[-1] / 8)
    bands = make(128, scaling="bands", scale=8.0, trained=8192.0, low=1.0, high=4.0)
    turns = 8192.0 * plain / (2 * math.pi)
    assert close(bands[turns >= 4], plain[turns >= 4]) and close(bands[turns <= 1], plain[turns <= 1] / 8)
    some = (turns > 1) & (turns < 4)
    part = (turns - 1) / 3
    assert bool(some.any()) and close(bands[some], (plain * (part + (1 - part) / 8))[some])


@pytest.mark.parametrize("change", [dict(rotary_dim=0), dict(rotary_dim=7), dict(base=0.0), dict(base=-1.0), dict(base=math.inf),
                                    dict(scale=0.0), dict(scale=math.nan), dict(scaling="bands"), dict(scaling="bands", trained=10.0, low=4.0),
                                    dict(scaling="bands", trained=math.inf), dict(scaling="base", rotary_dim=2)])
def test_frequencies_refuse(hip, change):
    with pytest.raises(hip.LcppHipError) as e:
        hip.rotary_frequencies(**({"rotary_dim": 64, "device": "cpu"} | change))
    assert e.value.status == hip.ERR_INVALID_ARGUMENT


def test_an_unknown_scaling_is_refused(hip):
    with pytest.raises(ValueError, match="plain, linear"):
        hip.rotary_frequencies(64, scaling="yes", device="cpu")
