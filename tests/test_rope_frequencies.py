"""rope_frequencies(): the formulas of each scaling, on the CPU."""

import math

import pytest
import torch

from flashattn_cuda import rope_frequencies


def plain(d, base=10000.0):
    return [base ** (-2 * i / d) for i in range(d // 2)]


def near(freqs, want):
    assert freqs.dtype == torch.float64
    assert freqs.tolist() == pytest.approx(want, rel=1e-12)


def test_plain_and_linear():
    f, a = rope_frequencies(64, device="cpu")
    near(f, plain(64))
    assert a == 1.0
    near(rope_frequencies(20, base=500000.0, device="cpu")[0], plain(20, 500000.0))
    near(rope_frequencies(64, scaling="linear", factor=4.0, device="cpu")[0],
         [x / 4 for x in plain(64)])


def test_base_scaling_divides_the_slowest_pair():
    f, a = rope_frequencies(128, scaling="base", factor=8.0, device="cpu")
    want = plain(128)
    assert f[0].item() == 1.0 and a == 1.0
    assert f[-1].item() == pytest.approx(want[-1] / 8.0, rel=1e-12)


def test_bands():
    f, a = rope_frequencies(128, base=500000.0, scaling="bands", factor=8.0,
                            original_length=8192, device="cpu")
    assert a == 1.0
    for got, x in zip(f.tolist(), plain(128, 500000.0)):
        turns = 8192 * x / (2 * math.pi)
        mix = min(1.0, max(0.0, (turns - 1) / 3))
        assert got == pytest.approx(mix * x + (1 - mix) * x / 8, rel=1e-12)
    assert f[0].item() == 1.0


def test_yarn():
    f, a = rope_frequencies(64, scaling="yarn", factor=16.0, original_length=4096,
                            device="cpu")
    assert a == pytest.approx(0.1 * math.log(16) + 1)
    pair_of = lambda turns: 64 * math.log(4096 / (2 * math.pi * turns)) / (2 * math.log(10000))
    first, last = math.floor(pair_of(32)), math.ceil(pair_of(1))
    for i, (got, x) in enumerate(zip(f.tolist(), plain(64))):
        mix = 1 - min(1.0, max(0.0, (i - first) / (last - first)))
        assert got == pytest.approx(mix * x + (1 - mix) * x / 16, rel=1e-12)


@pytest.mark.parametrize("kw", [
    dict(rotary_dim=63), dict(rotary_dim=0), dict(rotary_dim=64, base=1.0),
    dict(rotary_dim=64, factor=0.5), dict(rotary_dim=64, scaling="cubic"),
    dict(rotary_dim=64, scaling="bands", factor=2.0),
    dict(rotary_dim=64, scaling="yarn", factor=2.0, original_length=100, low=4.0, high=2.0),
    dict(rotary_dim=2, scaling="base", factor=2.0)])
def test_refusals(kw):
    with pytest.raises(ValueError):
        rope_frequencies(device="cpu", **kw)
