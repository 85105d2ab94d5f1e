"""Values of rotary_frequencies: every scaling against its definition, pair by pair."""
import math

import pytest
import torch

import simplical_attn_amd as sa


def _plain(dim, base):
    return [base ** (-2.0 * j / dim) for j in range(dim // 2)]


def _check(got, want):
    # a power, a logarithm and a handful of products in 64 bits: far below 1e-12
    assert got.dtype == torch.float64 and got.shape == (len(want),)
    assert (got - torch.tensor(want, dtype=torch.float64)).abs().div(torch.tensor(want, dtype=torch.float64)).max() <= 1e-12


@pytest.mark.parametrize("dim,base", [(2, 10000.0), (64, 10000.0), (128, 500000.0), (80, 1e6)])
def test_plain_linear_and_base(dim, base):
    _check(sa.rotary_frequencies(dim, base), _plain(dim, base))
    _check(sa.rotary_frequencies(dim, base, scaling="linear", factor=4.0), [f / 4.0 for f in _plain(dim, base)])
    if dim > 2:
        got = sa.rotary_frequencies(dim, base, scaling="base", factor=8.0)
        _check(got, _plain(dim, base * 8.0 ** (dim / (dim - 2))))
        # the slowest pair is divided by the factor, the fastest stays
        assert got[0] == 1.0 and abs(got[-1].item() * 8.0 / _plain(dim, base)[-1] - 1) < 1e-12


# the last three: the slowest pair makes more than slow_turns turns (2.4, 11 and 28), so that the ramp ends behind it
LENGTHS = [(128, 1e4, 4096), (64, 1e4, 8192), (64, 1e4, 2048), (128, 5e5, 8192), (16, 1e4, 100), (128, 1e4, 131072), (64, 1e4, 131072), (32, 1e4, 400000), (32, 1e4, 1000000)]


@pytest.mark.parametrize("slow,fast", [(1.0, 32.0), (2.0, 8.0)])
@pytest.mark.parametrize("dim,base,length", LENGTHS)
def test_parts(dim, base, length, slow, fast):
    factor = 8.0
    got = sa.rotary_frequencies(dim, base, scaling="parts", factor=factor, original_length=length, slow_turns=slow, fast_turns=fast)
    pair = lambda turns: dim * math.log(length / (2 * math.pi * turns)) / (2 * math.log(base))
    first, last = max(0, math.floor(pair(fast))), min(dim - 1, math.ceil(pair(slow)))
    want = []
    for j, f in enumerate(_plain(dim, base)):
        part = 0.0 if j <= first else 1.0 if j >= last else (j - first) / (last - first)
        want.append(f * (1 - part) + f / factor * part)
        turns = length * f / (2 * math.pi)
        if turns <= slow:
            assert abs(got[j].item() * factor / f - 1) < 1e-12
        elif turns > 1.0001 * slow and j > first:
            assert got[j].item() > f / factor
        if turns >= fast:
            assert got[j].item() == f
    _check(got, want)


def test_parts_by_hand():
    """Eight pairs of base 10^4, a length of 2 pi 10^4: pair j makes 10^(4 - j/2) turns, 32 and 1 turns are pairs 4.99 and 8."""
    got = sa.rotary_frequencies(16, 1e4, scaling="parts", factor=2.0, original_length=2 * math.pi * 1e4)
    kept = [1, 1, 1, 1, 1, 0.75, 0.5, 0.25]
    _check(got, [f * (0.5 + 0.5 * k) for f, k in zip(_plain(16, 1e4), kept)])


def test_parts_of_a_short_length():
    """No pair makes a whole turn: all are divided."""
    _check(sa.rotary_frequencies(16, 1e4, scaling="parts", factor=4.0, original_length=6), [f / 4.0 for f in _plain(16, 1e4)])
