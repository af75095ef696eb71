"""Very large and infinite values beside keys of far larger scores in attention behind shared first positions (Ops.attention_shared), against float64.

One key has value 1e36 and score 0, another one, before or behind it, score 100: e^-100 = 3.7e-44 is the weight of the first. Whatever the kernel makes of a weight below 2^-126, its part is off by
no more than itself, 1e36 * 3.8e-44; the rest is a weight of 1 and sums of few numbers that are not zero: sixteen roundings."""
import math

import pytest
import torch
from answers_testlib import SharedStep

pytestmark = pytest.mark.gpu
# (position of the large value, position of the large score): in a tile of 16, 32 or 48 keys, of a share, and in other shares and teams' parts, either way round
PAIRS = [(3, 20), (20, 3), (40, 41), (5, 33), (33, 5), (10, 60), (60, 10), (0, 63), (63, 100), (100, 63), (47, 48), (2, 300), (300, 2), (130, 639), (639, 0)]


def _step(groups, dim, dtype, gap):
    """Every score is 0 but those that `at` raises to `gap`."""
    s = SharedStep(groups, 8, 2, dim, dtype=dtype, seed=5)
    s.q.zero_()
    s.q.view(-1, 8, dim)[..., 0] = 1.0
    s.k.zero_()

    def at(i, pos, score=None, value=None):
        page, row = s.table_np[i, pos // s.page], pos % s.page
        if score is not None:
            s.k[page, :, row, 0] = score
        if value is not None:
            s.v[page, :, row, 3:dim - 2] = value

    return s, at


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("where", ["shared", "own", "both"])
def test_large_values_without_weight(where, dim, dtype):
    for large, high in PAIRS:
        # of shared positions and a decoding token's own ones, or a portion's; a token sees all that is asked for
        groups = {"shared": [(640, [(0, 1), (30, 1), (0, 20)])], "own": [(0, [(640, 1)]), (64, [(640, 40)]), (0, [(641, 3)])], "both": [(320, [(340, 1), (330, 40)])]}[where]
        s, at = _step(groups, dim, dtype, 100.0)
        firsts = {"shared": [0], "own": [0, 1, 2], "both": [0, 1]}[where]
        for i in firsts:
            at(i, large, value=1e36)
            at(i, high, score=100.0)
        want = s.want(scale=1.0)
        got = s.run(scale=1.0)[0].double()
        assert ((got - want).abs() <= 16 * 2.0 ** -24 * want.abs() + 1e36 * 3.8e-44).all(), (large, high, (got - want).abs().max())


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_infinite_values_without_weight(dim, dtype, value):
    """The weight is e^-300, beyond fp32, but not zero: an infinity stays one, whatever comes before or behind it."""
    for large, high in PAIRS[::2]:
        s, at = _step([(320, [(340, 1), (330, 40)]), (640, [(0, 1)])], dim, dtype, 300.0)
        for i in range(3):
            at(i, large, value=value)
            at(i, high, score=300.0)
        want, got = s.want(scale=1.0), s.run(scale=1.0)[0].double()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf()), (large, high)
        fine = want.isfinite()
        assert not fine.all() and torch.equal(got[want.isinf()], want[want.isinf()])
        assert ((got - want).abs()[fine] <= 16 * 2.0 ** -24 * want.abs()[fine] + 1e-30).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_values_as_large_as_they_may_be(dim, dtype):
    """Sums are taken before the division, with weights of up to 2^8: values of 2^119 divided by the number of keys stay numbers. Scores of size 1: 2^-24 * (8 + 16 + 20) of the largest value seen,
    three times that over the norm."""
    s = SharedStep([(700, [(0, 1), (200, 1), (10, 60)]), (0, [(900, 1), (0, 300)])], 8, 2, dim, dtype=dtype, seed=9)
    s.v = (s.v.sign() * 2.0 ** 119 / 1024).to(dtype)
    got, want = s.run()[0].double(), s.want()
    assert torch.isfinite(got).all() and (got - want).norm() <= 8e-6 * want.norm()
    assert (got - want).abs().max() <= 3e-5 * 2.0 ** 109
