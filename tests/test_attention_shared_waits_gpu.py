"""Attention behind shared first positions (Ops.attention_shared) when a wait of the tensor-core kernel runs out: the library's next call says so, nothing is read or written that is not the call's, and
later calls are whole again. Tolerance of whole results: 2^-24 * 44 of a value, three times that over the norm."""
import pytest
import torch
from answers_testlib import SharedStep

pytestmark = pytest.mark.gpu


def _after_waits_of(polls, step, want, times):
    from simplellminference_b200 import _lib
    lib = _lib.load()
    assert lib.sllm_status() == 0
    assert lib.sllm_tune(10, polls) == 0
    reported = 0
    try:
        for _ in range(times):
            try:
                got = step.run()[0].double()
                assert (got - want).norm() <= 8e-6 * want.norm()              # nothing ran out
            except _lib.SllmError as e:
                assert e.code == _lib.ETIMEOUT
                reported += 1
            assert lib.sllm_status() == 0
    finally:
        assert lib.sllm_tune(10, 1 << 24) == 0
    got = step.run()[0].double()
    assert (got - want).norm() <= 8e-6 * want.norm()
    return reported


@pytest.mark.parametrize("polls", [0, 1, 4])
@pytest.mark.parametrize("groups", [[(300, [(0, 1)] * 6)], [(0, [(200, 1)] * 5)], [(700, [(0, 40), (9, 1)]), (20, [(0, 300)])], [(2000, [(0, 300), (40, 1)])]], ids=str)
def test_the_whole_cta_stops(groups, polls):
    """In the first item of a CTA or a later one, of either kind."""
    for dim in (64, 128):
        s = SharedStep(groups, 8, 2, dim)
        reported = _after_waits_of(polls, s, s.want(), 5)
        assert reported == 5 or polls > 0


@pytest.mark.parametrize("polls", [0, 1])
@pytest.mark.parametrize("n", [300, 700])
def test_more_tiles_than_a_turn_of_the_plan(n, polls):
    """The plan is made for 256 groups and tiles at a time; the last kernel asks for all of it. The workspace holds ones in every bit before the call."""
    s = SharedStep([((13 * i) % 150, [((7 * i) % 60, 1 + (i % 101 == 7) * 20)]) for i in range(n // 2)] + [(64, [(i % 50, 1) for i in range(n // 2)])], 8, 2, 64)
    reported = _after_waits_of(polls, s, s.want(), 3)
    assert reported == 3 or polls > 0
