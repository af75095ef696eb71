"""Attention behind shared first positions (Ops.attention_shared) with lengths and options at the ends of their range. Tolerance: 2^-24 * 44 of a value, three times that over the norm."""
import pytest
import torch
from answers_testlib import SharedStep

pytestmark = pytest.mark.gpu
MOST = 2 ** 31 - 1


def _close(got, want):
    assert torch.isfinite(got).all() and (got.double() - want).norm() <= 8e-6 * want.norm()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_group_lengths_of_any_size(dim, dtype):
    """All that a token sees is then shared; positions that no table has room for have no page."""
    s = SharedStep([(100, [(0, 30)]), (64, [(3, 1)]), (0, [(200, 1)])], 8, 2, dim, dtype=dtype)
    want = s.want()
    for lens in ([MOST] * 3, [MOST - 31, MOST - 47, MOST - 63], [MOST - 255, 1 << 30, MOST - 300], [-MOST - 1, MOST, 150]):
        _close(s.run(groups=(s.group_start, torch.tensor(lens, dtype=torch.int32, device="cuda")))[0], want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_groups_of_any_size(dtype):
    """More of them than a CTA looks at in one turn, one request each."""
    s = SharedStep([((13 * i) % 150, [((7 * i) % 60, 1 + (i % 101 == 7) * 20)]) for i in range(300)], 8, 2, 64, dtype=dtype)
    _close(s.run(groups=(s.group_start, torch.full((300,), MOST, dtype=torch.int32, device="cuda")))[0], s.want())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_first_positions_that_stay_visible_without_end(dim, dtype):
    """Whatever the window, all positions are then seen."""
    s = SharedStep([(400, [(10, 1), (100, 1)]), (130, [(0, 70)]), (0, [(300, 1), (7, 200)])], 8, 2, dim, dtype=dtype)
    want = s.want()
    for window, keep in ((100, MOST), (1, MOST - 40), (MOST, MOST), (60, 1 << 30)):
        _close(s.run(window=window, keep_first=keep)[0], want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_segments_without_tokens(dtype):
    """Places of a captured step that are not taken: segments of no tokens, tiles of them among the listed ones, a group of nothing else."""
    groups = [(100, [(0, 1), (5, 0), (30, 40)]), (64, [(0, 0), (9, 0)]), (70, [(3, 0), (20, 1)]), (0, [(0, 0)])]
    s = SharedStep(groups, 8, 2, 64, dtype=dtype, tiles=[(0, 0), (1, 0), (2, 32), (2, 0), (3, 0), (4, 0), (5, 0), (6, 0), (7, 0)])
    _close(s.run()[0], s.want())
