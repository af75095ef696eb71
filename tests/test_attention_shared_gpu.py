"""Attention behind shared first positions (Ops.attention_shared) against float64, every request by itself over its own pages.

Tolerance: a score is a sum of dk products of size 1, off by some sqrt(dk) roundings of its running sum (of size sqrt(dk)) in fp32, a weight by what its score is; the sums over keys are off by a
few roundings a tile. With dk up to 256 and scores up to 8 that is 2^-24 * (8 + 16 + 20) = 2.6e-6 of a value's size; three times that over the norm of a row, ten times in a single number."""
import math

import pytest
import torch
from answers_testlib import SharedStep

pytestmark = pytest.mark.gpu
NORM, ONE = 8e-6, 3e-5


def _close(got, want, one=ONE):
    got = got.double()
    assert torch.isfinite(got).all()
    scale = want.abs().amax(-1, keepdim=True).clamp_min(0.05)
    off = (got - want).abs() / scale
    assert off.max() <= one, off.max()
    assert (got - want).norm() <= NORM * want.norm() + 1e-12, (got - want).norm() / want.norm()


def _owns(n, longest, new=1):
    return [((37 * i * i + 11 * i) % longest, new) for i in range(n)]


SHAPES = [(8, 2, 128), (12, 4, 64), (4, 4, 64), (8, 1, 128), (6, 2, 64)]


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("groups", [
    [(500, _owns(5, 90))], [(64, [(0, 1)])], [(1, [(0, 1), (5, 1)])], [(0, [(0, 1)])], [(0, _owns(4, 200))], [(1000, [(0, 1)] * 3)], [(63, _owns(3, 5)), (65, _owns(2, 300)), (0, [(31, 1)])],
    [(320, _owns(40, 70))], [(130, [(0, 37), (3, 1), (70, 5), (0, 64)])], [(0, [(0, 100)]), (200, [(0, 33), (20, 2)])], [(2000, [(0, 150), (1, 1)])]], ids=str)
def test_groups(groups, heads, kv_heads, dim, dtype):
    s = SharedStep(groups, heads, kv_heads, dim, dtype=dtype)
    _close(s.run()[0], s.want())


@pytest.mark.parametrize("page", [32, 64, 96, 128])
def test_pages(page):
    for groups in ([(page, _owns(3, 50))], [(3 * page - 1, _owns(3, 2 * page))], [(2 * page + 31, [(0, 40), (5, 1)])]):
        s = SharedStep(groups, 8, 2, 128, page=page, seed=page)
        _close(s.run()[0], s.want())


@pytest.mark.parametrize("dk,dv", [(8, 8), (40, 24), (128, 64), (64, 128), (192, 128), (256, 256), (96, 96)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_other_widths(dk, dv, dtype):
    s = SharedStep([(150, _owns(3, 40)), (70, [(0, 20)])], 6, 3, dk, dv, dtype=dtype)
    _close(s.run()[0], s.want())


@pytest.mark.parametrize("heads,kv_heads", [(16, 16), (10, 2), (16, 2), (24, 1), (40, 1), (7, 7)])
def test_head_groups(heads, kv_heads):
    s = SharedStep([(300, _owns(9, 100)), (40, [(2, 35)])], heads, kv_heads, 64)
    _close(s.run()[0], s.want())


OPTIONS = [dict(window=100), dict(window=100, keep=4), dict(window=1), dict(window=33, keep=70), dict(window=5000, keep=3), dict(cap=2.0), dict(cap=30.0), dict(window=77, keep=5, cap=5.0)]


@pytest.mark.parametrize("opts", OPTIONS, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128])
def test_options(opts, dtype, dim):
    s = SharedStep([(400, _owns(6, 200)), (130, [(0, 70), (9, 1)]), (0, [(90, 1)])], 8, 2, dim, dtype=dtype)
    got = s.run(window=opts.get("window", 0), keep_first=opts.get("keep", 0), softcap=opts.get("cap", 0.0))[0]
    _close(got, s.want(**opts))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_slopes(dtype):
    slopes = 2.0 ** -torch.arange(1, 9).float()
    s = SharedStep([(400, _owns(6, 200)), (130, [(0, 70), (9, 1)])], 8, 2, 64, dtype=dtype)
    _close(s.run(slopes=slopes)[0], s.want(slopes=slopes))
    _close(s.run(slopes=slopes, window=90, keep_first=4, softcap=8.0)[0], s.want(slopes=slopes, window=90, keep=4, cap=8.0))


@pytest.mark.parametrize("dim", [64, 128])
def test_large_and_small_scores(dim):
    """Weights far below the largest, all on one key, and nearly even ones."""
    s = SharedStep([(700, _owns(6, 200)), (100, [(0, 50)])], 8, 2, dim)
    for scale in (1e-4, 1.0, 20.0):
        _close(s.run(scale=scale)[0], s.want(scale=scale), one=ONE if scale < 20 else 3e-4)      # scores of some 1000 are off by 2^-24 * 1000 times the square root of a few roundings


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_results_in_bf16_are_those_in_fp32_rounded(dtype):
    s = SharedStep([(500, _owns(5, 90)), (77, [(0, 40)])], 8, 2, 128, dtype=dtype)
    a, b = s.run(out=True, out16=True)
    only = s.run(out=False, out16=True)[1]
    assert torch.equal(a.bfloat16(), b) and torch.equal(b, only)
    assert torch.equal(a, s.run()[0])


def test_rows_apart_and_rows_behind():
    """Strides wider than rows, unaligned ones, and rows of no token, which stay as they were."""
    s = SharedStep([(100, _owns(4, 30)), (40, [(0, 40)])], 8, 2, 64, tail=3)
    for ldq, ldo in ((516, 520), (513, 515), (512, 600)):
        got = s.run(ldq=ldq, ldo=ldo)[0]
        _close(got[:s.n_tokens, :512], s.want())
        assert (got[s.n_tokens:] == 7.0).all() and (got[:, 512:] == 7.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_tokens_in_no_tile_stay(dtype):
    groups = [(100, [(0, 70), (5, 1), (0, 40)]), (0, [(33, 1)])]
    s = SharedStep(groups, 8, 2, 64, dtype=dtype, tiles=[(0, 32), (2, 0), (3, 0)])
    got, want = s.run()[0], s.want()
    listed = torch.zeros(s.n_tokens, dtype=torch.bool)
    listed[32:64] = listed[71:103] = listed[111] = True
    _close(got[listed], want[listed])
    assert (got[~listed] == 7.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_hidden_rows_may_hold_anything(dtype, dim):
    """NaN and infinities behind the last position, in pages of nobody, and before a window."""
    s = SharedStep([(300, [(0, 1), (50, 1), (3, 30)]), (10, [(5, 1)])], 8, 2, dim, dtype=dtype)
    want = s.want()
    held = torch.zeros(s.n_pages, s.page, dtype=torch.bool)
    for i, (_, p, n) in enumerate(s.segs):
        for j in range(p + n):
            held[s.table_np[i, j // s.page], j % s.page] = True
    for pool in (s.k, s.v):
        pool.transpose(1, 2)[~held] = math.nan
    s.v.transpose(1, 2)[~held] = math.inf
    _close(s.run()[0], want)
    want = s.want(window=60)
    first = s.table_np[0, 0]                                                  # positions 0 .. 63 of the first group: behind every window
    s.k[first], s.v[first] = math.nan, math.nan
    _close(s.run(window=60)[0], want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_that_are_not_finite_reach_who_sees_them(dtype):
    """Inside a portion, and before some tokens' windows: the rows that see such a value have it, the others are as without it."""
    groups = [(100, [(0, 40), (30, 1)]), (90, [(0, 1), (60, 1)])]
    s = SharedStep(groups, 8, 2, 64, dtype=dtype)
    plain = s.want(window=110)
    s.v[s.table_np[0, 1], 0, 115 - 64, 7] = math.inf                          # position 115 of the first request: its tokens from there on
    s.v[s.table_np[2, 0], 1, 30, 3] = math.nan                                # position 30 of the second group: 90 and 91 see it, 150 and 151 do not
    got, want = s.run(window=110)[0].double(), s.want(window=110)
    assert want.isinf().any() and want.isnan().any()
    assert torch.equal(got.isfinite(), want.isfinite()) and torch.equal(got.isnan(), want.isnan())
    fine = want.isfinite()
    assert ((got - want).abs()[fine] <= ONE * plain.abs().amax()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 72, 128])
def test_pages_that_are_not_there(dtype, dim):
    """Missing and impossible pages hide their keys; a token with no other gives zeros."""
    s = SharedStep([(200, [(0, 1), (60, 1)]), (70, [(0, 20)]), (0, [(10, 1)])], 8, 2, dim, dtype=dtype)
    table = s.table_np
    table[0, 1] = table[1, 1] = -1
    table[1, 4] = s.n_pages + 5
    table[2, 1] = 1 << 30
    table[3, 0] = -7
    s.dev["block_table"].copy_(torch.tensor(table))
    want = s.want()
    assert (want[-1] == 0).all()
    _close(s.run()[0], want)


def test_a_group_is_read_through_its_first_segment():
    """Only the first member's table has the shared pages."""
    s = SharedStep([(256, _owns(4, 60))], 8, 2, 128)
    want = s.want()
    table = s.table_np.copy()
    table[1:, :4] = -1
    s.dev["block_table"].copy_(torch.tensor(table))
    _close(s.run()[0], want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_lengths_that_do_not_fit(dtype):
    """A group length beyond a token's own position shows it nothing of what comes later; one below zero shares nothing."""
    s = SharedStep([(100, [(0, 30)]), (64, [(3, 1)])], 8, 2, 64, dtype=dtype)
    want = s.want()
    for lens in ([120, 64], [5000, 10], [-3, -1], [100, 0]):
        got = s.run(groups=(s.group_start, torch.tensor(lens, dtype=torch.int32, device="cuda")))[0]
        _close(got, want)


def test_same_as_ordinary_attention():
    """With nothing shared in any group, and with all of it: the result of every request by itself."""
    s = SharedStep([(640, _owns(5, 90))], 8, 2, 128)
    a = s.run()[0]
    start = torch.arange(6, dtype=torch.int32, device="cuda")
    b = s.run(groups=(start, torch.zeros(5, dtype=torch.int32, device="cuda")))[0]
    _close(b, s.want())
    assert (a - b).abs().max() <= ONE * a.abs().max()


def test_repeats_are_equal():
    """Nothing depends on the order of CTAs; nothing is kept from one call to the next."""
    s = SharedStep([(700, _owns(20, 150)), (64, [(0, 70)])], 16, 4, 128)
    first = s.run(out16=True)
    for _ in range(3):
        again = s.run(out16=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_captured_with_lengths_that_grow():
    """A captured call reads positions, lengths and tables on the device: replayed after they have changed, it gives the new step's result."""
    from simplellminference_b200.config import BF16
    from simplellminference_b200.seqops import Ops
    early = SharedStep([(300, [(5, 1), (100, 1), (0, 1)])], 8, 2, 64, seed=3)
    late = SharedStep([(300, [(6, 1), (101, 1), (1, 1)])], 8, 2, 64, seed=3)
    if early.table_np.shape != late.table_np.shape or early.n_pages != late.n_pages:
        pytest.skip("the two steps need the same pages")
    ops = Ops(BF16)
    q, k, v = early.q.cuda(), early.k.cuda(), early.v.cuda()
    out = torch.zeros(3, 512, device="cuda")
    ws = torch.zeros(ops.attention_shared_ws_bytes(early.b, 1, 8, 2, 64, 64), dtype=torch.uint8, device="cuda")

    def call():
        ops.attention_shared(early.b, 1, early.group_start, early.group_len, q.data_ptr(), 512, 8, 2, 64, 64, 0.125, k, v, early.n_pages, ws, torch.cuda.current_stream().cuda_stream, out=out, ldo=512)

    call()
    torch.cuda.synchronize()
    _close(out.cpu(), early.want())
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        call()
        call()
    ops.overlap(g.raw_cuda_graph())
    g.instantiate()
    for a, b in ((q, late.q), (k, late.k), (v, late.v)):
        a.copy_(b.cuda())
    for name in early.dev:
        early.dev[name].copy_(late.dev[name])
    g.replay()
    torch.cuda.synchronize()
    _close(out.cpu(), late.want())


def test_waits_that_run_out_are_reported():
    """With no polls allowed the tensor-core kernel gives up its first waits; the library's next call says so, once, and later launches are whole again."""
    from simplellminference_b200 import _lib
    lib = _lib.load()
    s = SharedStep([(300, _owns(6, 90)), (20, [(0, 40)])], 8, 2, 128)
    assert lib.sllm_status() == 0
    assert lib.sllm_tune(10, 0) == 0
    try:
        with pytest.raises(_lib.SllmError) as e:
            s.run()
    finally:
        assert lib.sllm_tune(10, 1 << 24) == 0
    assert e.value.code == _lib.ETIMEOUT and lib.sllm_status() == 0
    _close(s.run()[0], s.want())


@pytest.mark.parametrize("opts", [{}, {"softcap": 30.0}, {"window": 700, "keep_first": 3}], ids=str)
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_enough_for_long_shares(dim, opts):
    """So many rows that a share of the keys is longer than what the tensor core adds up at a time; the scores of later keys are the largest. Scores of up to 40 in size: three times
    2^-24 * (40 + 16 + 20) over a row's norm, and over the sums of a share the tensor core's truncated additions (nine a tile, nine tiles), a unit of 2^-24 each at most, half of which the weights'
    sum loses too."""
    s = SharedStep([(1500, [(0, 400), (7, 200)]), (900, [(0, 1)] * 3)], 32, 8, dim, seed=dim)
    for at in s.table_np[0, 14:22]:
        s.k[at] *= 3
    got, want = s.run(**opts)[0].double(), s.want(window=opts.get("window", 0), keep=opts.get("keep_first", 0), cap=opts.get("softcap", 0.0))
    assert torch.isfinite(got).all()
    assert (got - want).norm() <= (3 * 2.0 ** -24 * 76 + 2.0 ** -25 * 81) * want.norm()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [257, 600])
def test_many_groups(n, dtype):
    """More groups than a CTA looks at in one turn."""
    s = SharedStep([((13 * i) % 150, _owns(1 + (i % 97 == 5) * 3, 60, 1 + (i % 101 == 7) * 20)) for i in range(n)], 4, 2, 64, dtype=dtype)
    _close(s.run()[0], s.want())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
@pytest.mark.parametrize("dim", [64, 128])
def test_later_keys_show_in_no_bit(dim, softcap, dtype):
    """A token's results are the same numbers whatever the keys and values behind it hold, although rows beside it see them."""
    s = SharedStep([(200, [(0, 150), (30, 100)]), (700, [(0, 2)])], 8, 2, dim, dtype=dtype, seed=11)
    first = s.run(softcap=softcap)[0]
    for i, at in ((0, 75), (1, 40), (2, 1)):
        _, pos, n = s.segs[i]
        for j in range(pos + at, pos + n):
            page, row = s.table_np[i, j // s.page], j % s.page
            s.k[page, :, row] *= 30
            s.v[page, :, row] = math.inf if j % 2 else 3e38
    again = s.run(softcap=softcap)[0]
    for rows in (slice(0, 75), slice(150, 190), slice(250, 251)):
        assert torch.equal(first[rows], again[rows]), rows
    assert not torch.equal(first, again)
