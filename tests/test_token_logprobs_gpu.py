"""Log probabilities, ranks, entropies and alternatives (Ops.token_logprobs) against float64.

Tolerances, in units of 2^-24: x - M is rounded once (|z|); a weight is off by the rounding of z log2(e) (|z|, some 30 where weights matter), of ex2.approx (4) and of its sum (32 additions a
thread, 14 levels above), which is what log S is off by; the entropy's second sum the same, of itself."""
import math

import pytest
import torch
from answers_testlib import logprobs_of

pytestmark = pytest.mark.gpu
UNIT = 2.0 ** -24


def _ops():
    from simplellminference_b200.config import BF16
    from simplellminference_b200.seqops import Ops
    return Ops(BF16)


def _run(x, token=None, top=0, ld=None, offset=0, n=None, want=("logprob", "entropy", "rank", "top_logprob"), stream=None):
    """x [rows][n] on the CPU, put `ld` apart behind `offset` values."""
    rows, n = x.shape
    ld = ld or n
    flat = torch.full((offset + rows * ld + 4,), math.nan)
    flat[offset:offset + rows * ld].view(rows, ld)[:, :n] = x
    flat = flat.cuda()
    out = {"logprob": torch.full((rows,), 9.0, device="cuda"), "entropy": torch.full((rows,), 9.0, device="cuda"), "rank": torch.full((rows,), -9, dtype=torch.int32, device="cuda"),
           "top_idx": torch.full((rows, max(top, 1)), -9, dtype=torch.int32, device="cuda"), "top_logprob": torch.full((rows, max(top, 1)), 9.0, device="cuda")}
    tok = None if token is None else torch.as_tensor(token, dtype=torch.int32).cuda()
    _ops().token_logprobs(flat.data_ptr() + 4 * offset, ld, rows, n, tok, stream or torch.cuda.current_stream().cuda_stream, logprob=out["logprob"] if tok is not None and "logprob" in want else None,
                          entropy=out["entropy"] if "entropy" in want else None, rank=out["rank"] if tok is not None and "rank" in want else None, top=top, top_idx=out["top_idx"] if top else None,
                          top_logprob=out["top_logprob"] if top and "top_logprob" in want else None)
    torch.cuda.synchronize()
    return {k: v.cpu() for k, v in out.items()}


def _check(x, token, top, **kw):
    got = _run(x, token, top, **kw)
    lp, rank, entropy, idx, tlp = logprobs_of(x, torch.as_tensor(token), top)
    for a, b in [(got["logprob"], lp)] + ([(got["top_logprob"], tlp)] if top else []):
        b = b.float().double()                    # a difference beyond fp32's range (3.4e38) is -infinity there
        same = (a == -math.inf) & (b == -math.inf)
        off = torch.where(same, 0.0, (a.double() - b).abs())
        assert (off <= UNIT * (4 * torch.where(same, 0.0, b).abs() + 128)).all(), off.max()
    assert ((got["entropy"].double() - entropy).abs() <= UNIT * (128 * entropy + 128)).all(), (got["entropy"].double() - entropy).abs().max()
    assert got["rank"].tolist() == rank.tolist()
    if top:
        assert got["top_idx"].tolist() == idx.tolist()


def _logits(rows, n, spread, seed, rounded=False):
    x = spread * torch.randn(rows, n, generator=torch.Generator().manual_seed(seed))
    return x.bfloat16().float() if rounded else x


@pytest.mark.parametrize("rows,n", [(3, 1), (3, 2), (5, 31), (5, 500), (4, 511), (4, 2047), (4, 2048), (4, 4097), (1, 32000), (7, 32001), (300, 1000), (40, 50257), (3, 128256), (70, 128256), (2, 131073),
                                    (2, 300001)])
@pytest.mark.parametrize("spread,rounded", [(0.05, False), (2.5, True), (12.0, False)])
def test_rows(rows, n, spread, rounded):
    x = _logits(rows, n, spread, rows + n, rounded)
    token = torch.randint(0, n, (rows,), generator=torch.Generator().manual_seed(n))
    token[0] = n - 1
    token[-1] = int(x[-1].argmax())
    for top in sorted({0, 1, min(n, 17), min(n, 32)}):
        _check(x, token, top)


@pytest.mark.parametrize("ld,offset", [(5000, 0), (5003, 0), (5000, 1), (5001, 3)])
def test_strides_and_alignment(ld, offset):
    _check(_logits(9, 4999, 2.5, 1), list(range(0, 4999, 600))[:9], 20, ld=ld, offset=offset)


@pytest.mark.parametrize("n", [40, 3000, 40000, 128256])
def test_equal_logits(n):
    """All equal; all equal but one; sorted both ways; two values only."""
    x = torch.zeros(5, n)
    x[1, n // 2] = 1.0
    x[2] = torch.arange(n) / n
    x[3] = -torch.arange(n) / n
    x[4] = (torch.arange(n) % 3 == 1).float()
    _check(x, [n - 1, 3, 0, n - 2, n // 2], 32)
    _check(x, [0, n // 2, n - 1, 5, 1], 5)


def test_signed_zeros_are_equal():
    x = torch.zeros(2, 700)
    x[0, ::2] = -0.0
    x[1, 1::2] = -0.0
    _check(x, [699, 3], 8)


@pytest.mark.parametrize("n", [600, 32000, 128256])
@pytest.mark.parametrize("left", [1, 3, 40])
def test_banned_logits(n, left):
    """All but a few are -infinity, banned ones among the tokens asked for and the alternatives."""
    x = torch.full((4, n), -math.inf)
    g = torch.Generator().manual_seed(left)
    for i in range(4):
        x[i, torch.randperm(n, generator=g)[:left]] = 3.0 * torch.randn(left, generator=g)
    token = [int(x[0].argmax()), int((x[1] == -math.inf).nonzero()[0]), n - 1, 0]
    _check(x, token, 20)


def test_extreme_values():
    """Numbers at the ends of the range: differences that overflow, the least numbers, one logit far above the others."""
    big = torch.finfo(torch.float32).max
    x = torch.zeros(5, 3000)
    x[0, 7], x[0, 8], x[0, 9] = big, -big, big
    x[1] = 1e-45 * (torch.arange(3000) % 5).float()
    x[2] = -1000.0
    x[2, 2999] = 1000.0
    x[3] = big
    x[4, 100] = 14.0
    _check(x, [8, 2, 2999, 5, 100], 10)


def test_infinite_logits_share_evenly():
    x = _logits(3, 5000, 2.0, 3)
    x[0, 11] = x[0, 4000] = math.inf
    x[1, 0] = math.inf
    got = _run(x, [4000, 5, 7], 3)
    assert abs(float(got["logprob"][0]) + math.log(2)) < 1e-6 and float(got["logprob"][1]) == -math.inf
    assert abs(float(got["entropy"][0]) - math.log(2)) < 1e-6 and float(got["entropy"][1]) == 0.0
    assert got["rank"][:2].tolist()[0] == 1 and got["top_idx"][0, :2].tolist() == [11, 4000] and int(got["top_idx"][1, 0]) == 0
    assert float(got["top_logprob"][0, 2]) == -math.inf
    assert math.isfinite(float(got["logprob"][2]))


def test_nan_and_nothing():
    """NaN makes its row NaN and comes last in the order; so does a row of nothing but -infinity; a token that is none has no probability."""
    n = 9000
    x = _logits(4, n, 2.0, 4)
    x[0, 5] = math.nan
    x[1] = -math.inf
    x[2, :] = math.nan
    x[2, 8000] = 1.0
    got = _run(x, [5, 3, 4, -1], 4)
    for name in ("logprob", "entropy"):
        assert got[name][:3].isnan().all(), name
    assert got["top_logprob"][:3].isnan().all()
    assert got["rank"].tolist() == [n - 1, 3, 5, -1]
    order = torch.where(x[0].isnan(), -math.inf, x[0]).sort(descending=True, stable=True).indices[:4].tolist()
    assert got["top_idx"][0].tolist() == order and got["top_idx"][1].tolist() == [0, 1, 2, 3] and got["top_idx"][2].tolist() == [8000, 0, 1, 2]
    assert math.isnan(float(got["logprob"][3])) and math.isfinite(float(got["entropy"][3]))
    assert int(_run(x[3:], [n], 0)["rank"][0]) == -1


@pytest.mark.parametrize("want", [("logprob",), ("entropy",), ("rank",), ("top_logprob",), ()])
def test_outputs_that_are_not_asked_for_stay(want):
    x = _logits(6, 3000, 2.0, 5)
    full, got = _run(x, range(6), 4), _run(x, range(6), 4, want=want)
    for name in ("logprob", "entropy", "rank", "top_logprob"):
        if name in want:
            assert torch.equal(got[name], full[name])
        else:
            assert (got[name] == (-9 if name == "rank" else 9.0)).all()
    assert torch.equal(got["top_idx"], full["top_idx"])


def test_a_row_does_not_depend_on_the_others():
    """The same row in steps of one and of many, where it has fewer CTAs: what is exact is the same, sums within their roundings."""
    x = _logits(200, 32000, 2.5, 6)
    many, one = _run(x, range(200), 8), _run(x[77:78], [77], 8)
    assert torch.equal(many["top_idx"][77], one["top_idx"][0]) and int(many["rank"][77]) == int(one["rank"][0])
    assert abs(float(many["logprob"][77] - one["logprob"][0])) <= UNIT * 256
    again = _run(x, range(200), 8)
    assert all(torch.equal(many[k], again[k]) for k in many)


def test_captured_and_on_another_stream():
    x = _logits(8, 20000, 2.5, 7)
    plain = _run(x, range(8), 5)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert torch.equal(_run(x, range(8), 5, stream=side.cuda_stream)["top_logprob"], plain["top_logprob"])
    ops, xd, tok = _ops(), x.cuda(), torch.arange(8, dtype=torch.int32, device="cuda")
    lp = torch.zeros(8, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.token_logprobs(xd.data_ptr(), 20000, 8, 20000, tok, torch.cuda.current_stream().cuda_stream, logprob=lp)
    xd.copy_(x.flip(0).cuda())
    tok.copy_(tok.flip(0))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(lp.cpu().flip(0), plain["logprob"])
