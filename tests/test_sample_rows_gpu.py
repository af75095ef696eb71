"""Draws from given random numbers (Ops.sample_rows) against float64. Weights are multiples of 2^-44 of the largest: the borders of a draw are off by 2^-45 times the root of the
number of candidates at most, so that a draw that differs would need a random number within some 1e-12 of a border; the drawn one's probability is fp32 (2^-24 of it, and 2^-45 of the
largest weight: 2^-23 for those at least 2^-20 of it)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _ops():
    from simplellminference_b200.config import BF16
    from simplellminference_b200.seqops import Ops
    return Ops(BF16)


def _want(x, t=1.0, k=0, p=1.0, m=0.0, u=0.5):
    """(index, probability) of one row, in float64 on the CPU."""
    x = torch.where(x.isnan(), -math.inf, x.double())
    top, n = x.max(), x.numel()
    if top == -math.inf:
        return 0, 0.0
    if not t > 0:
        return int((x == top).nonzero()[0]), 1.0
    w = torch.where(x == top, 1.0, torch.exp((x - top) / t) if top < math.inf else torch.zeros(()).double())
    alive = torch.ones(n, dtype=torch.bool)
    if 0 < k < n:
        alive = x >= x.sort(descending=True).values[k - 1]
    if 0 < p < 1:
        values, where = x[alive].unique(return_inverse=True)
        mass = torch.zeros(values.numel(), dtype=torch.float64).index_add_(0, where, w[alive]).flip(0).cumsum(0)
        alive = alive & (x >= values.flip(0)[int((mass < p * mass[-1]).sum())])
    if m > 0:
        alive = alive & (w >= min(m, 1.0))
    w = torch.where(alive, w, 0.0)
    run = w.cumsum(0)
    i = min(int((run <= min(max(u, 0.0), 1.0) * run[-1]).sum()), int(w.nonzero()[-1]))
    return i, float(w[i] / run[-1])


def _run(x, t=None, k=None, p=None, m=None, u=None, ld=None, prob=True, n=None):
    rows, n = x.shape[0], n or x.shape[1]
    dev = lambda v, dt=torch.float32: None if v is None else torch.tensor(v, dtype=dt, device="cuda")   # noqa: E731
    idx = torch.full((rows,), -5, dtype=torch.int32, device="cuda")
    pr = torch.full((rows,), math.nan, device="cuda") if prob else None
    held = [dev(t), dev(k, torch.int32), dev(p), dev(m), dev(u)]
    _ops().sample_rows(x.data_ptr(), ld or x.stride(0), rows, n, *held, idx, torch.cuda.current_stream().cuda_stream, prob=pr)
    torch.cuda.synchronize()
    return (idx.tolist(), pr.tolist()) if prob else idx.tolist()


def _f32(v):
    return float(torch.tensor(v, dtype=torch.float32))


def _check(x, t, k, p, m, u):
    got, prob = _run(x.cuda(), t, k, p, m, u)
    for i in range(x.shape[0]):
        want, pw = _want(x[i], _f32(t[i]), k[i], _f32(p[i]), _f32(m[i]), _f32(u[i]))
        assert got[i] == want, (i, got[i], want, t[i], k[i], p[i], m[i], u[i])
        assert abs(prob[i] - pw) <= 2.0 ** -23 * pw + 2.0 ** -44, i


def _settings(rows, seed):
    g = torch.Generator().manual_seed(seed)
    r = torch.rand(rows, 5, generator=g)
    which = [i % 6 for i in range(rows)]
    t = [0.0 if w == 5 else 0.3 + 1.7 * float(r[i, 0]) for i, w in enumerate(which)]
    k = [1 + int(100 * r[i, 1]) if w in (0, 1) else 0 for i, w in enumerate(which)]
    p = [0.5 + 0.5 * float(r[i, 2]) if w in (1, 2, 3) else 1.0 for i, w in enumerate(which)]
    m = [0.2 * float(r[i, 3]) if w in (3, 4) else 0.0 for i, w in enumerate(which)]
    return t, k, p, m, r[:, 4].tolist()


@pytest.mark.parametrize("rows,n", [(12, 1), (12, 2), (12, 31), (12, 500), (18, 4097), (1, 32000), (6, 50257), (40, 32000), (7, 128256), (300, 1000), (3, 300001)])
@pytest.mark.parametrize("spread", [0.05, 2.5, 12.0])
def test_rows_with_settings_of_their_own(rows, n, spread):
    x = spread * torch.randn(rows, n, generator=torch.Generator().manual_seed(n))
    _check(x, *_settings(rows, rows + n))


@pytest.mark.parametrize("n", [700, 32000, 128256])
def test_equal_logits(n):
    """Logits of eight bits: equal ones are in or out together; a row of one value; two values."""
    g = torch.Generator().manual_seed(n)
    x = (2.5 * torch.randn(18, n, generator=g)).to(torch.bfloat16).float()
    x[0], x[1] = 3.0, torch.where(torch.arange(n) % 3 == 0, 1.0, -1.0)
    x[6], x[7], x[8] = -2.0, x[1], -7.25
    _check(x, *_settings(18, 5))


def test_infinities_and_nan():
    x = torch.randn(18, 5000, generator=torch.Generator().manual_seed(1))
    x[:, ::3] = -math.inf
    x[:, 5] = math.nan
    x[3], x[4] = -math.inf, math.nan
    x[6, 100], x[7, 4000], x[7, 70] = math.inf, math.inf, math.inf
    x[9, 1:] = -math.inf
    x[10] = torch.finfo(torch.float32).min
    x[10, 77] = torch.finfo(torch.float32).max
    _check(x, *_settings(18, 2))


@pytest.mark.parametrize("base,step", [(0.0, 1e-30), (300.0, 0.0), (-1e30, 1e27), (1e-38, 1e-40)])
def test_logits_of_any_size(base, step):
    """Far from zero, far apart, closer together than their distance to the largest shows."""
    n = 3000
    x = (base + step * torch.randn(12, n, generator=torch.Generator().manual_seed(4), dtype=torch.float64)).float()
    if step == 0.0:
        x[:, :40] -= torch.arange(40) * 20.0
    t, k, p, m, u = _settings(12, 9)
    if abs(base) >= 1e30:
        t = [v * 1e27 for v in t]
    _check(x, t, k, p, m, u)


def test_edges_of_the_settings():
    x = 3 * torch.randn(1, 2000, generator=torch.Generator().manual_seed(8))
    for t, k, p, m, u in [(1.0, 1, 1.0, 0.0, 0.99), (1.0, 0, 1e-6, 0.0, 0.99), (1.0, 0, 1.0, 1.0, 0.99), (1.0, 0, 1.0, 5.0, 0.3), (1e-4, 0, 1.0, 0.0, 0.7), (1e4, 0, 1.0, 0.0, 0.7),
                          (1.0, 5000, 0.9, 0.0, 0.5), (1.0, -3, 0.0, -1.0, 0.5), (1.0, 2000, 2.0, 0.0, 0.5), (1.0, 1999, 1.0, 0.0, 0.0), (1.0, 0, 1.0, 0.0, 0.99999994),
                          (1.0, 0, 1.0, 0.0, 1.0), (1.0, 0, 1.0, 0.0, -1.0), (-1.0, 3, 0.5, 0.1, 0.5), (math.nan, 3, 0.5, 0.1, 0.5)]:
        _check(x, [t], [k], [p], [m], [u])


def test_rows_apart_and_without_settings():
    x = torch.full((5, 1009), 50.0)
    x[:, 2:1003] = torch.randn(5, 1001, generator=torch.Generator().manual_seed(3))
    u = [0.0, 0.2, 0.5, 0.9, 0.999]
    xs = x.cuda()
    idx = torch.empty(5, dtype=torch.int32, device="cuda")
    us = torch.tensor(u, device="cuda")
    _ops().sample_rows(xs.data_ptr() + 8, 1009, 5, 1001, None, None, None, None, us, idx, torch.cuda.current_stream().cuda_stream)
    assert idx.tolist() == [_want(x[i, 2:1003], u=_f32(u[i]))[0] for i in range(5)]


def test_draws_follow_the_distribution():
    """20000 evenly spaced numbers hit every candidate as often as its weight says, to within one."""
    x, n = torch.tensor([0.0, 1.0, -1.0, 2.0, 0.5]), 20000
    got, _ = _run(x.cuda().repeat(n, 1), u=[(i + 0.5) / n for i in range(n)])
    for i, w in enumerate(torch.softmax(x.double(), 0).tolist()):
        assert abs(got.count(i) - w * n) <= 1.01


def test_same_every_time_and_captured():
    x = 2.5 * torch.randn(64, 50000, generator=torch.Generator().manual_seed(6)).cuda()
    s = _settings(64, 3)
    first = _run(x, *s)
    assert all(_run(x, *s) == first for _ in range(3))
    dev = [torch.tensor(v, dtype=torch.int32 if i == 1 else torch.float32, device="cuda") for i, v in enumerate(s)]
    idx, prob, side, graph = torch.empty(64, dtype=torch.int32, device="cuda"), torch.empty(64, device="cuda"), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        _ops().sample_rows(x.data_ptr(), 50000, 64, 50000, *dev, idx, side.cuda_stream, prob=prob)
    graph.replay()
    torch.cuda.synchronize()
    assert (idx.tolist(), prob.tolist()) == first


@pytest.mark.parametrize("n", [900, 60000])
def test_temperatures_of_any_size(n):
    """Up to where a distance over the temperature, or the distance itself, leaves fp32's range; logits of -inf weigh nothing at any."""
    x = torch.randn(6, n, generator=torch.Generator().manual_seed(n))
    x[:, ::5] = -math.inf
    x[3], x[4] = x[3] * 1e37, torch.where(torch.arange(n) % 2 == 0, 3e38, -3e38)
    for t in (1e-38, 1e-30, 1e30, 1e37, 3e38):
        for p, m, k in ((1.0, 0.0, 0), (0.7, 0.0, 0), (0.9, 0.01, n // 3)):
            rows = [0, 1, 3] if t < 1e37 else [0, 1]
            _check(x[rows], [t] * len(rows), [k] * len(rows), [p] * len(rows), [m] * len(rows), [0.1, 0.6, 0.9][:len(rows)])


@pytest.mark.parametrize("n,grain", [(50257, 0.25), (128256, 2.0 ** -9), (20000, 1.0)])
def test_borders_in_crowded_places(n, grain):
    """Logits on a grid: hundreds and thousands of equal ones where top_k's and top_p's borders lie, together and with a min_p."""
    x = (2.5 * torch.randn(12, n, generator=torch.Generator().manual_seed(n)) / grain).round() * grain
    k = [0, 0, n // 2, n // 2, n // 7, 700, 0, 3000, n // 2, 0, n - 1, 129]
    p = [0.5, 0.99, 1.0, 0.9, 0.999, 0.8, 0.999999, 1.0, 0.3, 0.01, 0.95, 0.6]
    _check(x, [0.6 + 0.1 * i for i in range(12)], k, p, [0.0, 0.001, 0.0] * 4, [i / 12 for i in range(12)])
