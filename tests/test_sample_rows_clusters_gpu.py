"""Draws of whole steps (Ops.sample_rows) by clusters of every size, at the ends of what a row may be; the numbers as in test_sample_rows_gpu.py."""
import pytest
import torch
from test_sample_rows_gpu import _check, _ops, _settings

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [2000, 4095, 8191, 16383, 32771])
def test_rows_while_other_kernels_run(n):
    """Clusters of 1, 2, 4, 8 and 16 CTAs that start while others' CTAs hold the machine: two streams of draws beside products give what one row after the other gives."""
    x = 2.5 * torch.randn(12, n, generator=torch.Generator().manual_seed(n))
    s = _settings(12, n)
    _check(x, *s)
    xs, dev = x.cuda(), [torch.tensor(v, dtype=torch.int32 if i == 1 else torch.float32, device="cuda") for i, v in enumerate(s)]
    ops, a = _ops(), torch.randn(2048, 2048, device="cuda")
    want = torch.empty(12, dtype=torch.int32, device="cuda")
    ops.sample_rows(xs.data_ptr(), n, 12, n, *dev, want, torch.cuda.current_stream().cuda_stream)
    streams, out = [torch.cuda.Stream() for _ in range(3)], torch.full((2, 60, 12), -5, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    for i in range(60):
        with torch.cuda.stream(streams[2]):
            a @ a
        for j in range(2):
            for row in range(0, 12, 4):                          # a few rows a launch: large clusters
                ops.sample_rows(xs[row:].data_ptr(), n, 4, n, *(d[row:] for d in dev), out[j, i, row:], streams[j].cuda_stream)
    torch.cuda.synchronize()
    assert (out == want).all()


@pytest.mark.parametrize("n", [720896, 720895, 655360 + 17])
def test_the_longest_rows(n):
    """All that a row may hold: 16 CTAs with 44 * 1024 logits each, and, where all are equal, a sum of 720896 * 2^44, as near to 2^64 as it gets. A weight that is not the largest is rounded to
    2^-45 of that, by chance up or down: sums of all are off by some 2^-45 sqrt(n) = 2^-35 of it at most, where a draw has thousands of them."""
    g = torch.Generator().manual_seed(n)
    x = 2.5 * torch.randn(8, n, generator=g)
    x[0] = x[1] = x[2] = -3.25
    x[3] = torch.where(torch.arange(n) % 2 == 0, 1.0, 0.5)
    t, k, p, m = [1.0, 0.7, 1.3, 1.0, 1.0, 0.9, 1.0, 0.8], [0, n // 3, 0, n - 1, 0, 300000, 0, 60], [1.0, 1.0, 0.9, 0.75, 1.0, 1.0, 0.95, 0.9], [0.0] * 6 + [1e-4, 0.0]
    _check(x, t, k, p, m, [0.999999, 0.5, 0.0, 0.3, 0.77, 0.123456, 0.4, 0.9])
    _check(x, [1e30] * 8, [0] * 8, [1.0] * 8, [0.0] * 8, [(i + 0.5) / 8 for i in range(8)])


@pytest.mark.parametrize("overlap", [False, True])
def test_captured_behind_the_kernel_that_writes_the_rows(overlap):
    """Draws from what an attention leaves, their kernel resident early or not, the step replayed: what the calls give one by one."""
    from test_kv8_attention_gpu import _case, _workspace
    ops, heads, kv_heads, dim = _ops(), 32, 8, 128
    step, q, k, v = _case([(300, 1), (64, 1), (4000, 1), (7, 1)], heads, kv_heads, dim)
    ws, out = _workspace(ops, step, heads, kv_heads, dim, dim), torch.empty(4, heads * dim, device="cuda")
    idx = torch.full((4,), -5, dtype=torch.int32, device="cuda")
    p, u = torch.full((4,), 0.9, device="cuda"), torch.tensor([0.1, 0.4, 0.7, 0.95], device="cuda")

    def calls(st):
        ops.attention8(step.b, q.data_ptr(), heads * dim, heads, kv_heads, dim, dim, dim ** -0.5, *k, *v, step.n_pages, ws, st, out=out, ldo=heads * dim)
        ops.sample_rows(out.data_ptr(), heads * dim, 4, heads * dim, None, None, p, None, u, idx, st)

    calls(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want, side, graph = idx.clone(), torch.cuda.Stream(), torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph, stream=side):
        calls(side.cuda_stream)
    if overlap:
        assert ops.overlap(graph.raw_cuda_graph()) > 0
    graph.instantiate()
    for _ in range(20):
        out.fill_(0.0)
        idx.fill_(-5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(idx, want)
