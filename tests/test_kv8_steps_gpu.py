"""Steps of a server at the ends of what Ops.attention8 takes: long contexts whose sums are added up outside the tensor core, more segments than a CTA or the plan keeps at hand, two
streams at once, a step captured with overlapping kernels. Against float64 with the bounds of test_kv8_attention_gpu.py (the same numbers are rounded, whoever adds them), or bit by bit
against the same call made otherwise."""
import math

import pytest
import torch
from kv8_testlib import Step, attention, cache_rows, off, random_pool
from test_kv8_attention_gpu import BF16_BOUND, F32_BOUND, _case, _check, _ops, _run, _want, _workspace

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("segs", [[(6000, 256)], [(0, 2048)], [(3000, 130), (5000, 1), (0, 900)]], ids=["behind_a_context", "prompt", "mixed"])
def test_long_portions(segs):
    """More key tiles a CTA than its sums stay in tensor memory for."""
    _check(*_case(segs, 32, 8, 128), 32)


def test_nan_in_a_long_context():
    """Seen through one of many parts of an item."""
    step, q, k, v = _case([(6000, 96)], 32, 8, 128)
    for at in (100, 5999, 6050):
        codes = v[0].view(torch.uint8)
        where = (int(step.table_np[0, at // step.page]), 3, at % step.page, 70)
        kept = int(codes[where])
        codes[where] = 0xff
        want = _want(step, q, k, v, 32)
        for bf16 in (False, True):
            got = _run(step, q, k, v, 32, bf16=bf16)
            assert torch.equal(got.isnan(), want.isnan()), (at, bf16)
            assert off(got[~want.isnan()], want[~want.isnan()]) < (BF16_BOUND if bf16 else F32_BOUND)
        codes[where] = kept


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 16, 64), (4, 4, 128)])
def test_many_short_segments(heads, kv_heads, dim):
    """1200 runs of queries: more than their masks fit shared memory for, and (16 head sets) more items a CTA than are kept there."""
    _check(*_case([(i * 37 % 50, 2 + i % 3) for i in range(1200)], heads, kv_heads, dim, page=32), heads)


@pytest.mark.parametrize("each", [2, 1])
def test_more_segments_than_the_plan_takes(each):
    """4200 segments: of two tokens they are the general kernel's, beside single ones."""
    _check(*_case([(i % 40, each if i % 3 else 1) for i in range(4200)], 2, 1, 64, page=32), 2)


def test_many_single_tokens():
    """More tiles than the kernel for single tokens keeps at hand, two of them empty."""
    segs = [(i * 53 % 600, 1) for i in range(300)]
    step, q, k, v = _case(segs, 12, 1, 128, page=32)
    step.dev["block_table"][7] = -1
    step.dev["block_table"][299] = 10 ** 7
    got, want = _run(step, q, k, v, 12), _want(step, q, k, v, 12)
    assert (got[[7, 299]] == 0).all()
    rows = torch.ones(300, dtype=torch.bool)
    rows[[7, 299]] = False
    assert off(got[rows], want[rows]) < F32_BOUND


def test_two_segments_of_one_sequence():
    """Two portions that read the same pages."""
    heads, kv_heads, dim = 8, 2, 128
    step, q, k, v = _case([(200, 60), (130, 1), (64, 33)], heads, kv_heads, dim, slots=[0, 0, 0])
    kv = (cache_rows(step, *k, 0), cache_rows(step, *v, 0))
    want = attention(step, q, [tuple(x[:, :p + n] for x in kv) for p, n in step.segs], heads, dim ** -0.5)
    for bf16, bound in ((False, F32_BOUND), (True, BF16_BOUND)):
        assert off(_run(step, q, k, v, heads, bf16=bf16), want) < bound


@pytest.mark.parametrize("cap", [3.0, 30.0])
@pytest.mark.parametrize("size", [0.5, 4.0, 40.0])
def test_capped_scores_on_both_sides_of_the_cap(cap, size):
    """Scores up to ten times the cap and far below it. A capped score's error is the score's own at most (the slope of tanh is 1 at most), which grows with the queries, and that of tanh,
    2.2e-7 of 1 at its worst place, behind two products rounded by 2^-24 each: 4e-7 of the cap."""
    step, q, k, v = _case([(100, 70), (300, 1)], 8, 2, 128)
    q = q * size
    want = _want(step, q, k, v, 8, softcap=cap)
    assert off(_run(step, q, k, v, 8, softcap=cap), want) < F32_BOUND * max(1.0, size) + 4e-7 * cap


def test_two_streams_at_once():
    """Two steps on two streams, each with a workspace of its own, give what they give alone."""
    ops, heads, kv_heads, dim = _ops(), 32, 8, 128
    cases = [_case(s, heads, kv_heads, dim, seed=i) for i, s in enumerate(([(4000, 200), (700, 1)], [(5000, 1), (0, 700), (90, 1)]))]
    want = [_run(*c, heads, ops=ops) for c in cases]
    ws = [_workspace(ops, c[0], heads, kv_heads, dim, dim) for c in cases]
    outs = [[torch.full((c[0].T, heads * dim), math.nan, device="cuda") for _ in range(8)] for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for i in range(8):
        for (step, q, k, v), w, out, st in zip(cases, ws, outs, streams):
            ops.attention8(step.b, q.data_ptr(), q.stride(0), heads, kv_heads, dim, dim, dim ** -0.5, *k, *v, step.n_pages, w, st.cuda_stream, out=out[i], ldo=heads * dim)
    torch.cuda.synchronize()
    for out, w in zip(outs, want):
        assert all(torch.equal(o, w) for o in out)


@pytest.mark.parametrize("overlap", [False, True])
def test_layers_captured_one_behind_the_other(overlap):
    """Append, attention and append into another layer's pools, twice in one captured step over one workspace, its kernels resident early or not: bit by bit what the calls give one by one."""
    ops, heads, kv_heads, dim = _ops(), 8, 2, 128
    step = Step([(300, 80), (64, 1), (0, 33)], 64)
    g = torch.Generator().manual_seed(4)
    x = torch.randn(step.T, (heads + 2 * kv_heads) * dim, generator=g).cuda()
    angles = torch.randn(step.T, 64, 2, generator=g).cuda()
    pools = [[random_pool(step, kv_heads, dim, 10 * i + j) for j in range(2)] for i in range(2)]
    start = [[(a.clone(), b.clone()) for a, b in layer] for layer in pools]
    ws = _workspace(ops, step, heads, kv_heads, dim, dim)
    q = [torch.empty(step.T, heads * dim, device="cuda") for _ in range(2)]
    out = [torch.empty(step.T, heads * dim, device="cuda") for _ in range(2)]

    def layers(st):
        for i, (k, v) in enumerate(pools):
            at, row = x.data_ptr(), x.stride(0)
            ops.rotary_kv8(step.b, at, row, heads, dim, at + 4 * heads * dim, row, kv_heads, at + 4 * (heads + kv_heads) * dim, row, dim, angles, 64, 1, q[i].data_ptr(), heads * dim, *k, *v,
                           step.n_pages, st)
            ops.attention8(step.b, q[i].data_ptr(), heads * dim, heads, kv_heads, dim, dim, dim ** -0.5, *k, *v, step.n_pages, ws, st, out=out[i], ldo=heads * dim)

    def again():
        for layer, was in zip(pools, start):
            for (a, b), (c, d) in zip(layer, was):
                a.copy_(c)
                b.copy_(d)
        torch.cuda.synchronize()

    layers(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want = [o.clone() for o in out]
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph, stream=side):
        layers(side.cuda_stream)
    if overlap:
        assert ops.overlap(graph.raw_cuda_graph()) > 0
    graph.instantiate()
    for _ in range(5):
        again()
        for o in out:
            o.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(out, want))


@pytest.mark.parametrize("opts", [{}, dict(window=40, keep_first=3), dict(softcap=20.0), dict(chunk=50)], ids=str)
@pytest.mark.parametrize("segs", [[(300, 1), (64, 1), (0, 1)], [(300, 70), (64, 1), (0, 33)]], ids=["decode", "portions"])
def test_queries_and_keys_of_zero(segs, opts):
    """Both scales are the least there are, and their product is below fp32's range: every score is 0, every visible value counts the same; with a query of ordinary size, too."""
    step, q, k, v = _case(segs, 8, 2, 128)
    for pool in ((torch.zeros_like(k[0].view(torch.uint8)).view(k[0].dtype), torch.full_like(k[1], 2.0 ** -100)), k):
        for x in (torch.zeros_like(q), q * 2.0 ** -120, q):
            want = _want(step, x, pool, v, 8, **opts)
            for bf16, bound in ((False, F32_BOUND), (True, BF16_BOUND)):
                assert off(_run(step, x, pool, v, 8, bf16=bf16, **opts), want) < bound
