"""Bits of the attention over the 8-bit cache (Ops.attention8) where few of them are left: results in bf16, against those in fp32; scores of
any size; thousands of weights far below one."""
import math

import pytest
import torch
from kv8_testlib import BLOCK, Step, attention, cache_rows, codes_of, off, scale_for
from test_kv8_attention_gpu import BF16_BOUND, F32_BOUND, _case, _ops, _run, _want, _workspace

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("segs", [[(700, 1), (5, 1)], [(0, 500), (130, 333), (700, 40), (9, 1)], [(3000, 260), (17, 1)]], ids=["decode", "portions", "mixed"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (4, 4, 64), (6, 1, 128)])
@pytest.mark.parametrize("opts", [{}, dict(softcap=20.0), dict(window=100, keep_first=4)], ids=str)
def test_bf16_results_are_the_fp32_results_rounded(segs, heads, kv_heads, dim, opts):
    """Whatever else is asked for: a result of fewer bits is the same result."""
    step, q, k, v = _case(segs, heads, kv_heads, dim)
    fp32 = _run(step, q, k, v, heads, **opts)
    assert off(fp32, _want(step, q, k, v, heads, **opts)) < F32_BOUND
    alone, (both, both16) = _run(step, q, k, v, heads, bf16=True, **opts), _run(step, q, k, v, heads, both=True, **opts)
    assert torch.equal(both, fp32) and torch.equal(alone, both16)
    assert torch.equal(alone, fp32.to(torch.bfloat16))


@pytest.mark.parametrize("shift", [-40, -8, 0, 8, 9, 40])
@pytest.mark.parametrize("segs", [[(700, 1), (64, 1)], [(700, 40), (64, 1)]], ids=["decode", "portions"])
def test_large_scores_beside_scales_of_values(shift, segs):
    """Scores whose steps are as large as the exponents of value scales: no weight leaves fp16's range, and a key that wins by more than the steps takes all the weight."""
    heads, kv_heads, dim = 8, 2, 128
    step, q, k, v = _case(segs, heads, kv_heads, dim)
    v = (v[0], v[1] * 2.0 ** shift)
    for size in (2.0 ** e for e in range(18, 32)):
        got, at = _run(step, q * size, k, v, heads).double(), 0
        assert got.isfinite().all(), size
        for i, (p, n) in enumerate(segs):
            kk, vv = (cache_rows(step, *x, i).repeat_interleave(heads // kv_heads, 0) for x in (k, v))
            s = q[at:at + n].double().view(n, heads, dim).transpose(0, 1) @ kk.mT * dim ** -0.5
            s = s.masked_fill(torch.arange(p + n, device="cuda") > torch.arange(p, p + n, device="cuda")[:, None], -math.inf)
            (best, second), where = s.topk(2).values.unbind(-1), s.argmax(-1)
            sure = (best - second) * size > torch.clamp(2.0 ** -18 * best.abs() * size, min=60.0)
            want = vv.gather(1, where[..., None].expand(-1, -1, dim)).transpose(0, 1)
            have, sure = got[at:at + n].view(n, heads, dim), sure.T
            assert (((have - want).norm(dim=-1) / want.norm(dim=-1))[sure] < F32_BOUND).all(), (size, i)
            at += n


def _pool(x, step):
    """[pages][kv_heads][page][width] as the append leaves it."""
    x = x.view(*x.shape[:2], step.page // BLOCK, BLOCK, -1)
    scale = scale_for(x.abs().amax((-1, -2)))
    return codes_of(x / scale[..., None, None]).flatten(2, 3).cuda(), scale.cuda()


@pytest.mark.parametrize("gap", [10.0, 14.0, 18.0])
@pytest.mark.parametrize("sink", ["ordinary", "zero"])
@pytest.mark.parametrize("segs", [[(8000, 1), (3000, 1)], [(8000, 40), (3000, 3)]], ids=["decode", "portions"])
@pytest.mark.parametrize("dim", [64, 128])
def test_one_key_far_ahead_of_thousands(gap, sink, segs, dim):
    """A key whose score is `gap` above all others', whose weights are e^-gap then, and add up to N e^-gap: of values that share a sign, they are a part of the result, or all of it where the
    key's own value is 0. Then the key's score, of size gap, counts for every weight (2^-23 of it), and so does what the weights are rounded to: 2^-39 of the power of two above the largest
    at most, 2^-38 of the largest, by chance up or down, which N of them have 1 / sqrt(3 N) of on average; four times that."""
    heads, kv_heads = 8, 2
    step = Step(segs, 64)
    g = torch.Generator().manual_seed(int(gap))
    q = torch.randn(step.T, heads, dim, generator=g)
    q[..., 0] = gap * dim ** 0.5 / 16
    k, v = (torch.randn(step.n_pages, kv_heads, step.page, dim, generator=g) for _ in range(2))
    k, v = 0.1 * k, v.abs() + 0.5
    k[..., 0] = 0.0
    for i in range(len(segs)):
        page, row = int(step.table_np[i, 100 // step.page]), 100 % step.page
        k[page, :, row] = 0.0
        k[page, :, row, 0] = 16.0
        if sink == "zero":
            v[page, :, row] = 0.0
    q, k, v = q.flatten(1).cuda(), _pool(k, step), _pool(v, step)
    want, got, got16, at = _want(step, q, k, v, heads), _run(step, q, k, v, heads), _run(step, q, k, v, heads, bf16=True), 0
    for p, n in segs:
        bound = F32_BOUND + (gap * 2.0 ** -23 + 4 * 2.0 ** -38 * math.exp(gap) / math.sqrt(3 * p) if sink == "zero" else 0.0)
        assert off(got[at:at + n], want[at:at + n]) < bound, (p, n)
        assert off(got16[at:at + n], want[at:at + n]) < BF16_BOUND, (p, n)
        at += n


@pytest.mark.parametrize("segs", [[(300, 1), (64, 1)], [(300, 70), (64, 1)]], ids=["decode", "portions"])
@pytest.mark.parametrize("dim", [64, 128, 192])
def test_queries_at_the_end_of_fp32(segs, dim):
    """Queries of 2^126 to 2^128 over keys of the least scale and a score scale of 2^-38: scores of an ordinary size, as if both were scaled by powers of two."""
    heads, kv_heads = 8, 2
    step, q, k, v = _case(segs, heads, kv_heads, dim)
    k = (k[0], torch.full_like(k[1], 2.0 ** -100))
    q = torch.sign(q) * torch.clamp(q.abs(), 0.25, 0.999)
    ops, out, out16 = _ops(), torch.empty(step.T, heads * dim, device="cuda"), torch.empty(step.T, heads * dim, device="cuda", dtype=torch.bfloat16)
    ws = _workspace(ops, step, heads, kv_heads, dim, dim)
    kv = [(cache_rows(step, *k, i), cache_rows(step, *v, i)) for i in range(len(segs))]
    for up in (2.0 ** 126, 2.0 ** 127):
        x = (q * up * 2.0).clamp(-3.4e38, 3.4e38)
        want = attention(step, x, kv, heads, 2.0 ** -38)
        ops.attention8(step.b, x.data_ptr(), heads * dim, heads, kv_heads, dim, dim, 2.0 ** -38, *k, *v, step.n_pages, ws, torch.cuda.current_stream().cuda_stream, out=out, ldo=heads * dim,
                       out16=out16)
        assert off(out, want) < F32_BOUND and off(out16, want) < BF16_BOUND, up


@pytest.mark.parametrize("segs", [[(500, 1), (31, 1)], [(500, 40), (31, 3), (0, 70)]], ids=["decode", "portions"])
@pytest.mark.parametrize("opts", [dict(softcap=20.0), dict(softcap=20.0, window=50, keep_first=3), dict(softcap=2.0)], ids=str)
def test_hidden_rows_change_no_bit_of_capped_scores(segs, opts):
    """Rows behind a sequence or a window that hold zeros, the largest codes there are, or NaN; and what an earlier call has left in shared memory."""
    heads, kv_heads, dim = 6, 1, 128
    step, q, k, v = _case(segs, heads, kv_heads, dim)
    hidden = torch.ones(step.n_pages, step.page, dtype=torch.bool)
    for i, (p, n) in enumerate(segs):
        for y in range(p + n):
            if "window" not in opts or y > p - opts["window"] or y < opts["keep_first"]:
                hidden[int(step.table_np[i, y // step.page]), y % step.page] = False
    loud, results = _case([(900, 200)], heads, kv_heads, dim, seed=3), []
    for code in (0x00, 0x7e, 0x7f, 0x00):
        pools = []
        for pool, scale in (k, v):
            codes = pool.view(torch.uint8).clone()
            codes[hidden.cuda()[:, None, :, None].expand_as(codes)] = code
            pools.append((codes.view(torch.float8_e4m3fn), scale))
        results.append(_run(step, q, *pools, heads, **opts))
        _run(loud[0], loud[1] * 100, *loud[2:], heads)
    assert all(torch.equal(r, results[0]) for r in results[1:])
