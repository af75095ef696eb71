"""Attention over the 8-bit cache (Ops.attention8) against float64 on the cache's own values. Results in fp32: scores and weights carry 22 bits or more, sums are fp32; a score's
error is some 2^-24 of the sum of |q k| * scale (about 10 here), its weight's the same: 4e-6 of the norm. Results in bf16 are rounded by 2^-9 of a value on average of half that,
behind operands of 11 bits (2^-12 of the sum's norm each): 2^-8 of the norm."""
import math

import pytest
import torch
from kv8_testlib import Step, attention, cache_rows, off, random_pool

pytestmark = pytest.mark.gpu

F32_BOUND, BF16_BOUND = 4e-6, 2.0 ** -8


def _ops():
    from simplellminference_b200.config import BF16
    from simplellminference_b200.seqops import Ops
    return Ops(BF16)


def _case(segs, heads, kv_heads, dk, dv=None, page=64, seed=0, spread=1.0, **kw):
    step = Step(segs, page, seed=seed, **kw)
    g = torch.Generator().manual_seed(seed + 5)
    q = torch.randn(step.T, heads * dk, generator=g).cuda()
    return step, q, random_pool(step, kv_heads, dk, seed + 6, 0.3 * spread), random_pool(step, kv_heads, dv or dk, seed + 7, spread)


def _workspace(ops, step, heads, kv_heads, dk, dv):
    return torch.zeros(ops.attention8_ws_bytes(step.b, heads, kv_heads, dk, dv), dtype=torch.uint8, device="cuda")


def _run(step, q, k, v, heads, bf16=False, both=False, ws=None, ops=None, ldq=None, q_ptr=None, **opts):
    ops, kv_heads, dk, dv = ops or _ops(), k[0].shape[1], k[0].shape[3], v[0].shape[3]
    ws = _workspace(ops, step, heads, kv_heads, dk, dv) if ws is None else ws
    out = torch.full((step.b.T, heads * dv), math.nan, device="cuda") if both or not bf16 else None
    out16 = torch.full((step.b.T, heads * dv), math.nan, device="cuda", dtype=torch.bfloat16) if both or bf16 else None
    ops.attention8(step.b, q_ptr or q.data_ptr(), ldq or q.stride(0), heads, kv_heads, dk, dv, dk ** -0.5, *k, *v, step.n_pages, ws, torch.cuda.current_stream().cuda_stream, out=out,
                   ldo=heads * dv, out16=out16, opts=ops.attention_options(**opts) if opts else None)
    torch.cuda.synchronize()
    return (out, out16) if both else out16 if bf16 else out


def _want(step, q, k, v, heads, **opts):
    kv = [(cache_rows(step, *k, i), cache_rows(step, *v, i)) for i in range(len(step.segs))]
    return attention(step, q, kv, heads, k[0].shape[3] ** -0.5, **opts)


def _check(step, q, k, v, heads, by_segment=True, **opts):
    want = _want(step, q, k, v, heads, **opts)
    for bf16, bound in ((False, F32_BOUND), (True, BF16_BOUND)):
        got = _run(step, q, k, v, heads, bf16=bf16, **opts)
        at = 0
        for p, n in step.segs:
            assert off(got[at:at + n], want[at:at + n]) < bound, (bf16, p, n)
            at += n


DECODE = [[(0, 1)], [(31, 1)], [(32, 1)], [(7999, 1)], [(p, 1) for p in (500, 0, 33, 97, 1000, 63, 64)], [(i * 61 % 700, 1) for i in range(70)]]
PORTIONS = [[(0, 2)], [(0, 33)], [(0, 128)], [(0, 500), (130, 333), (700, 40), (9, 1)], [(3000, 65), (17, 1), (2500, 1), (0, 1)], [(90, 3), (0, 31), (1, 32)]]
HEADS = [(8, 2, 128, 128), (4, 4, 64, 64), (32, 4, 64, 64), (6, 2, 128, 128), (5, 1, 128, 128), (16, 1, 64, 64), (2, 1, 128, 64)]


def _ids(s):
    return f"{len(s)}x{sum(n for _, n in s)}_{s[0][0]}"


@pytest.mark.parametrize("segs", DECODE + PORTIONS, ids=_ids)
@pytest.mark.parametrize("heads,kv_heads,dk,dv", HEADS)
def test_against_float64(segs, heads, kv_heads, dk, dv):
    _check(*_case(segs, heads, kv_heads, dk, dv), heads)


@pytest.mark.parametrize("dk,dv", [(48, 48), (80, 96), (256, 256), (16, 240), (192, 128)])
@pytest.mark.parametrize("segs", [DECODE[4], PORTIONS[3]], ids=["decode", "portions"])
def test_other_widths(dk, dv, segs):
    _check(*_case(segs, 6, 2, dk, dv, page=96), 6)


OPTIONS = [dict(window=100), dict(window=1), dict(window=40, keep_first=70), dict(softcap=2.0, window=257), dict(slopes=True), dict(chunk=100), dict(softcap=20.0), dict(window=33, keep_first=1)]


@pytest.mark.parametrize("o", OPTIONS, ids=str)
@pytest.mark.parametrize("segs", [DECODE[4], PORTIONS[3]], ids=["decode", "portions"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 2, 128, 32), (3, 3, 64, 160)])
def test_options(o, segs, heads, kv_heads, dim, page):
    step, q, k, v = _case(segs, heads, kv_heads, dim, page=page)
    if "slopes" in o:
        slopes = 0.01 * torch.arange(1, heads + 1, device="cuda").float()
        want = _want(step, q, k, v, heads, slopes=slopes)
        assert off(_run(step, q, k, v, heads, slopes=slopes), want) < F32_BOUND and off(_run(step, q, k, v, heads, bf16=True, slopes=slopes), want) < BF16_BOUND
    else:
        _check(step, q, k, v, heads, **o)


@pytest.mark.parametrize("segs", [[(2000, 1), (70, 1)], [(2000, 70), (70, 1)]], ids=["decode", "portions"])
def test_scales_far_apart(segs):
    """Blocks of values up to 2^60 and down to 2^-60 of the others: what the result is made of keeps its bits."""
    heads, kv_heads, dim = 8, 2, 128
    step, q, k, v = _case(segs, heads, kv_heads, dim)
    e = torch.randint(-60, 61, v[1].shape, generator=torch.Generator().manual_seed(1)).cuda()
    v = (v[0], v[1] * torch.exp2(e.float()))
    want = _want(step, q, k, v, heads)
    got = _run(step, q, k, v, heads)
    assert off(got, want) < F32_BOUND
    assert (((got.double() - want).norm(dim=1) / want.norm(dim=1)) < 2e-5).all()
    v = (v[0], torch.full_like(v[1], 2.0 ** -100))                    # and all of them tiny
    want = _want(step, q, k, v, heads)
    assert off(_run(step, q, k, v, heads), want) < F32_BOUND
    # queries of any size: scores stay as they are when keys are as small as queries are large
    k = (k[0], k[1] * 2.0 ** -40)
    assert off(_run(step, q * 2.0 ** 40, k, v, heads), want) < F32_BOUND


@pytest.mark.parametrize("segs", [[(500, 1), (31, 1), (64, 1)], [(500, 40), (31, 2), (64, 1)]], ids=["decode", "portions"])
@pytest.mark.parametrize("bf16", [False, True])
def test_hidden_rows_may_hold_anything(segs, bf16):
    """NaN codes in rows behind a sequence, behind a window and in other sequences' pages change nothing."""
    heads, kv_heads, dim = 8, 2, 128
    step, q, k, v = _case(segs, heads, kv_heads, dim)
    for opts in ({}, dict(window=50, keep_first=3)):
        want = _run(step, q, k, v, heads, bf16=bf16, **opts)
        hidden = torch.ones(step.n_pages, step.page, dtype=torch.bool)
        for i, (p, n) in enumerate(segs):
            for y in range(p + n):
                if not opts or y > p - opts["window"] or y < opts["keep_first"]:
                    hidden[int(step.table_np[i, y // step.page]), y % step.page] = False
        wild = []
        for pool, scale in (k, v):
            codes = pool.view(torch.uint8).clone()
            codes[hidden.cuda()[:, None, :, None].expand_as(codes)] = 0x7f
            wild.append((codes.view(torch.float8_e4m3fn), scale))
        assert torch.equal(_run(step, q, *wild, heads, bf16=bf16, **opts), want)


@pytest.mark.parametrize("segs", [[(500, 1)], [(500, 40)]], ids=["decode", "portions"])
@pytest.mark.parametrize("bf16", [False, True])
def test_nan_where_it_is_seen(segs, bf16):
    """A NaN value reaches its column of the tokens that see it, a NaN key all columns; earlier tokens of the portion, which do not, stay as they are."""
    heads, kv_heads, dim = 8, 2, 128
    step, q, k, v = _case(segs, heads, kv_heads, dim)
    last = sum(segs[0]) - 1
    for at in (100, last, last - segs[0][1] + 1):
        for pool, key in ((v[0], False), (k[0], True)):
            codes = pool.view(torch.uint8)
            where = (int(step.table_np[0, at // step.page]), 1, at % step.page, 5)
            kept = int(codes[where])
            codes[where] = 0x7f
            got, want = _run(step, q, k, v, heads, bf16=bf16), _want(step, q, k, v, heads)
            codes[where] = kept
            assert torch.equal(got.isnan(), want.isnan()), (at, key)
            fine = ~want.isnan()
            assert off(got[fine], want[fine]) < (BF16_BOUND if bf16 else F32_BOUND)


@pytest.mark.parametrize("segs", [[(100, 1), (5, 1)], [(100, 3), (5, 1)]], ids=["decode", "portions"])
def test_pages_that_are_not_there(segs):
    """Keys without a page are hidden; a token all of whose keys are gives zeros."""
    heads, kv_heads, dim = 4, 2, 64
    step, q, k, v = _case(segs, heads, kv_heads, dim, page=32)
    kv = []
    for i in range(2):
        kv.append([cache_rows(step, *k, i), cache_rows(step, *v, i)])
    step.dev["block_table"][0, 1] = -1
    step.dev["block_table"][0, 2] = 10 ** 6
    step.dev["block_table"][1, 0] = -7
    got = _run(step, q, k, v, heads)
    assert (got[segs[0][1]:] == 0).all()
    n, p = segs[0][1], segs[0][0]
    keep = torch.tensor([y < 32 or y >= 96 for y in range(p + n)], device="cuda")
    for i in range(n):
        for h in range(heads):
            kk, vv = kv[0][0][h // 2], kv[0][1][h // 2]
            s = (kk @ q[i, h * dim:(h + 1) * dim].double() * dim ** -0.5).masked_fill(~keep | (torch.arange(p + n, device="cuda") > p + i), -math.inf)
            assert off(got[i, h * dim:(h + 1) * dim], torch.softmax(s, 0) @ vv) < F32_BOUND


def test_listed_tiles_only():
    """Rows of tokens in no listed tile stay as they are."""
    heads, kv_heads, dim = 8, 2, 128
    segs = [(0, 130), (300, 1), (64, 70)]
    step, q, k, v = _case(segs, heads, kv_heads, dim, tiles=[(0, 32), (0, 128), (2, 0)])
    got, want = _run(step, q, k, v, heads), _want(step, q, k, v, heads)
    rows = torch.zeros(step.T, dtype=torch.bool, device="cuda")
    rows[32:64] = rows[128:130] = rows[131:163] = True
    assert got[~rows].isnan().all() and off(got[rows], want[rows]) < F32_BOUND


def test_rows_of_any_stride_and_both_results():
    heads, kv_heads, dim = 8, 2, 64
    for segs in ([(500, 1), (31, 1)], [(100, 50), (31, 1)]):
        step, q, k, v = _case(segs, heads, kv_heads, dim)
        want = _want(step, q, k, v, heads)
        wide = torch.zeros(step.T, heads * dim + 7, device="cuda")
        wide[:, 3:3 + heads * dim] = q
        out, out16 = _run(step, wide, k, v, heads, both=True, q_ptr=wide.data_ptr() + 12)
        assert off(out, want) < F32_BOUND and torch.equal(out.to(torch.bfloat16), out16)


def test_one_workspace_many_calls():
    """The workspace of the largest step serves every step, in any order, captured or not; results are the same every time."""
    ops, heads, kv_heads, dim = _ops(), 8, 2, 128
    cases = [_case(s, heads, kv_heads, dim, seed=i) for i, s in enumerate(([(7000, 1), (10, 1)], [(500, 200), (3, 1)], [(i * 97 % 900, 1) for i in range(40)], [(3000, 64)]))]
    ws = max((_workspace(ops, c[0], heads, kv_heads, dim, dim) for c in cases), key=lambda t: t.numel())
    first = [_run(*c, heads, ws=ws, ops=ops) for c in cases]
    for c, f in zip(cases, first):
        assert off(f, _want(*c, heads)) < F32_BOUND
    side, graphs, outs = torch.cuda.Stream(), [], []
    for step, q, k, v in cases:
        out = torch.full((step.T, heads * dim), math.nan, device="cuda")
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=side):
            ops.attention8(step.b, q.data_ptr(), q.stride(0), heads, kv_heads, dim, dim, dim ** -0.5, *k, *v, step.n_pages, ws, side.cuda_stream, out=out, ldo=heads * dim)
        graphs.append(g)
        outs.append(out)
    for i in (0, 1, 2, 3, 3, 2, 0, 1, 0):
        outs[i].fill_(math.nan)
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i], first[i]), i


def test_append_then_attention_then_draw():
    """The three operators one behind the other, as a server's step has them: what the cache takes in is what the attention reads."""
    ops, heads, kv_heads, dim, vocab = _ops(), 8, 2, 128, 1000
    g = torch.Generator().manual_seed(11)
    segs = [(0, 70), (64, 1), (130, 1)]
    step = Step(segs, 64)
    k, v = random_pool(step, kv_heads, dim, 1), random_pool(step, kv_heads, dim, 2)
    x = torch.randn(step.T, (heads + 2 * kv_heads) * dim, generator=g).cuda()
    head = torch.randn(vocab, heads * dim, generator=g).cuda() / 8
    freq = (10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)).cuda()
    angles = torch.empty(step.T, 64, 2, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    ops.angles(step.b, freq, 64, angles, st)
    q, at, row = torch.empty(step.T, heads * dim, device="cuda"), x.data_ptr(), x.stride(0)
    ops.rotary_kv8(step.b, at, row, heads, dim, at + 4 * heads * dim, row, kv_heads, at + 4 * (heads + kv_heads) * dim, row, dim, angles, 64, 1, q.data_ptr(), heads * dim, *k, *v,
                   step.n_pages, st)
    out = torch.empty(step.T, heads * dim, device="cuda")
    ops.attention8(step.b, q.data_ptr(), heads * dim, heads, kv_heads, dim, dim, dim ** -0.5, *k, *v, step.n_pages, _workspace(ops, step, heads, kv_heads, dim, dim), st, out=out,
                   ldo=heads * dim)
    last = torch.tensor([69, 70, 71], device="cuda")
    logits = out[last] @ head.T
    u, idx = torch.tensor([0.1, 0.5, 0.9], device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")
    ops.sample_rows(logits.data_ptr(), vocab, 3, vocab, None, None, None, None, u, idx, st)
    # in float64, from the queries and the cache as they are, which the append's own tests check; keys of the portion are there within a code's rounding
    want = _want(step, q, k, v, heads)
    assert off(out, want) < F32_BOUND
    fresh = cache_rows(step, *k, 0)[:, :70]
    z = torch.view_as_complex(x[:70, heads * dim:(heads + kv_heads) * dim].double().view(70, kv_heads, 2, 64).transpose(2, 3).contiguous())
    turn = torch.polar(torch.ones(70, 64, dtype=torch.float64, device="cuda"), torch.arange(70, device="cuda").double()[:, None] * freq)
    keys = torch.view_as_real(z * turn[:, None]).transpose(2, 3).flatten(2).transpose(0, 1)
    assert off(fresh, keys) < 2.0 ** -4
    p = torch.softmax(logits.double(), -1).cumsum(-1)
    assert idx.tolist() == [(p[i] <= float(u[i])).sum().item() for i in range(3)]


@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 29, 2.0 ** 34, 2.0 ** 60])
@pytest.mark.parametrize("segs", [[(700, 1), (64, 1)], [(700, 40), (64, 1)]], ids=["decode", "portions"])
def test_scores_of_any_size(size, segs):
    """Scores of up to 2^60: fp32 gives each to 2^-22 of itself, so that the largest wins by more than its error wherever it is 2^-20 of itself ahead; it takes all the weight."""
    heads, kv_heads, dim = 8, 2, 128
    step, q, k, v = _case(segs, heads, kv_heads, dim)
    got, at = _run(step, q * size, k, v, heads).double(), 0
    for i, (p, n) in enumerate(segs):
        kk, vv = cache_rows(step, *k, i), cache_rows(step, *v, i)
        for j in range(n):
            for h in range(heads):
                s = kk[h // 4][:p + j + 1] @ q[at + j, h * dim:(h + 1) * dim].double() * dim ** -0.5
                best, second = s.topk(2).values.tolist()
                if (best - second) * size > max(40.0, 2.0 ** -18 * abs(best) * size):
                    assert off(got[at + j, h * dim:(h + 1) * dim], vv[h // 4][int(s.argmax())]) < F32_BOUND, (i, j, h)
        at += n


def test_a_step_that_is_not_of_single_tokens_is_reported():
    """Two segments, two tokens, but both in one of them."""
    from simplellminference_b200 import _lib
    heads, kv_heads, dim = 4, 2, 64
    step, q, k, v = _case([(100, 1), (5, 1)], heads, kv_heads, dim)
    step.dev["seg_len"].copy_(torch.tensor([2, 0]))
    got = _run(step, q, k, v, heads)
    assert _lib.load().sllm_status() == _lib.EINVAL and got.isnan().all()
