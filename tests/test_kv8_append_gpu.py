"""Keys and values appended to the 8-bit cache (Ops.rotary_kv8): codes and scales bit for bit against the same roundings on the CPU (products, sums, the division by a power of two,
the rounding to e4m3), and the values against float64: e4m3 rounds by 2^-4 of a value at most, by 2^-10 scales where a code is subnormal, and turning in fp32 by 2^-22 of the pair."""
import math

import pytest
import torch
from kv8_testlib import BLOCK, Step, append, cache_rows, random_pool, turned

pytestmark = pytest.mark.gpu


def _ops():
    from simplellminference_b200.config import BF16
    from simplellminference_b200.seqops import Ops
    return Ops(BF16)


def _angles(step, n_freq, base=10000.0):
    freq = base ** (-torch.arange(max(n_freq, 1), dtype=torch.float64) / max(n_freq, 1))
    t = torch.tensor(step.tok_pos_np, dtype=torch.float64)[:, None] * freq
    return torch.stack([torch.cos(t), torch.sin(t)], -1).float()


def _call(step, x, heads, kv_heads, dk, dv, angles, n_freq, layout, kp, ks, vp, vs, in_place=False, pad=0, stream=None, n_pages=None):
    """x [T][heads * dk + kv_heads * (dk + dv) + pad] on the device."""
    ops, T, row = _ops(), x.shape[0], x.stride(0)
    out = x if in_place else torch.full((T, heads * dk), math.nan, device="cuda")
    at = x.data_ptr()
    dev_angles = angles.cuda().contiguous()
    ops.rotary_kv8(step.b, at, row, heads, dk, at + 4 * heads * dk, row, kv_heads, at + 4 * (heads + kv_heads) * dk, row, dv, dev_angles, n_freq, layout,
                   out.data_ptr(), out.stride(0), kp, ks, vp, vs, n_pages or step.n_pages, (stream or torch.cuda.current_stream()).cuda_stream)
    torch.cuda.synchronize()
    return out[:, :heads * dk]


def _case(segs, heads, kv_heads, dk, dv, page, seed=0, pad=0, scale=1.0):
    step = Step(segs, page, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    x = torch.randn(step.T, heads * dk + kv_heads * (dk + dv) + pad, generator=g) * scale
    return step, x, random_pool(step, kv_heads, dk, seed + 2), random_pool(step, kv_heads, dv, seed + 3)


def _parts(x, heads, kv_heads, dk, dv):
    T, a, b = x.shape[0], heads * dk, (heads + kv_heads) * dk
    return x[:, :a].reshape(T, heads, dk), x[:, a:b].reshape(T, kv_heads, dk), x[:, b:b + kv_heads * dv].reshape(T, kv_heads, dv)


def _check(step, x, heads, kv_heads, dk, dv, n_freq, layout, k, v, **how):
    angles = _angles(step, n_freq)
    q, kx, vx = _parts(x, heads, kv_heads, dk, dv)
    (kp, ks), (vp, vs) = k, v
    want_k, want_v = append(step, kp, ks, turned(kx, angles, n_freq, layout)), append(step, vp, vs, vx)
    got_q = _call(step, x.cuda(), heads, kv_heads, dk, dv, angles, n_freq, layout, kp, ks, vp, vs, **how)
    assert torch.equal(got_q.cpu(), turned(q, angles, n_freq, layout).flatten(1))
    for (pool, scale), (codes, scales) in (((kp, ks), want_k), ((vp, vs), want_v)):
        assert torch.equal(scale.cpu(), scales)
        assert torch.equal(pool.cpu().view(torch.uint8), codes)
    return angles


SEGS = [[(0, 1)], [(31, 1)], [(32, 1)], [(4000, 1)], [(0, 32)], [(0, 33)], [(17, 64)], [(5, 3), (0, 1), (63, 2), (700, 1)], [(p, 1) for p in range(70)],
        [(0, 200), (300, 37), (31, 1), (64, 129), (95, 2)], [(i * 37 % 200, 1 + i * 13 % 40) for i in range(45)]]


@pytest.mark.parametrize("segs", SEGS, ids=lambda s: f"{len(s)}x{sum(n for _, n in s)}")
@pytest.mark.parametrize("heads,kv_heads,dk,dv,page", [(8, 2, 128, 128, 64), (3, 3, 64, 64, 32), (6, 1, 96, 48, 96), (2, 2, 256, 16, 128)])
@pytest.mark.parametrize("layout", [0, 1])
def test_codes_scales_and_queries(segs, heads, kv_heads, dk, dv, page, layout):
    step, x, k, v = _case(segs, heads, kv_heads, dk, dv, page)
    _check(step, x, heads, kv_heads, dk, dv, dk // 2, layout, k, v)


@pytest.mark.parametrize("n_freq", [0, 1, 6, 16, 31])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("layout,pad", [(0, 0), (1, 3), (1, 4)])
def test_part_of_the_dimensions_turns(n_freq, in_place, layout, pad):
    step, x, k, v = _case([(3, 40), (100, 1)], 4, 2, 64, 64, 64, pad=pad)
    _check(step, x, 4, 2, 64, 64, n_freq, layout, k, v, in_place=in_place)


def test_values_in_float64():
    heads, kv_heads, dim = 8, 2, 128
    step, x, k, v = _case([(100000, 300), (9, 1)], heads, kv_heads, dim, dim, 64)
    angles = _angles(step, dim // 2, 500000.0)
    _call(step, x.cuda(), heads, kv_heads, dim, dim, angles, dim // 2, 1, *k, *v)
    a = torch.complex(angles[..., 0].double(), angles[..., 1].double())[:, None]
    z = torch.complex(*_parts(x, heads, kv_heads, dim, dim)[1].double().chunk(2, -1)) * a
    want, at = torch.cat([z.real, z.imag], -1), 0
    for i, (p, n) in enumerate(step.segs):
        got = cache_rows(step, *k, i)[:, p:].cpu().transpose(0, 1)
        w = want[at:at + n]
        ids = torch.tensor([[int(step.table_np[i, y // 64]), y % 64 // BLOCK] for y in range(p, p + n)])
        sc = k[1].cpu().double()[ids[:, 0], :, ids[:, 1]]
        pair = z.abs()[at:at + n].repeat(1, 1, 2)
        assert ((got - w).abs() <= 2.0 ** -4 * w.abs() + 2.0 ** -10 * sc[..., None] + 1.07 * 2.0 ** -22 * pair).all()
        at += n


def test_a_block_that_grows_token_by_token():
    """Each token sixteen times the last: the scale grows, the older rows move to it, and what comes out is what one append of all of them gives. A code of 2^-6 or more is not subnormal,
    and was larger before every move (scales only grow): it was rounded once, in both. Below, every move rounds to a step of 2^-9 again, by half of one at most, and the moves behind it make
    that 16 times smaller: less than (1/2) (1 + 1/16 + ...) < 0.54 steps in all, and half of one for the single rounding, so that two codes are one step apart at most."""
    kv_heads, dim, page = 2, 64, 32
    g = torch.Generator().manual_seed(3)
    x = torch.randn(6, kv_heads * dim * 3, generator=g) * 16.0 ** torch.arange(6)[:, None]
    step = Step([(0, 6)], page)
    whole = [random_pool(step, kv_heads, dim, i) for i in (1, 2)]
    single = [(p.clone(), s.clone()) for p, s in whole]
    angles = _angles(step, dim // 2)
    _call(step, x.cuda(), kv_heads, kv_heads, dim, dim, angles, dim // 2, 1, *whole[0], *whole[1])
    for i in range(6):
        one = Step([(i, 1)], page)
        one.dev["block_table"].copy_(step.dev["block_table"])
        _call(one, x[i:i + 1].cuda(), kv_heads, kv_heads, dim, dim, angles[i:i + 1], dim // 2, 1, *single[0], *single[1], n_pages=step.n_pages)
    for (a, sa), (b, sb) in zip(whole, single):
        assert torch.equal(sa, sb)
        va, vb = a.float()[int(step.table_np[0, 0]), :, :6], b.float()[int(step.table_np[0, 0]), :, :6]
        normal = va.abs() >= 2.0 ** -6
        assert int(normal.sum()) > normal.numel() // 4 and torch.equal(va[normal], vb[normal])
        assert (va - vb).abs().max() <= 2.0 ** -9 * 1.5           # (a whole number of steps: one)
        assert torch.equal(a.view(torch.uint8)[:, :, 6:], b.view(torch.uint8)[:, :, 6:])


@pytest.mark.parametrize("amax", [448.0, math.nextafter(448.0, 500.0), 1.75, 1.7500001, 2.0 ** -140, 0.0, 3.4028234e38, 2.0 ** -92, 2.0 ** -91.5])
def test_scales_at_their_borders(amax):
    kv_heads, dim = 1, 16
    step = Step([(0, 2)], 32)
    x = torch.zeros(2, 3 * dim)
    x[1, dim + 5] = x[0, 2 * dim + 3] = amax
    k, v = random_pool(step, 1, dim, 1), random_pool(step, 1, dim, 2)
    _check(step, x, 1, 1, dim, dim, 0, 0, k, v)
    if amax == 0.0:
        assert (k[1][int(step.table_np[0, 0])] == 2.0 ** -100).all()


def test_infinities_and_nan():
    """They become NaN codes, and the scale is that of the finite values."""
    step, x, k, v = _case([(10, 40)], 2, 2, 64, 64, 64)
    x[3, 2 * 64 + 7], x[5, 4 * 64 + 9], x[6, 4 * 64 + 1], x[39, 2 * 64 + 64] = math.inf, -math.inf, math.nan, math.nan
    angles = _angles(step, 0)
    want_k, want_v = (append(step, p, s, part) for (p, s), part in zip((k, v), _parts(x, 2, 2, 64, 64)[1:]))
    _call(step, x.cuda(), 2, 2, 64, 64, angles, 0, 0, *k, *v)
    for (pool, scale), (codes, scales) in ((k, want_k), (v, want_v)):
        assert torch.equal(scale.cpu(), scales)
        got, want = pool.cpu().float(), codes.view(torch.float8_e4m3fn).float()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    assert int(k[0].float().isnan().sum()) == 2 and int(v[0].float().isnan().sum()) == 2


def test_places_without_a_token_and_rows_of_others():
    """A step padded to more tokens than its segments have: their queries stay as they are, and no other page or row of the cache changes."""
    from simplellminference_b200 import _lib
    heads, kv_heads, dim = 4, 2, 64
    step, x, k, v = _case([(5, 3), (40, 1)], heads, kv_heads, dim, dim, 64)
    more = torch.cat([x, torch.full((3, x.shape[1]), 7.0)]).cuda()
    slot = torch.cat([step.dev["tok_slot"], torch.full((3,), -1, dtype=torch.int32, device="cuda")])
    pos = torch.cat([step.dev["tok_pos"], torch.zeros(3, dtype=torch.int32, device="cuda")])
    step.b.T, step.b.tok_slot, step.b.tok_pos = 7, slot.data_ptr(), pos.data_ptr()
    angles = _angles(step, dim // 2)
    wants = [append(step, *k, turned(_parts(x, heads, kv_heads, dim, dim)[1], angles, dim // 2, 1)), append(step, *v, _parts(x, heads, kv_heads, dim, dim)[2])]
    got = _call(step, more, heads, kv_heads, dim, dim, torch.cat([angles, angles[:3]]), dim // 2, 1, *k, *v)
    assert got[4:].isnan().all() and not got[:4].isnan().any()
    for (pool, scale), (codes, scales) in zip((k, v), wants):
        assert torch.equal(scale.cpu(), scales) and torch.equal(pool.cpu().view(torch.uint8), codes)
    assert _lib.load().sllm_status() == 0


def test_missing_pages_and_one_sequence_twice_are_reported():
    """Nothing is written outside the pages there are, and the library's next call says so."""
    from simplellminference_b200 import _lib
    heads, kv_heads, dim = 2, 2, 64
    status = _lib.load().sllm_status
    for bad in (-1, 10 ** 6, "twice", "beyond"):
        step, x, k, v = _case([(30, 5), (70, 2)], heads, kv_heads, dim, dim, 32)
        before = [t.view(torch.uint8).clone() for t in (k[0], v[0])]
        if bad == "twice":
            step.dev["seg_slot"][1] = 0
        elif bad == "beyond":
            step.dev["seg_pos0"][1] = 10 ** 6
        else:
            step.dev["block_table"][1, 2] = bad
        _call(step, x.cuda(), heads, kv_heads, dim, dim, _angles(step, 32), 32, 1, *k, *v)
        assert status() == _lib.EINVAL and status() == 0, bad
        for i, t in enumerate((k[0], v[0])):
            same = (t.view(torch.uint8) == before[i]).flatten(1).all(1)
            written = set() if bad == "twice" else {int(step.table_np[0, 0]), int(step.table_np[0, 1])}
            assert {n for n in range(step.n_pages) if not same[n]} == written, bad


def test_captured_on_another_stream():
    heads, kv_heads, dim = 4, 2, 128
    step, x, k, v = _case([(40, 1), (7, 1)], heads, kv_heads, dim, dim, 64)
    angles = _angles(step, 64)
    wants = [append(step, *k, turned(_parts(x, heads, kv_heads, dim, dim)[1], angles, 64, 1)), append(step, *v, _parts(x, heads, kv_heads, dim, dim)[2])]
    ops, xs, da, out, side = _ops(), x.cuda(), angles.cuda(), torch.zeros(2, heads * dim, device="cuda"), torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        at, row = xs.data_ptr(), xs.stride(0)
        ops.rotary_kv8(step.b, at, row, heads, dim, at + 4 * heads * dim, row, kv_heads, at + 4 * (heads + kv_heads) * dim, row, dim, da, 64, 1, out.data_ptr(), heads * dim,
                       *k, *v, step.n_pages, side.cuda_stream)
    for _ in range(3):                                              # the same rows again: nothing changes after the first time
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out.cpu(), turned(_parts(x, heads, kv_heads, dim, dim)[0], angles, 64, 1).flatten(1))
    for (pool, scale), (codes, scales) in zip((k, v), wants):
        assert torch.equal(scale.cpu(), scales) and torch.equal(pool.cpu().view(torch.uint8), codes)
