"""Rows of 8-bit codes (Ops.quantise_rows), exactly, and products of them (Ops.linear8): sums are exact, so that a result is off by the roundings of the sum, of two products, and of what is
added to it, 2^-24 each."""
import math

import pytest
import torch
from answers_testlib import codes_of

pytestmark = pytest.mark.gpu
UNIT = 2.0 ** -24


def _ops():
    from simplellminference_b200.config import BF16
    from simplellminference_b200.seqops import Ops
    return Ops(BF16)


def _st():
    return torch.cuda.current_stream().cuda_stream


def _wide(k):
    return -(-k // 16) * 16


def _quantise(x, ldx=None, ldc=None, offset=0, fill=99):
    rows, k = x.shape
    ldx, ldc = ldx or k, ldc or _wide(k)
    flat = torch.full((offset + rows * ldx + 8,), math.nan, dtype=x.dtype)
    flat[offset:offset + rows * ldx].view(rows, ldx)[:, :k] = x
    flat = flat.cuda()
    codes = torch.full((rows, ldc), fill, dtype=torch.int8, device="cuda")
    scale = torch.full((rows + 1,), -1.0, device="cuda")
    _ops().quantise_rows(flat.data_ptr() + offset * x.element_size(), x.dtype == torch.bfloat16, ldx, codes.data_ptr(), ldc, scale, rows, k, _st())
    torch.cuda.synchronize()
    assert (codes[:, k:] == fill).all() and float(scale[rows]) == -1.0
    return codes[:, :k].cpu(), scale[:rows].cpu()


def _check_codes(x, **kw):
    codes, scale = _quantise(x, **kw)
    want, ws = codes_of(x)
    assert torch.equal(scale, ws) and torch.equal(codes, want), (codes != want).nonzero()[:5]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 5), (7, 16), (5, 31), (9, 64), (130, 100), (1, 4096), (33, 4096), (3, 4099), (6, 2056), (2, 16384), (3, 16400), (2, 40001), (500, 512)])
def test_codes(rows, k, dtype):
    g = torch.Generator().manual_seed(rows + k)
    _check_codes((torch.randn(rows, k, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))).to(dtype))


@pytest.mark.parametrize("ldx,ldc,offset", [(4100, 4096, 0), (4097, 4096, 0), (4096, 4112, 3), (4104, 5008, 8)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_codes_of_rows_apart(ldx, ldc, offset, dtype):
    _check_codes(torch.randn(11, 4096, generator=torch.Generator().manual_seed(1)).to(dtype), ldx=ldx, ldc=ldc, offset=offset)


def test_codes_next_to_borders():
    """Quotients at and next to half-way points, where the even code is taken: multiples of half a scale and the numbers beside them."""
    rows = []
    for scale in (1.0, 0.37, 2.0 ** -40, 3e30, 1.1e-38):
        s = torch.tensor(scale) / 127 * 127
        x = (torch.arange(-254, 255).float() / 2) * (s / 127)
        rows.append(torch.cat([x, torch.nextafter(x, torch.tensor(math.inf)), torch.nextafter(x, torch.tensor(-math.inf)), s[None]]))
    _check_codes(torch.stack(rows))


def test_codes_of_zeros_and_the_least_numbers():
    x = torch.zeros(4, 300)
    x[1, 5] = 1e-45
    x[2] = 2.0 ** -126
    x[3, 7] = torch.finfo(torch.float32).max
    _check_codes(x)


def test_rows_that_are_not_finite():
    x = torch.randn(6, 500, generator=torch.Generator().manual_seed(2))
    x[1, 3], x[3, 499], x[4, 0] = math.inf, math.nan, -math.inf
    codes, scale = _quantise(x)
    want, ws = codes_of(x[[0, 2, 5]])
    assert scale[[1, 3, 4]].isnan().all() and (codes[[1, 3, 4]] == 0).all()
    assert torch.equal(scale[[0, 2, 5]], ws) and torch.equal(codes[[0, 2, 5]], want)


def _product(T, n, k, seed=0, bias=False, accumulate=False, lda=None, ldw=None, ldc=None, extreme=False):
    g = torch.Generator().manual_seed(seed)
    lda, ldw, ldc = lda or _wide(k), ldw or _wide(k), ldc or n
    a = torch.randint(-127, 128, (T, lda), generator=g, dtype=torch.int8)          # what lies behind column k is anything
    w = torch.randint(-127, 128, (n, ldw), generator=g, dtype=torch.int8)
    if extreme:
        a[:], w[:] = 127, -127
    sa, sw = torch.rand(T, generator=g) + 0.1, torch.rand(n, generator=g) + 0.1
    bi = torch.randn(n, generator=g) * 100 if bias else None
    c = torch.randn(T + 1, ldc, generator=g)
    cd, ad, wd, sad, swd = c.cuda(), a.cuda(), w.cuda(), sa.cuda(), sw.cuda()
    bd = None if bi is None else bi.cuda()
    ops = _ops()
    ops.linear8(ad.data_ptr(), lda, sad, wd, ldw, swd, bd, cd.data_ptr(), ldc, T, n, k, _st(), accumulate=accumulate)
    torch.cuda.synchronize()
    ops._ck(ops.lib.sllm_status())
    got = cd.cpu()
    assert torch.equal(got[T], c[T]) and torch.equal(got[:, n:], c[:, n:])
    sums = ad[:, :k].double() @ wd[:, :k].double().T
    v = (sums * sad.double()[:, None] * swd.double()).cpu()
    size = v.abs()
    if bias:
        v, size = v + bi.double(), size + bi.double().abs()
    if accumulate:
        v, size = v + c[:T, :n].double(), size + c[:T, :n].double().abs()
    assert ((got[:T, :n].double() - v).abs() <= 5 * UNIT * size).all(), (got[:T, :n].double() - v).abs().max()
    return got


@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 33, 64, 100, 128, 129, 250, 300])
@pytest.mark.parametrize("n,k", [(1, 1), (64, 64), (130, 77), (500, 1000), (1024, 4096), (257, 2056)])
def test_products(T, n, k):
    _product(T, n, k, seed=T + n, bias=T % 2 == 0, accumulate=T % 3 == 0)


@pytest.mark.parametrize("T,n,k", [(1, 4096, 14336), (64, 14336, 4096), (64, 4096, 14336), (700, 4096, 4096), (2000, 1000, 512), (513, 6176, 2048), (40, 32, 131072), (1, 5, 131072)])
def test_larger_products(T, n, k):
    _product(T, n, k, seed=k, bias=True)


@pytest.mark.parametrize("T", [1, 8, 70])
def test_sums_at_the_end_of_the_range(T):
    _product(T, 40, 131072, extreme=True)


@pytest.mark.parametrize("T", [1, 3, 20, 150])
def test_rows_apart(T):
    _product(T, 300, 1000, lda=1024, ldw=1040, ldc=303, bias=True, accumulate=True)


def test_a_product_does_not_depend_on_the_other_tokens():
    """The same row alone and among many: sums are exact, so the results are equal in every bit."""
    g = torch.Generator().manual_seed(3)
    a = torch.randint(-127, 128, (300, 4096), generator=g, dtype=torch.int8).cuda()
    w = torch.randint(-127, 128, (777, 4096), generator=g, dtype=torch.int8).cuda()
    sa, sw = torch.rand(300, generator=g).cuda(), torch.rand(777, generator=g).cuda()
    bias = torch.randn(777, generator=g).cuda()
    ops, outs = _ops(), {}
    for first, T in ((0, 300), (200, 1), (199, 3), (170, 40), (100, 128)):
        c = torch.zeros(T, 777, device="cuda")
        ops.linear8(a[first:].data_ptr(), 4096, sa[first:], w, 4096, sw, bias, c.data_ptr(), 777, T, 777, 4096, _st())
        torch.cuda.synchronize()
        outs[first, T] = c[200 - first].cpu()
    assert all(torch.equal(v, outs[0, 300]) for v in outs.values())


def test_weights_quantised_and_multiplied():
    """As a program uses them: a matrix's rows quantised once, then tokens every step; against the product of the numbers themselves. A code is off by half a step of its row's scale, so that
    a sum of K products is off by less than K * (|x| step_w + |w| step_x) / 2 + K step_x step_w / 4."""
    g = torch.Generator().manual_seed(4)
    T, n, k = 21, 600, 1024
    x, w = torch.randn(T, k, generator=g), torch.randn(n, k, generator=g) / 32
    cx, sx = _quantise(x)
    cw, sw = _quantise(w.bfloat16())
    c = torch.empty(T, n, device="cuda")
    held = [t.cuda() for t in (cx, sx, cw, sw)]
    _ops().linear8(held[0].data_ptr(), k, held[1], held[2], k, held[3], None, c.data_ptr(), n, T, n, k, _st())
    torch.cuda.synchronize()
    bound = 0.5 * (x.abs().double() @ torch.ones(k, n).double() * sw.double() + sx.double()[:, None] * w.bfloat16().double().abs().sum(-1)) + 0.25 * k * sx.double()[:, None] * sw.double()
    assert ((c.cpu().double() - x.double() @ w.bfloat16().double().T).abs() <= bound * (1 + 1e-5)).all()


def test_captured_and_replayed():
    g = torch.Generator().manual_seed(5)
    x = torch.randn(9, 512, generator=g).cuda()
    w = torch.randint(-127, 128, (300, 512), generator=g, dtype=torch.int8).cuda()
    sw = torch.rand(300, generator=g).cuda()
    codes, s, c = torch.zeros(9, 512, dtype=torch.int8, device="cuda"), torch.zeros(9, device="cuda"), torch.zeros(9, 300, device="cuda")
    ops = _ops()

    def step():
        ops.quantise_rows(x.data_ptr(), False, 512, codes.data_ptr(), 512, s, 9, 512, _st())
        ops.linear8(codes.data_ptr(), 512, s, w, 512, sw, None, c.data_ptr(), 300, 9, 300, 512, _st())

    step()
    torch.cuda.synchronize()
    first = c.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    x.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(c, -first)


@pytest.mark.parametrize("T,n,k", [(200, 700, 1000), (20, 256, 4096)], ids=["tiles", "shared tiles"])
def test_waits_that_run_out_are_reported(T, n, k):
    """With no polls allowed the tensor-core kernel gives up its first waits; the library's next call says so, once, and later products are whole again."""
    from simplellminference_b200 import _lib
    lib = _lib.load()
    assert lib.sllm_status() == 0
    assert lib.sllm_tune(10, 0) == 0
    try:
        with pytest.raises(_lib.SllmError) as e:
            _product(T, n, k)
    finally:
        assert lib.sllm_tune(10, 1 << 24) == 0
    assert e.value.code == _lib.ETIMEOUT and lib.sllm_status() == 0
    _product(T, n, k)
