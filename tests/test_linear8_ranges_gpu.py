"""Sums of products of 8-bit codes (Ops.linear8) at the ends of their range: exact, then rounded to fp32 once (scales are 1, nothing is added)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 2, 3, 8, 70, 300])
@pytest.mark.parametrize("a,w,K", [(-128, -128, 131071), (-128, 127, 131072), (-127, -127, 131072), (127, -128, 131071)])
def test_sums_of_the_least_codes(T, a, w, K):
    from simplellminference_b200.config import BF16
    from simplellminference_b200.seqops import Ops
    ops, n = Ops(BF16), 40
    x, y = torch.full((T, 131072), a, dtype=torch.int8, device="cuda"), torch.full((n, 131072), w, dtype=torch.int8, device="cuda")
    one, out = torch.ones(max(T, n), device="cuda"), torch.zeros(T, n, device="cuda")
    ops.linear8(x.data_ptr(), 131072, one, y, 131072, one, None, out.data_ptr(), n, T, n, K, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    ops._ck(ops.lib.sllm_status())
    assert abs(a * w * K) < 2 ** 31 and (out == torch.tensor(float(a * w * K), dtype=torch.float32, device="cuda")).all()
