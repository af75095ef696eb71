"""Bits of the attention over the 8-bit cache (Ops.attention8) where few of them are left: results in bf16, against those in fp32."""
import pytest
import torch
from kv8_testlib import off
from test_kv8_attention_gpu import F32_BOUND, _case, _run, _want

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
