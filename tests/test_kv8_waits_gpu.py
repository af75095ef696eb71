"""Waits inside the attention over the 8-bit cache that run out: the report, and that nothing of it stays behind once the workspace is zeros again."""
import pytest
import torch
from kv8_testlib import off
from test_kv8_attention_gpu import F32_BOUND, _case, _ops, _run, _want, _workspace

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("segs", [[(700, 1), (2500, 1)], [(700, 200), (2500, 1), (0, 33)]], ids=["decode", "portions"])
def test_waits_that_run_out_are_reported(segs):
    from simplellminference_b200 import _lib
    lib, ops, heads, kv_heads, dim = _lib.load(), _ops(), 8, 2, 128
    step, q, k, v = _case(segs, heads, kv_heads, dim)
    want, ws = _want(step, q, k, v, heads), _workspace(ops, step, heads, kv_heads, dim, dim)
    assert lib.sllm_status() == 0
    assert lib.sllm_tune(10, 0) == 0                               # no polls: every wait is given up at once
    try:
        _run(step, q, k, v, heads, ws=ws, ops=ops)
    finally:
        assert lib.sllm_tune(10, 1 << 24) == 0
    with pytest.raises(_lib.SllmError) as e:
        _run(step, q, k, v, heads, ws=ws, ops=ops)
    assert e.value.code == _lib.ETIMEOUT
    assert lib.sllm_status() == 0
    ws.zero_()
    for _ in range(3):
        assert off(_run(step, q, k, v, heads, ws=ws, ops=ops), want) < F32_BOUND
