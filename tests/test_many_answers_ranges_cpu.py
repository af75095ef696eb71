"""Sizes at the ends of their range that the operators of many answers to one prompt refuse on the host, before anything is launched (no device)."""
import ctypes as C

import pytest

from simplellminference_b200 import _lib
from test_many_answers_cpu import LINEAR, LOGPROB, QUANTISE, SHARED, _batch, _opts


def _shared(b, **change):
    a = {**SHARED, **change}
    if a["opts"] is not None:
        a["opts"] = C.byref(a["opts"])
    return _lib.load().sllm_seq_attention_shared(C.byref(b), *a.values(), None)


@pytest.mark.parametrize("max_pages,page_len", [(1 << 25, 64), (1 << 16, 1 << 15), ((1 << 31) - 1, 32), (32505857, 64)])
def test_tables_of_more_positions_than_are_counted(max_pages, page_len):
    """Positions, the keys of a share added to them and whole tiles stay within 32 bits."""
    assert _shared(_batch(max_pages=max_pages, page_len=page_len)) == _lib.ENOTSUP
    assert b"positions" in _lib.load().sllm_last_error()


@pytest.mark.parametrize("n", [(1 << 30) + 1, (1 << 31) - 1])
def test_rows_of_more_logits_than_are_counted(n):
    """Indices of logits go on to the end of a CTA's turn, which has to be a number of 32 bits, too."""
    assert _lib.load().sllm_token_logprobs(*{**LOGPROB, "n": n, "ld": n}.values(), None) == _lib.ENOTSUP
    assert b"token_logprobs" in _lib.load().sllm_last_error()


@pytest.mark.parametrize("cap", [float("inf"), float("nan"), -1.0])
def test_caps_that_are_no_numbers(cap):
    """An infinite cap times the tanh of a score divided by it is NaN; a call without a cap is what is meant."""
    assert _shared(_batch(), opts=_opts(softcap=cap)) == _lib.EINVAL
    assert b"bad options" in _lib.load().sllm_last_error()


MOST = (1 << 31) - 1


@pytest.mark.parametrize("size", [(1 << 30) + 1, MOST - 7, MOST])
def test_more_rows_than_are_counted(size):
    """Rows are rounded up to whole tiles, which has to stay within 32 bits."""
    f = _lib.load()
    assert f.sllm_seq_quantise_rows(*{**QUANTISE, "T": size}.values(), None) == _lib.ENOTSUP and b"seq_quantise_rows" in f.sllm_last_error()
    for change in ({"T": size}, {"N": size, "ldc": size}, {"N": size, "ldc": size, "T": 1}):
        assert f.sllm_seq_linear8(*{**LINEAR, **change}.values(), None) == _lib.ENOTSUP and b"seq_linear8" in f.sllm_last_error()
