"""What the operators of many answers to one prompt refuse, on the host, before anything is launched (no device)."""
import ctypes as C

import pytest

from simplellminference_b200 import _lib

BASE = 0x7F0000000000       # never dereferenced: the checks come first
AT = [BASE + (i << 24) for i in range(24)]


def _batch(**change):
    b = _lib.SeqBatch()
    b.T, b.nseg, b.n_qtiles, b.max_pages, b.page_len = 4, 2, 2, 8, 64
    for i, name in enumerate(("tok_slot", "tok_pos", "seg_start", "seg_len", "seg_slot", "seg_pos0", "block_table", "qt_seg", "qt_off", "seg_tile0")):
        setattr(b, name, AT[i])
    for name, v in change.items():
        setattr(b, name, v)
    return b


def _opts(**kw):
    from simplellminference_b200.seqops import Ops
    return Ops.attention_options(**kw)


SHARED = dict(n_groups=2, group_start=AT[10], group_len=AT[11], q=AT[12], ldq=1024, heads=8, kv_heads=2, dk=128, dv=128, scale=0.1, k_pool=AT[13], v_pool=AT[14], kv_dtype=1, n_pages=10, ws=AT[15],
              ws_bytes=1 << 40, opts=None, out=AT[16], ldo=1024, out16=None)


@pytest.mark.parametrize("change,code", [
    (dict(n_groups=0), _lib.EINVAL), (dict(n_groups=3), _lib.EINVAL), (dict(group_start=None), _lib.EINVAL), (dict(group_len=None), _lib.EINVAL), (dict(q=None), _lib.EINVAL),
    (dict(k_pool=None), _lib.EINVAL), (dict(v_pool=None), _lib.EINVAL), (dict(out=None), _lib.EINVAL), (dict(n_pages=0), _lib.EINVAL), (dict(ws=None), _lib.EINVAL),
    (dict(ws=AT[15] + 8), _lib.EINVAL), (dict(ws_bytes=100), _lib.EINVAL), (dict(heads=7), _lib.EINVAL), (dict(kv_heads=0), _lib.EINVAL), (dict(dk=100), _lib.ENOTSUP),
    (dict(dv=264, ldo=4096), _lib.ENOTSUP), (dict(ldq=1023), _lib.EINVAL), (dict(ldo=1000), _lib.EINVAL), (dict(k_pool=AT[13] + 8), _lib.EINVAL), (dict(v_pool=AT[14] + 4), _lib.EINVAL),
    (dict(kv_dtype=2), _lib.ENOTSUP), (dict(kv_dtype=7), _lib.ENOTSUP), (dict(scale=0.0), _lib.EINVAL), (dict(scale=float("nan")), _lib.EINVAL), (dict(scale=float("inf")), _lib.EINVAL),
    (dict(opts=_opts(window=-1)), _lib.EINVAL), (dict(opts=_opts(softcap=-1.0)), _lib.EINVAL), (dict(opts=_opts(window=9, keep_first=-1)), _lib.EINVAL), (dict(opts=_opts(chunk=7)), _lib.ENOTSUP),
    (dict(opts=_opts(values_in_keys=True)), _lib.ENOTSUP), (dict(opts=_opts(cross_values=True)), _lib.ENOTSUP), (dict(b=_batch(T=0)), _lib.EINVAL), (dict(b=_batch(nseg=0)), _lib.EINVAL),
    (dict(b=_batch(n_qtiles=0)), _lib.EINVAL), (dict(b=_batch(tok_pos=None)), _lib.EINVAL), (dict(b=_batch(block_table=None)), _lib.EINVAL), (dict(b=_batch(page_len=48)), _lib.ENOTSUP),
    (dict(b=_batch(page_len=0)), _lib.ENOTSUP), (dict(b=_batch(max_pages=0)), _lib.EINVAL)], ids=str)
def test_shared_attention_refuses(change, code):
    a = {**SHARED, **change}
    b = a.pop("b", None) or _batch()
    if a["opts"] is not None:
        a["opts"] = C.byref(a["opts"])
    assert _lib.load().sllm_seq_attention_shared(C.byref(b), *a.values(), None) == code
    assert b"seq_attention_shared" in _lib.load().sllm_last_error()


def test_workspace_is_host_arithmetic():
    f = _lib.load().sllm_seq_attention_shared_ws_bytes
    assert f(C.byref(_batch()), 2, 8, 2, 128, 128) > 0
    assert f(C.byref(_batch()), 2, 8, 3, 128, 128) == _lib.EINVAL and f(C.byref(_batch()), 0, 8, 2, 128, 128) == _lib.EINVAL and f(C.byref(_batch(T=0)), 2, 8, 2, 128, 128) == _lib.EINVAL


QUANTISE = dict(x=AT[0], x_bf16=0, ldx=1000, codes=AT[1], ldc=1008, scales=AT[2], T=4, K=1000)


@pytest.mark.parametrize("change", [dict(x=None), dict(codes=None), dict(scales=None), dict(T=0), dict(K=0), dict(ldx=999), dict(ldc=999), dict(x=AT[0] + 2), dict(x=AT[0] + 1, x_bf16=1)], ids=str)
def test_quantised_rows_refuse(change):
    assert _lib.load().sllm_seq_quantise_rows(*{**QUANTISE, **change}.values(), None) == _lib.EINVAL
    assert b"seq_quantise_rows" in _lib.load().sllm_last_error()


LINEAR = dict(a=AT[0], lda=1008, a_scale=AT[1], w=AT[2], ldw=1008, w_scale=AT[3], bias=None, C=AT[4], ldc=500, T=4, N=500, K=1000, accumulate=0)


@pytest.mark.parametrize("change,code", [
    (dict(a=None), _lib.EINVAL), (dict(a_scale=None), _lib.EINVAL), (dict(w=None), _lib.EINVAL), (dict(w_scale=None), _lib.EINVAL), (dict(C=None), _lib.EINVAL), (dict(T=0), _lib.EINVAL),
    (dict(N=0), _lib.EINVAL), (dict(K=0), _lib.EINVAL), (dict(lda=992), _lib.EINVAL), (dict(ldw=992), _lib.EINVAL), (dict(ldc=499), _lib.EINVAL), (dict(lda=1009), _lib.EINVAL),
    (dict(ldw=1012), _lib.EINVAL), (dict(a=AT[0] + 8), _lib.EINVAL), (dict(w=AT[2] + 1), _lib.EINVAL), (dict(K=131073, lda=131088, ldw=131088), _lib.ENOTSUP)], ids=str)
def test_integer_products_refuse(change, code):
    assert _lib.load().sllm_seq_linear8(*{**LINEAR, **change}.values(), None) == code
    assert b"seq_linear8" in _lib.load().sllm_last_error()


LOGPROB = dict(logits=AT[0], ld=1000, rows=4, n=1000, token=AT[1], logprob=AT[2], entropy=AT[3], rank=AT[4], top=5, top_idx=AT[5], top_logprob=AT[6])


@pytest.mark.parametrize("change,code", [
    (dict(logits=None), _lib.EINVAL), (dict(rows=0), _lib.EINVAL), (dict(n=0), _lib.EINVAL), (dict(ld=999), _lib.EINVAL), (dict(token=None), _lib.EINVAL), (dict(token=None, logprob=None), _lib.EINVAL),
    (dict(top=-1), _lib.EINVAL), (dict(top=33), _lib.ENOTSUP), (dict(top=6, n=5), _lib.EINVAL), (dict(top_idx=None), _lib.EINVAL), (dict(top=0), _lib.EINVAL), (dict(top=0, top_idx=None), _lib.EINVAL),
    (dict(token=None, logprob=None, rank=None, entropy=None, top=0, top_idx=None, top_logprob=None), _lib.EINVAL)], ids=str)
def test_log_probabilities_refuse(change, code):
    assert _lib.load().sllm_token_logprobs(*{**LOGPROB, **change}.values(), None) == code
    assert b"token_logprobs" in _lib.load().sllm_last_error()
