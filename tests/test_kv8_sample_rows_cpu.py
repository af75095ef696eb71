"""What the operators of the 8-bit cache and the draw of rows refuse, on the host, before anything is launched (no device)."""
import ctypes as C

import pytest

from simplellminference_b200 import _lib

BASE = 0x7F0000000000       # never dereferenced: the checks come first
AT = [BASE + (i << 24) for i in range(20)]


def _batch(**change):
    b = _lib.SeqBatch()
    b.T, b.nseg, b.n_qtiles, b.max_pages, b.page_len = 4, 2, 2, 8, 64
    for i, name in enumerate(("tok_slot", "tok_pos", "seg_start", "seg_len", "seg_slot", "seg_pos0", "block_table", "qt_seg", "qt_off", "seg_tile0")):
        setattr(b, name, AT[i])
    for name, v in change.items():
        setattr(b, name, v)
    return b


APPEND = dict(q=AT[10], ldq=1024, heads=8, dk=128, k=AT[11], ldk=256, kv_heads=2, v=AT[12], ldv=256, dv=128, angles=AT[13], n_freq=64, layout=1, q_out=AT[14], ldqo=1024, k_pool=AT[15],
              k_scale=AT[16], v_pool=AT[17], v_scale=AT[18], n_pages=10)


@pytest.mark.parametrize("change,code", [
    (dict(q=None), _lib.EINVAL), (dict(k=None), _lib.EINVAL), (dict(v=None), _lib.EINVAL), (dict(q_out=None), _lib.EINVAL), (dict(k_pool=None), _lib.EINVAL),
    (dict(k_scale=None), _lib.EINVAL), (dict(v_pool=None), _lib.EINVAL), (dict(v_scale=None), _lib.EINVAL), (dict(angles=None), _lib.EINVAL), (dict(n_pages=0), _lib.EINVAL),
    (dict(heads=0), _lib.EINVAL), (dict(kv_heads=-1), _lib.EINVAL), (dict(dk=120), _lib.ENOTSUP), (dict(dv=272, ldv=1024), _lib.ENOTSUP), (dict(n_freq=65), _lib.EINVAL),
    (dict(n_freq=-1), _lib.EINVAL), (dict(layout=2), _lib.EINVAL), (dict(ldq=1000), _lib.EINVAL), (dict(ldqo=1023), _lib.EINVAL), (dict(ldk=255), _lib.EINVAL), (dict(ldv=0), _lib.EINVAL),
    (dict(k_pool=AT[15] + 8), _lib.EINVAL), (dict(v_pool=AT[17] + 4), _lib.EINVAL), (dict(q_out=AT[10], ldqo=1028), _lib.EINVAL),
    (dict(b=_batch(T=0)), _lib.EINVAL), (dict(b=_batch(nseg=0)), _lib.EINVAL), (dict(b=_batch(block_table=None)), _lib.EINVAL), (dict(b=_batch(tok_slot=None)), _lib.EINVAL),
    (dict(b=_batch(page_len=48)), _lib.ENOTSUP), (dict(b=_batch(page_len=0)), _lib.ENOTSUP), (dict(b=_batch(max_pages=0)), _lib.EINVAL),
    (dict(b=_batch(T=2 ** 30, nseg=2 ** 30), kv_heads=4, ldk=512, ldv=512), _lib.ENOTSUP)], ids=str)
def test_append_refuses(change, code):
    a = {**APPEND, **change}
    b = a.pop("b", None) or _batch()
    assert _lib.load().sllm_seq_rotary_kv8(C.byref(b), *a.values(), None) == code
    assert b"seq_rotary_kv8" in _lib.load().sllm_last_error()


ATTEND = dict(q=AT[10], ldq=1024, heads=8, kv_heads=2, dk=128, dv=128, scale=0.1, k_pool=AT[11], k_scale=AT[12], v_pool=AT[13], v_scale=AT[14], n_pages=10, ws=AT[15], ws_bytes=1 << 40,
              opts=None, out=AT[16], ldo=1024, out16=None)


def _opts(**kw):
    from simplellminference_b200.seqops import Ops
    return Ops.attention_options(**kw)


@pytest.mark.parametrize("change,code", [
    (dict(q=None), _lib.EINVAL), (dict(k_pool=None), _lib.EINVAL), (dict(k_scale=None), _lib.EINVAL), (dict(v_pool=None), _lib.EINVAL), (dict(v_scale=None), _lib.EINVAL),
    (dict(out=None), _lib.EINVAL), (dict(n_pages=0), _lib.EINVAL), (dict(ws=None), _lib.EINVAL), (dict(ws=AT[15] + 8), _lib.EINVAL), (dict(ws_bytes=100), _lib.EINVAL),
    (dict(heads=7), _lib.EINVAL), (dict(kv_heads=0), _lib.EINVAL), (dict(dk=100), _lib.ENOTSUP), (dict(dv=264), _lib.ENOTSUP), (dict(ldq=1023), _lib.EINVAL), (dict(ldo=1000), _lib.EINVAL),
    (dict(k_pool=AT[11] + 8), _lib.EINVAL), (dict(v_pool=AT[13] + 1), _lib.EINVAL), (dict(opts=_opts(window=-1)), _lib.EINVAL), (dict(opts=_opts(softcap=-1.0)), _lib.EINVAL),
    (dict(scale=0.0), _lib.EINVAL), (dict(scale=-0.1), _lib.EINVAL), (dict(scale=float("inf")), _lib.EINVAL), (dict(scale=float("nan")), _lib.EINVAL),
    (dict(opts=_opts(window=5, chunk=7)), _lib.EINVAL), (dict(opts=_opts(values_in_keys=True)), _lib.ENOTSUP), (dict(opts=_opts(cross_values=True)), _lib.ENOTSUP),
    (dict(b=_batch(n_qtiles=0)), _lib.EINVAL), (dict(b=_batch(qt_off=None)), _lib.EINVAL), (dict(b=_batch(page_len=40)), _lib.ENOTSUP), (dict(b=_batch(seg_pos0=None)), _lib.EINVAL)], ids=str)
def test_attention_refuses(change, code):
    a = {**ATTEND, **change}
    b = a.pop("b", None) or _batch()
    if a["opts"] is not None:
        a["opts"] = C.byref(a["opts"])
    assert _lib.load().sllm_seq_attention8(C.byref(b), *a.values(), None) == code
    assert b"seq_attention8" in _lib.load().sllm_last_error()


def test_workspace_is_host_arithmetic():
    f = _lib.load().sllm_seq_attention8_ws_bytes
    assert f(C.byref(_batch()), 8, 2, 128, 128) > 0
    assert f(C.byref(_batch()), 8, 3, 128, 128) == _lib.EINVAL and f(C.byref(_batch(T=0)), 8, 2, 128, 128) == _lib.EINVAL


SAMPLE = dict(logits=AT[0], ld=1000, rows=4, n=1000, temperature=None, top_k=None, top_p=None, min_p=None, u=AT[1], idx=AT[2], prob=None)


@pytest.mark.parametrize("change,code", [(dict(logits=None), _lib.EINVAL), (dict(u=None), _lib.EINVAL), (dict(idx=None), _lib.EINVAL), (dict(rows=0), _lib.EINVAL), (dict(n=0), _lib.EINVAL),
                                         (dict(ld=999), _lib.EINVAL), (dict(n=720897, ld=720897), _lib.ENOTSUP)], ids=str)
def test_draws_refuse(change, code):
    assert _lib.load().sllm_sample_rows(*{**SAMPLE, **change}.values(), None) == code
    assert b"sample_rows" in _lib.load().sllm_last_error()
