"""Refusals of the paged-cache operators: every one is made on the host, before the device is
touched.  CPU only (the pointers are never read)."""
from __future__ import annotations

import math

import pytest

from tqb200 import lib

P = 1 << 20  # a 16-byte aligned address


def cache(**kw):
    a = dict(k=P, v=P, type=lib.EL_F32, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64,
             page_stride=2 * 16 * 64, head_stride=16 * 64, slot_stride=64)
    a.update(kw)
    return lib.PagedCache(*a.values())


def batch(**kw):
    a = dict(q_start=P, kv_len=P, page_table=P, n_seqs=1, table_stride=2, n_tokens=3, max_q_len=3)
    a.update(kw)
    return lib.PagedBatch(*a.values())


def refused(call, text, status=1):
    with pytest.raises(lib.TQB200Error) as e:
        call()
    assert e.value.status == status and text in str(e.value), str(e.value)


def attend(c=None, b=None, **kw):
    a = dict(q_ptr=P, out_ptr=2 * P, el_type=lib.EL_F32, n_heads=8, q_stride=512, out_stride=512, scale=0.125,
             cache=c or cache(), batch=b or batch(), workspace_ptr=3 * P, workspace_bytes=1 << 40, stream=0)
    a.update(kw)
    lib.dev_paged_attention(**a)


def append(c=None, b=None, **kw):
    a = dict(q_ptr=P, k_ptr=2 * P, v_ptr=3 * P, q_out_ptr=4 * P, el_type=lib.EL_F32, n_heads=8, rotary_dim=64,
             q_stride=512, k_stride=128, v_stride=128, q_out_stride=512, q_norm_ptr=None, k_norm_ptr=None,
             eps=1e-6, theta=1e4, positions_ptr=None, cache=c or cache(), batch=b or batch(), stream=0)
    a.update(kw)
    lib.dev_paged_append(**a)


def rotate(**kw):
    a = dict(q_ptr=P, k_ptr=2 * P, q_out_ptr=P, k_out_ptr=2 * P, el_type=lib.EL_F32, n_tokens=3, n_heads=8,
             n_kv_heads=2, head_dim=64, rotary_dim=64, q_stride=512, k_stride=128, q_out_stride=512,
             k_out_stride=128, q_norm_ptr=None, k_norm_ptr=None, eps=1e-6, theta=1e4, positions_ptr=P, stream=0)
    a.update(kw)
    lib.dev_qk_norm_rope(**a)


CACHES = [
    (dict(k=None), "cache k is null"), (dict(v=P + 2), "cache v is not 4-byte aligned"),
    (dict(type=7), "unknown cache type"), (dict(n_pages=0), "0 pages"), (dict(page_size=0), "of 0 slots"),
    (dict(n_kv_heads=0), "0 KV heads"), (dict(head_dim=60), "head_dim 60"), (dict(head_dim=264), "head_dim 264"),
    (dict(slot_stride=63), "inside 64"), (dict(head_stride=16 * 64 - 1), "inside"),
    (dict(page_stride=100), "inside"), (dict(page_stride=-1), "cache stride -1"),
    (dict(page_stride=1 << 45), "cache stride"), (dict(type=lib.EL_BF16), "over a cache of type 2"),
]
BATCHES = [
    (dict(q_start=None), "q_start is null"), (dict(kv_len=None), "kv_len is null"),
    (dict(page_table=P + 1), "page_table is not 4-byte"), (dict(n_seqs=-1), "-1 sequences"),
    (dict(n_tokens=-1), "-1 rows"), (dict(max_q_len=-1), "at most -1"), (dict(table_stride=-1), "-1 pages"),
    (dict(n_seqs=1 << 25), "sequences"),
]


@pytest.mark.parametrize("kw,text", CACHES)
def test_bad_caches_are_refused(kw, text):
    refused(lambda: attend(cache(**kw)), text)
    refused(lambda: append(cache(**kw)), text)


@pytest.mark.parametrize("kw,text", BATCHES)
def test_bad_batches_are_refused(kw, text):
    refused(lambda: attend(None, batch(**kw)), text)
    refused(lambda: append(None, batch(**kw)), text)


@pytest.mark.parametrize("kw,text", [
    (dict(q_ptr=None), "q is null"), (dict(out_ptr=None), "out is null"), (dict(q_ptr=P + 2), "q is not 4-byte"),
    (dict(n_heads=0), "0 query heads"), (dict(n_heads=7), "7 query heads over 2"), (dict(n_heads=5000), "5000"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=math.nan), "scale"),
    (dict(scale=math.inf), "scale"), (dict(out_stride=511), "out row stride"), (dict(q_stride=-8), "q row stride"),
    (dict(out_ptr=P), "out is q"), (dict(workspace_ptr=None), "workspace is null"),
    (dict(workspace_ptr=P + 8), "workspace is not 16-byte"), (dict(workspace_bytes=8), "workspace of 8 bytes"),
    (dict(el_type=lib.EL_F16), "over a cache of type 0"), (dict(el_type=3), "unknown element type"),
    (dict(status_ptr=2), "status not 4-byte"),
])
def test_bad_attention_arguments_are_refused(kw, text):
    refused(lambda: attend(**kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(k_ptr=None), "k is null"), (dict(v_ptr=None), "v is null"), (dict(q_out_ptr=None), "q_out is null"),
    (dict(rotary_dim=66), "rotary_dim 66"), (dict(rotary_dim=3), "rotary_dim 3"), (dict(rotary_dim=-2), "rotary_dim"),
    (dict(theta=0.0), "theta"), (dict(theta=math.inf), "theta"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"),
    (dict(q_out_stride=500), "q_out row stride"), (dict(q_out_ptr=P, q_out_stride=1024), "in place"),
    (dict(q_norm_ptr=P + 1), "q norm"), (dict(k_norm_ptr=P + 2), "k norm"), (dict(positions_ptr=P + 2), "positions"),
    (dict(el_type=lib.EL_BF16), "over a cache"), (dict(n_heads=-1), "-1 query"),
])
def test_bad_append_arguments_are_refused(kw, text):
    refused(lambda: append(**kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(el_type=4), "element type"), (dict(n_tokens=-1), "-1 tokens"), (dict(head_dim=12), "head_dim 12"),
    (dict(head_dim=0), "head_dim 0"), (dict(positions_ptr=None), "positions is null"), (dict(q_ptr=None), "q is null"),
    (dict(k_out_ptr=None), "k_out is null"), (dict(q_out_stride=511), "q_out row stride"),
    (dict(q_out_stride=513), "in place"), (dict(n_heads=9999), "9999"), (dict(theta=-1.0), "theta"),
])
def test_bad_norm_rope_arguments_are_refused(kw, text):
    refused(lambda: rotate(**kw), text)


def test_nothing_to_do_is_no_error():
    rotate(n_tokens=0)
    rotate(n_heads=0, n_kv_heads=0)
    append(None, batch(n_tokens=0))
    append(None, batch(n_seqs=0, q_start=None, kv_len=None, page_table=None))
    attend(None, batch(n_tokens=0))
    attend(None, batch(n_seqs=0, q_start=None, kv_len=None, page_table=None))


def test_without_a_device_the_calls_say_so():
    if lib.device_count() > 0:
        pytest.skip("a GPU is visible")
    for call in (attend, append, rotate):
        refused(call, "no CUDA device", status=4)


def test_workspace_bytes():
    assert lib.paged_attention_workspace_bytes(cache(), batch(), 8) > 0
    assert lib.paged_attention_workspace_bytes(cache(), batch(), 7) == 0  # refused by the call too
    small = lib.paged_attention_workspace_bytes(cache(), batch(), 8)
    assert lib.paged_attention_workspace_bytes(cache(), batch(n_seqs=500, n_tokens=500), 8) >= small


def test_workspace_bytes_depend_on_head_dim_alone():
    want = lib.paged_attention_workspace_bytes(cache(), batch(), 8)
    for c, b, heads in ((cache(), batch(n_seqs=500, n_tokens=500, max_q_len=1), 8), (cache(n_pages=1 << 20), batch(), 32),
                        (cache(type=lib.EL_F16, page_size=1, page_stride=128, head_stride=64, slot_stride=64), batch(), 2)):
        assert lib.paged_attention_workspace_bytes(c, b, heads) == want
