"""Bad arguments of the operators that serve several sequences are refused on
the host, before anything touches a device."""
from __future__ import annotations

import ctypes as ct

import numpy as np
import pytest

KEEP = np.zeros(1 << 16, np.uint8)  # addresses that are never followed
AT = (KEEP.ctypes.data + 63) & ~63


def cache(uocr, **change):
    d = dict(qtype=1, kv_heads=2, head_dim=64, page_tokens=16, n_pages=4, n_seqs=2, table_stride=2, reserved0=0, page_stride=0, k=AT, v=AT,
             k_scales=None, v_scales=None, page_table=AT)
    d.update(change)
    return uocr.CKvPages(**d)


def refused(uocr, fn, *args, match):
    lib = uocr.load_library()
    assert getattr(lib, fn)(*args) == uocr.UOCR_ERROR_INVALID_ARGUMENT
    text = lib.uocr_hip_op_error().decode()
    assert match in text, text


BAD_CACHES = [
    (dict(k=None), "no k, v or page_table"), (dict(v=None), "no k, v or page_table"), (dict(page_table=None), "no k, v or page_table"),
    (dict(qtype=4), "not type 4"), (dict(qtype=2), "not type 2"), (dict(head_dim=96), "head_dim is 64 or 128"),
    (dict(head_dim=0), "head_dim is 64 or 128"), (dict(kv_heads=0), "kv_heads 1 to"), (dict(kv_heads=4096), "kv_heads 1 to"),
    (dict(n_seqs=0), "n_seqs 1 to"), (dict(n_seqs=1 << 20), "n_seqs 1 to"), (dict(n_pages=0), "n_pages"), (dict(n_pages=1 << 31), "n_pages"),
    (dict(table_stride=0), "table_stride"), (dict(reserved0=1), "reserved0"), (dict(page_tokens=0), "power of two"),
    (dict(page_tokens=24), "power of two"), (dict(page_tokens=1 << 17), "power of two"),
    (dict(page_tokens=1 << 16, table_stride=1 << 15), "below 2^31"), (dict(page_stride=2 * 16 * 64 - 64), "page_stride"),
    (dict(page_stride=2 * 16 * 64 + 32), "page_stride"), (dict(page_stride=1 << 45), "page_stride"), (dict(n_pages=(1 << 31) - 1, page_stride=1 << 16), "page_stride"), (dict(k=AT + 8), "16-byte"),
    (dict(v=AT + 2), "16-byte"), (dict(page_table=AT + 2), "16-byte"), (dict(qtype=3), "Q8_0 pages"),
    (dict(qtype=3, k_scales=AT), "Q8_0 pages"), (dict(qtype=3, k_scales=AT, v_scales=AT + 2), "Q8_0 pages"),
]


@pytest.mark.parametrize("change,match", BAD_CACHES, ids=lambda v: str(v).replace(" ", "") if isinstance(v, dict) else "")
def test_cache_refusals(uocr, change, match):
    c = ct.byref(cache(uocr, **change))
    refused(uocr, "uocr_op_kv_append", c, 1, None, AT, 2, 1e4, AT, 128, AT, 128, AT, 128, None, 0, AT, 128, match="kv_append: ")
    assert match in uocr.load_library().uocr_hip_op_error().decode()
    refused(uocr, "uocr_op_kv_gather", c, 1, None, AT, AT, 128, AT, 128, match=match)
    refused(uocr, "uocr_op_paged_attention", c, AT, 2, 0.0, AT, 128, AT, AT, 128, match=match)


def test_no_cache(uocr):
    refused(uocr, "uocr_op_kv_gather", None, 1, None, AT, AT, 128, AT, 128, match="no k, v")


APPEND = dict(tokens=2, seqs=None, pos=AT, heads=2, theta=1e4, q=AT, qs=128, q_out=AT, qos=128, k=AT, ks=128, k_out=None, kos=0, v=AT, vs=128)


@pytest.mark.parametrize("change,match", [
    (dict(pos=None), "positions"), (dict(pos=AT + 1), "positions"), (dict(seqs=AT + 2), "positions"), (dict(tokens=3), "a sequence for each"),
    (dict(tokens=1 << 31, seqs=AT), "positions"), (dict(tokens=1 << 23, seqs=AT), "positions"), (dict(heads=0), "q and q_out"), (dict(heads=2000), "q and q_out"), (dict(q_out=None), "q and q_out"),
    (dict(q=None), "q and q_out"), (dict(qs=127), "q and q_out"), (dict(qos=64), "q and q_out"), (dict(q=AT + 1), "q and q_out"),
    (dict(q_out=AT, qos=256), "q and q_out"), (dict(k=None), "k and v rows"), (dict(ks=100), "k and v rows"), (dict(v=None), "k and v rows"),
    (dict(vs=0), "k and v rows"), (dict(k_out=AT, kos=64), "k and v rows"), (dict(k_out=AT, kos=256), "k and v rows"),
    (dict(v=AT + 1), "k and v rows"), (dict(theta=-1.0), "rope_theta"), (dict(theta=float("nan")), "rope_theta"), (dict(theta=float("inf")), "rope_theta"),
    (dict(theta=0.5), "rope_theta"),
], ids=str)
def test_append_refusals(uocr, change, match):
    a = {**APPEND, **change}
    refused(uocr, "uocr_op_kv_append", ct.byref(cache(uocr)), *a.values(), match=match)


@pytest.mark.parametrize("change,match", [
    (dict(pos=None), "positions"), (dict(seqs=AT + 1), "positions"), (dict(tokens=3), "a sequence for each"), (dict(tokens=1 << 23, seqs=AT), "positions"), (dict(k=None, v=None), "k_out or v_out"),
    (dict(ks=127), "k_out or v_out"), (dict(vs=127), "k_out or v_out"), (dict(v=AT + 1), "k_out or v_out"),
], ids=str)
def test_gather_refusals(uocr, change, match):
    a = {**dict(tokens=2, seqs=None, pos=AT, k=AT, ks=128, v=AT, vs=128), **change}
    refused(uocr, "uocr_op_kv_gather", ct.byref(cache(uocr)), *a.values(), match=match)


@pytest.mark.parametrize("change,match", [
    (dict(lengths=None), "lengths"), (dict(lengths=AT + 2), "lengths"), (dict(heads=0), "multiple of kv_heads"), (dict(heads=3), "multiple of kv_heads"),
    (dict(heads=2048), "multiple of kv_heads"), (dict(scale=-1.0), "a scale"), (dict(scale=float("nan")), "a scale"), (dict(scale=float("inf")), "a scale"), (dict(scale=1e20), "a scale"),
    (dict(q=None), "lengths"), (dict(qs=255), "lengths"), (dict(ws=None), "workspace"), (dict(ws=AT + 8), "workspace"), (dict(out=None), "lengths"),
    (dict(os=255), "lengths"), (dict(out=AT + 1), "lengths"), (dict(q=AT, out=AT, os=512), "lengths"),
], ids=str)
def test_paged_refusals(uocr, change, match):
    a = {**dict(lengths=AT, heads=4, scale=0.0, q=AT, qs=256, ws=AT, out=AT, os=256), **change}
    refused(uocr, "uocr_op_paged_attention", ct.byref(cache(uocr)), *a.values(), match=match)


@pytest.mark.parametrize("change,match", [
    (dict(n=0), "n_seqs"), (dict(n=1 << 20), "n_seqs"), (dict(qst=None), "starts"), (dict(qst=AT + 2), "starts"), (dict(kst=AT + 1), "starts"),
    (dict(qt=1 << 31), "tokens"), (dict(kt=1 << 31), "tokens"), (dict(kst=None, kt=9), "as many keys"), (dict(heads=0), "head_dim"), (dict(heads=5), "head_dim"),
    (dict(heads=2048), "head_dim"), (dict(kvh=0), "head_dim"), (dict(dim=80), "head_dim"), (dict(scale=-0.5), "head_dim"), (dict(scale=float("nan")), "head_dim"),
    (dict(q=None), "q and out"), (dict(qs=255), "q and out"), (dict(out=None), "q and out"), (dict(os=0), "q and out"), (dict(q=AT + 1), "q and out"),
    (dict(out=AT, os=512), "q and out"), (dict(qt=1 << 30), "(q_tokens / 64"), (dict(n=1 << 16, heads=512), "(q_tokens / 64"), (dict(k=None), "k and v"), (dict(v=None), "k and v"), (dict(ks=127), "k and v"), (dict(vs=1 << 22), "k and v"),
], ids=str)
def test_packed_refusals(uocr, change, match):
    a = {**dict(n=2, qst=AT, qt=8, kst=AT, kt=8, heads=4, kvh=2, dim=64, scale=0.0, q=AT, qs=256, k=AT, ks=128, v=AT, vs=128, out=AT, os=256), **change}
    refused(uocr, "uocr_op_packed_attention", *a.values(), match=match)


@pytest.mark.parametrize("change,match", [
    (dict(type=3), "not type 3"), (dict(vocab=0), "vocab 1"), (dict(vocab=(1 << 24) + 1, stride=1 << 25), "vocab 1"), (dict(rows=1 << 20), "vocab 1"),
    (dict(logits=None), "vocab 1"), (dict(logits=AT + 1), "vocab 1"), (dict(type=2, logits=AT + 2), "vocab 1"), (dict(stride=99), "vocab 1"),
    (dict(uniform=None), "uniform"), (dict(ws=None), "uniform"), (dict(ws=AT + 4), "uniform"), (dict(tokens=None), "uniform"), (dict(tokens=AT + 2), "uniform"),
    (dict(temperature=AT + 1), "uniform"), (dict(probs=AT + 2), "uniform"),
], ids=str)
def test_sample_refusals(uocr, change, match):
    a = {**dict(type=1, rows=2, vocab=100, logits=AT, stride=100, temperature=None, top_k=None, top_p=None, min_p=None, uniform=AT, ws=AT, tokens=AT,
                probs=None), **change}
    refused(uocr, "uocr_op_sample", *a.values(), match=match)


def test_paged_too_many_rows(uocr):
    c = ct.byref(cache(uocr, n_seqs=1 << 16))
    refused(uocr, "uocr_op_paged_attention", c, AT, 128, 0.0, AT, 1 << 13, AT, AT, 1 << 13, match="n_seqs * heads")


def test_workspace_sizes(uocr):
    assert uocr.paged_attention_workspace_bytes(4, 10, 10, 128) > 0
    for bad in ((0, 4, 2, 64), (1, 0, 1, 64), (1, 5, 2, 64), (1, 4, 0, 64), (1, 4, 2, 80), (1 << 20, 4, 2, 64)):
        assert uocr.paged_attention_workspace_bytes(*bad) == 0
    assert uocr.paged_attention_workspace_bytes(1 << 16, 128, 2, 64) == 0
    assert uocr.sample_workspace_bytes(1, 129280) > 0
    assert uocr.sample_workspace_bytes(1 << 16, 1 << 24) > 0
    for bad in ((1, 0), (1, (1 << 24) + 1), (1, 0xffffffff), ((1 << 16) + 1, 100)):
        assert uocr.sample_workspace_bytes(*bad) == 0
