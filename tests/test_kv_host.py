"""The KV cache operators' host side, without a GPU: the shapes they take, the bytes of a cache, null arguments."""
from __future__ import annotations

import ctypes as C

import pytest


def shape(ocr, **kw):
    return ocr.KvCacheC(**{**dict(type=8, n_slot=3, n_kv=2, d_head=128, n_rows=50, window=0, sinks=0, ring=0), **kw})


@pytest.mark.parametrize("kind,d,quants,scales", [("f16", 128, 256, 0), ("f16", 64, 128, 0), ("q8_0", 128, 128, 8),
                                                  ("q8_0", 64, 64, 4), ("q4_0", 128, 64, 8), ("q4_0", 64, 32, 4)])
def test_cache_bytes(ocr, kind, d, quants, scales):
    c = shape(ocr, type=ocr.KV_TYPES[kind], d_head=d)
    assert ocr.kv_cache_bytes(c) == (3 * 2 * 50 * quants, 3 * 2 * 50 * scales)
    big = shape(ocr, type=ocr.KV_TYPES[kind], d_head=d, n_slot=1000, n_rows=1 << 20)  # (past 32 bits)
    assert ocr.kv_cache_bytes(big) == (1000 * 2 * (1 << 20) * quants, 1000 * 2 * (1 << 20) * scales)


@pytest.mark.parametrize("kw,match", [(dict(type=3), "type 3"), (dict(d_head=96), "64 or 128"), (dict(n_slot=0), "shape"),
                                      (dict(n_kv=0), "shape"), (dict(n_rows=0), "shape"), (dict(window=-1), "below 0"),
                                      (dict(sinks=-1), "below 0"), (dict(ring=1), "ring cache"),
                                      (dict(ring=1, window=48, sinks=3), "ring cache")])
def test_shapes_are_refused(ocr, kw, match):
    with pytest.raises(ocr.OcrError, match=match):
        ocr.kv_cache_bytes(shape(ocr, **kw))


def test_null_arguments(ocr):
    L = ocr.lib()
    c, r = shape(ocr), ocr.Rows()
    assert L.ocr_kv_cache_bytes(None, None, None) == 1
    assert L.ocr_kv_cache_bytes(C.byref(c), None, None) == 1
    assert L.ocr_session_kv_cache(None, 0, C.byref(c)) == 1
    assert L.ocr_op_kv_write(None, C.byref(c), C.byref(r), C.byref(r), 1, None, None) == 1
    assert L.ocr_op_kv_read(None, C.byref(c), C.byref(r), C.byref(r), 1, None, None) == 1
    assert L.ocr_op_attention_window(None, C.byref(c), C.byref(r), 2, 1, None, None, 0.1, C.byref(r)) == 1
    assert L.ocr_op_attention_tree(None, C.byref(c), C.byref(r), 2, 1, None, None, None, 0.1, C.byref(r)) == 1
    assert L.ocr_op_kv_keep(None, C.byref(c), 1, 1, None, None, None) == 1
    assert "null" in L.ocr_last_error().decode()
