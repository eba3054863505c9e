"""Results that overlap inputs are refused by the C entries before anything launches (CPU)."""

import ctypes

import pytest

from kvboost_b200 import _build, _lib


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_build.LIB_PATH):
        _build.build(verbose=False)
    return _lib.load()


# bf16 rows of 1000 from 1 << 20; (batch, out dtype, stride, out's offset in bytes, its stride)
@pytest.mark.parametrize("batch,out_dtype,stride,off,out_stride", [
    (1, 0, 1000, 2, 1000),              # shifted by one element
    (1, 2, 1000, 1996, 1000),           # float32 from the last element on
    (1, 2, 1000, -3996, 1000),          # float32 that ends in the first
    (3, 0, 2000, 1998, 2000),           # rows side by side but for one element
    (3, 0, 1000, 2000, 1000),           # the second row on
    (2, 0, 1000, -2000, 2000),          # rows that meet further on
    (4, 2, 3000, 2000, 1600),
])
def test_logits_refuse_an_overlapping_result(lib, batch, out_dtype, stride, off, out_stride):
    p = _lib.KvbLogitsParams(0, out_dtype, batch, 1000, 0, 0, 1 << 20, (1 << 20) + off, stride, out_stride)
    assert lib.kvb_process_logits(ctypes.byref(p), None) == _lib.KVB_ERR_INVALID
    assert "overlap" in lib.kvb_last_error().decode()


@pytest.mark.parametrize("batch,batch_stride,head_stride", [
    (2, 0, 128), (2, 1024, 0), (2, 1016, 128), (3, 128, 256), (1, 0, 64), (2, 1024, 120)])
def test_decode_refuses_a_result_whose_heads_overlap(lib, batch, batch_stride, head_stride):
    """8 heads of 128: a broadcast result, rows closer than their heads, heads closer than their width."""
    at = 1 << 20
    p = _lib.KvbPagedDecodeParams(0, 128, batch, 8, 2, 16, 1, 0.1, at, at, at, 1024, 128, batch_stride, head_stride, 8,
                                  at, None, None, 10, 4, 4, at, at, 0, 0, at, None, 0)
    assert lib.kvb_paged_decode_fwd(ctypes.byref(p), None) == _lib.KVB_ERR_INVALID
    assert "overlap" in lib.kvb_last_error().decode()
    assert lib.kvb_paged_decode_workspace_bytes(ctypes.byref(p)) == -1


@pytest.mark.parametrize("batch,heads,batch_stride,head_stride", [
    (2, 8, 1024, 128), (1, 8, 0, 128), (3, 1, 128, 0), (3, 8, 128, 384), (2, 8, 4096, 512), (0, 8, 0, 0)])
def test_decode_takes_results_whose_heads_do_not(lib, batch, heads, batch_stride, head_stride):
    at = 1 << 20
    p = _lib.KvbPagedDecodeParams(0, 128, batch, heads, 1, 16, 1, 0.1, at, at, at, 1024, 128, batch_stride, head_stride, 8,
                                  at, None, None, 10, 4, 4, at, at, 0, 0, at, None, 0)
    assert lib.kvb_paged_decode_workspace_bytes(ctypes.byref(p)) == 0


@pytest.mark.parametrize("field,at", [("k_new", 0), ("v_new", 0), ("k_new", -16), ("v_new", 10 * 2 * 2 * 16 * 128 * 2 - 16)])
def test_append_refuses_sources_inside_the_pool(lib, field, at):
    """A pool of 10 blocks, 2 heads of 128; 3 tokens whose vectors lie in it, or reach into it."""
    pool = 1 << 24
    p = _lib.KvbAppendPagedParams(128, 2, 3, 10, 4096, 4096, 256, 128, 256, 128, pool, 4096, 4096)
    setattr(p, field, pool + at)
    assert lib.kvb_append_paged_kv(ctypes.byref(p), None) == _lib.KVB_ERR_INVALID
    assert "overlap" in lib.kvb_last_error().decode()
