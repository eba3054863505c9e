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
