"""Scales whose product with log2(e), which the kernels use, passes float32's range would make NaN of every score: refused."""
import ctypes as C

import pytest

from spmm_amd import attention as A


@pytest.mark.parametrize("scale,ok", [(2.35e38, True), (-2.35e38, True), (2.4e38, False), (-2.4e38, False), (3.4e38, False)], ids=str)
def test_range(scale, ok):
    d = A._Desc(0, A.BF16, 4, 2, 64, 8, 2, scale, 2, 16, 16, 0, 0)
    n = C.c_size_t()
    assert A.lib.spmm_attn_window_work(d, 0, n) == A.lib.spmm_attn_paged_work(d, 64, n) == (0 if ok else -1)
    assert ok or b"scale" in A.lib.spmm_attn_last_error_detail()
