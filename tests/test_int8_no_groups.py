"""CPU: rows without a group to belong to are refused; the result would be memory that nothing wrote."""
import ctypes

import pytest


@pytest.mark.parametrize("device_sizes", [None, 256])
def test_rows_without_groups_are_refused(device_sizes):
    from fp8_gmm_b200 import _lib as L

    g = L.Int8GemmArgs(a=256, b=256, c=256, a_scales=256, b_scales=256, num_groups=0, rows=8, n=32, k=64, device_m_sizes=device_sizes)
    assert L.lib.fp8gmm_int8_grouped_gemm(ctypes.byref(g), None) == 1
    assert b"no groups" in L.lib.fp8gmm_last_error(), L.lib.fp8gmm_last_error()
    q = L.QuantizeRowsArgs(in_=256, in_ld=64, top_k=1, in_rows=8, rows=8, cols=64, activation=0, codes=256, scales=256)
    assert L.lib.fp8gmm_int8_linear(ctypes.byref(q), ctypes.byref(g), None) == 1      # before anything is launched
    assert b"no groups" in L.lib.fp8gmm_last_error()
    g.rows = 0
    assert L.lib.fp8gmm_int8_grouped_gemm(ctypes.byref(g), None) == 0
