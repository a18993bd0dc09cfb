"""The 8-bit entry points refuse contracted sizes whose sums could pass 32 bits before any
CUDA call."""

import ctypes

import pytest

P16 = ctypes.c_void_p(16)


@pytest.mark.parametrize("K", [131057, 131071, 131072])
def test_linear_int8_refuses_long_rows_before_it_launches(K):
    from mlx_gptq_b200 import _lib as L

    st = L.lib().gq_linear_int8(P16, L.GQ_BF16, 4, K, K, P16, P16, 8, 131072, None, 0, P16, L.GQ_BF16, 8, P16,
                                1 << 40, None, None)
    assert st == L.GQ_ERR_ARG and "131056" in L.last_error() and str(K) in L.last_error()
