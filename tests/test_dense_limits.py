"""Sizes that one launch of the dense operators does not take are declined before anything touches a device (cf. test_dense_refusals)."""
import ctypes as C

import pytest

ERR, DECLINED = -1, 1
P, Q = 0x10000, 0x20000  # addresses that nothing reads
F32, F16, BF16, MX = 0, 1, 30, 39


@pytest.fixture(scope="module")
def lib():
    from denno_beta_b200 import _lib

    return _lib.load()


@pytest.fixture(scope="module")
def ctx():
    return C.cast(C.create_string_buffer(1 << 16), C.c_void_p)


@pytest.mark.parametrize("rows,k", [((1 << 31) - 1, 1 << 20), (1 << 30, 1024 + 32), ((1 << 31) - 1, 640)])
def test_rows_beyond_a_launch(lib, ctx, rows, k):
    """A quarter of the rows, times their parts of 128, from 2^31 on."""
    for ty in (F32, F16, BF16, MX):
        assert lib.dnb_mx4_quantize_dev(ctx, ty, P, k, rows, k, P, Q) == DECLINED
    for ty in (F32, F16, BF16):
        assert lib.dnb_mx4_dequantize_dev(ctx, P, Q, rows, k, ty, P, k) == DECLINED


@pytest.mark.parametrize("nt,n", [(1 << 22, 1 << 24), (1 << 24, 1 << 20)])
def test_gradients_beyond_a_launch(lib, ctx, nt, n):
    assert lib.dnb_gated_backward_dev(ctx, 0, BF16, None, 8, None, None, P, Q, n, nt, 8, n, P, None, 8, None, None) == DECLINED
