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


def test_the_longest_rows(lib):
    """The last multiple of 32 below 2^31: nothing on the way to its sizes passes 32 bits."""
    from denno_beta_b200 import cuda as cu

    k = (1 << 31) - 32
    assert cu.mx4_bytes(1, k) == (k // 2, (1 << 24) * 512)
    assert cu.mx4_bytes(129, k) == (129 * (k // 2), 2 * (1 << 24) * 512)
    assert cu.mx4_bytes((1 << 31) - 1, k) == (((1 << 31) - 1) * (k // 2), (1 << 24) * (1 << 24) * 512)


@pytest.mark.gpu
def test_one_of_the_longest_rows_there_and_back():
    import torch

    import dense_helpers as dh
    from denno_beta_b200 import cuda as cu

    k = (1 << 31) - 32
    c = cu.CudaCtx(0)
    try:
        c.set_stream(1)
        x = torch.zeros(1, k, dtype=torch.bfloat16, device="cuda")
        spots = [0, 128, (1 << 30) - 32, 1 << 30, k - 160, k - 32]
        made = torch.randn(len(spots), 32, generator=torch.Generator().manual_seed(7)).bfloat16()
        for at, v in zip(spots, made):
            x[0, at:at + 32] = v
        codes, scales = (torch.empty(n, dtype=torch.uint8, device="cuda") for n in cu.mx4_bytes(1, k))
        assert c.mx4_quantize_dev(cu.BF16, x.data_ptr(), 1, k, codes.data_ptr(), scales.data_ptr())
        x.fill_(7)
        assert c.mx4_dequantize_dev(codes.data_ptr(), scales.data_ptr(), 1, k, cu.BF16, x.data_ptr())
        torch.cuda.synchronize()
        want = dh.values(*dh.quantise(made))
        for at, w in zip(spots, want):
            assert torch.equal(x[0, at:at + 32].cpu().double(), w)
            x[0, at:at + 32] = 0
        assert not x.any()
        assert c.device_status() == 0
    finally:
        c.close()


@pytest.mark.parametrize("nt,n", [(1 << 22, 1 << 24), (1 << 24, 1 << 20)])
def test_gradients_beyond_a_launch(lib, ctx, nt, n):
    assert lib.dnb_gated_backward_dev(ctx, 0, BF16, None, 8, None, None, P, Q, n, nt, 8, n, P, None, 8, None, None) == DECLINED
