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


def test_sums_beyond_a_launch(lib, ctx):
    """A tile's sum has to end before the wait for it does: 2^19 chunks of 256 elements in 4 bits, of 64 in 16."""
    k, long = 1 << 27, (1 << 27) + 32
    assert lib.dnb_mx4_gemm_dev(ctx, P, Q, P, Q, 0, k, 10, F32, P, 10) == 0  # no rows: a length that is taken
    assert lib.dnb_mx4_gemm_dev(ctx, P, Q, P, Q, 0, long, 10, F32, P, 10) == DECLINED
    assert lib.dnb_mx4_gemm_dev(ctx, P, Q, P, Q, 3, long, 10, F32, P, 10) == DECLINED
    assert lib.dnb_mx4_gated_dev(ctx, 0, P, Q, P, Q, P, Q, 3, long, 32, MX, P, Q, 0) == DECLINED
    k, long = 1 << 25, (1 << 25) + 8
    assert lib.dnb_gated_dev(ctx, 0, BF16, P, k, P, Q, 0, k, 16, P, 16, None) == 0
    assert lib.dnb_gated_dev(ctx, 0, BF16, P, long, P, Q, 1, long, 16, P, 16, None) == DECLINED
    back = lambda nt, n, dx, dw: lib.dnb_gated_backward_dev(ctx, 0, F16, P, 8, P, Q, P, Q, n, nt, 8, n, P, P if dx else None, 8, P if dw else None, Q if dw else None)  # noqa: E731
    assert back(1, (1 << 24) + 8, True, False) == DECLINED  # dx sums over the features of both
    assert back((1 << 25) + 1, 8, False, True) == DECLINED  # the weights' gradients over tokens
    assert back((1 << 25) + 1, 8, True, True) == DECLINED


@pytest.mark.gpu
def test_the_longest_sums():
    """A few terms that are not zero, all over sums of the greatest length: exact, and no wait has given up."""
    import torch

    from denno_beta_b200 import cuda as cu

    c = cu.CudaCtx(0)
    try:
        c.set_stream(1)
        nt, k, n = 1 << 25, 8, 8
        spots = torch.tensor([0, 63, 64, (1 << 23) - 1, 1 << 23, (1 << 24) + 5, 3 << 23, nt - 1])
        x, dout, dpre = (torch.zeros(*s, dtype=torch.bfloat16, device="cuda") for s in ((nt, k), (nt, n), (2, nt, n)))
        pre = torch.ones(2, nt, n, device="cuda")
        pre[0] = 64  # silu(64) = 64 and its slope 1, to the last bit
        vx, vd = (torch.randint(-8, 9, (len(spots), w), generator=torch.Generator().manual_seed(w)).double() for w in (k, n))
        x[spots.cuda()], dout[spots.cuda()] = vx.bfloat16().cuda(), vd.bfloat16().cuda()
        dg, du = torch.empty(n, k, dtype=torch.bfloat16, device="cuda"), torch.empty(n, k, dtype=torch.bfloat16, device="cuda")
        assert c.gated_backward_dev(cu.ACT_SILU, cu.BF16, x.data_ptr(), None, None, pre.data_ptr(), dout.data_ptr(), nt, k, n, dpre.data_ptr(), None, dg.data_ptr(), du.data_ptr())
        torch.cuda.synchronize()
        want = vd.T @ vx
        assert torch.equal(dg.cpu(), want.bfloat16()) and torch.equal(du.cpu(), (64 * want).bfloat16())
        assert c.device_status() == 0
        del x, dout, dpre, pre
        k = 1 << 27
        for nt in (2, 129):
            n, blocks = 3, torch.tensor([0, 1, (k >> 7) - 1, k >> 7, k >> 6, (k >> 5) - 1])
            made = []
            for rows in (nt, n):
                codes, scales = (torch.zeros(b, dtype=torch.uint8, device="cuda") for b in cu.mx4_bytes(rows, k))
                for r in range(rows):
                    for i, b in enumerate(blocks.tolist()):
                        codes[(r * k + 32 * b) // 2] = 1 + (r + i) % 7  # one element of the block
                        scales[((r // 128) * (k // 128) + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4] = 127
                made += [codes, scales]
            out = torch.empty(nt, n, device="cuda")
            assert c.mx4_gemm_dev(*(m.data_ptr() for m in made), nt, k, n, cu.F32, out.data_ptr())
            torch.cuda.synchronize()
            grid = torch.tensor([0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
            value = lambda rows: grid[(torch.arange(rows).reshape(-1, 1) + torch.arange(len(blocks))) % 7]  # noqa: E731
            assert torch.equal(out.cpu(), value(nt) @ value(n).T)
            assert c.device_status() == 0
            del made, codes, scales
    finally:
        c.close()


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
