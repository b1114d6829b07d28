"""What the dense operators refuse, before anything touches a device: the checks look at sizes, types, pointers and row distances only, so that a
context that does not exist (memory of zeros) does for them."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    from denno_beta_b200 import _lib

    return _lib.load()


@pytest.fixture(scope="module")
def ctx():
    return C.cast(C.create_string_buffer(1 << 16), C.c_void_p)


ERR, DECLINED = -1, 1
P, Q, ODD = 0x10000, 0x20000, 0x10008  # addresses that nothing reads
F32, F16, BF16, MX, Q4_K = 0, 1, 30, 39, 12


def test_sizes(lib):
    from denno_beta_b200 import cuda as cu

    assert cu.mx4_bytes(1, 32) == (16, 512)
    assert cu.mx4_bytes(129, 160) == (129 * 80, 2 * 2 * 512)
    assert cu.mx4_bytes(0, 32) == (0, 0)
    assert cu.mx4_bytes(70000, 65536) == (70000 * 32768, 547 * 512 * 512)  # beyond 2^31
    assert cu.mx4_bytes(4, 48) is None
    a = C.c_size_t()
    assert lib.dnb_mx4_bytes(-1, 32, C.byref(a), C.byref(a)) == ERR
    assert lib.dnb_mx4_bytes(1, 0, C.byref(a), C.byref(a)) == ERR
    assert lib.dnb_mx4_bytes(1, 32, None, C.byref(a)) == ERR


@pytest.mark.parametrize("want,change", [
    (ERR, dict(ctx=None)), (ERR, dict(rows=-1)), (ERR, dict(k=0)), (ERR, dict(x=None)), (ERR, dict(codes=None)), (ERR, dict(scales=None)), (ERR, dict(ldx=31)),
    (DECLINED, dict(k=48, ldx=48)), (DECLINED, dict(codes=ODD)), (DECLINED, dict(scales=ODD)), (DECLINED, dict(ty=Q4_K)), (DECLINED, dict(ty=F32, x=P + 2)),
    (DECLINED, dict(ty=F16, x=P + 1)), (DECLINED, dict(ty=MX, ldx=48)),
])
def test_quantise(lib, ctx, want, change):
    a = dict(ctx=ctx, ty=F32, x=P, ldx=64, rows=2, k=32, codes=P, scales=Q)
    a.update(change)
    assert lib.dnb_mx4_quantize_dev(*(a[n] for n in ("ctx", "ty", "x", "ldx", "rows", "k", "codes", "scales"))) == want


@pytest.mark.parametrize("want,change", [
    (ERR, dict(ctx=None)), (ERR, dict(out=None)), (ERR, dict(ldo=63)), (ERR, dict(rows=-5)), (DECLINED, dict(ty=MX)), (DECLINED, dict(ty=F32, out=P + 2)),
    (DECLINED, dict(k=60)), (DECLINED, dict(codes=ODD)),
])
def test_dequantise(lib, ctx, want, change):
    a = dict(ctx=ctx, codes=P, scales=Q, rows=2, k=64, ty=BF16, out=P, ldo=64)
    a.update(change)
    assert lib.dnb_mx4_dequantize_dev(*(a[n] for n in ("ctx", "codes", "scales", "rows", "k", "ty", "out", "ldo"))) == want


@pytest.mark.parametrize("want,change", [
    (ERR, dict(ctx=None)), (ERR, dict(xc=None)), (ERR, dict(ws=None)), (ERR, dict(nt=-1)), (ERR, dict(n=0)), (ERR, dict(n=-3)), (ERR, dict(out=None)),
    (ERR, dict(ldo=9)), (DECLINED, dict(k=80)), (DECLINED, dict(n=(1 << 30) + 1, ldo=1 << 31)), (DECLINED, dict(nt=(1 << 30) + 1)), (DECLINED, dict(xs=ODD)), (DECLINED, dict(wc=ODD)), (DECLINED, dict(ty=MX)), (DECLINED, dict(ty=Q4_K)),
    (DECLINED, dict(ty=F16, out=P + 1)),
])
def test_product(lib, ctx, want, change):
    a = dict(ctx=ctx, xc=P, xs=Q, wc=P, ws=Q, nt=3, k=96, n=10, ty=F32, out=P, ldo=10)
    a.update(change)
    assert lib.dnb_mx4_gemm_dev(*(a[n] for n in ("ctx", "xc", "xs", "wc", "ws", "nt", "k", "n", "ty", "out", "ldo"))) == want


@pytest.mark.parametrize("want,change", [
    (ERR, dict(ctx=None)), (ERR, dict(act=2)), (ERR, dict(act=-1)), (ERR, dict(us=None)), (ERR, dict(ty=MX, out_scales=None)), (ERR, dict(ty=F32, ldo=31)),
    (DECLINED, dict(ty=MX, n=40)), (DECLINED, dict(ty=MX, out=ODD)), (DECLINED, dict(ty=MX, out_scales=ODD)), (DECLINED, dict(k=33)), (DECLINED, dict(uc=ODD)),
])
def test_gated4(lib, ctx, want, change):
    a = dict(ctx=ctx, act=0, xc=P, xs=Q, gc=P, gs=Q, uc=P, us=Q, nt=3, k=96, n=32, ty=MX, out=P, out_scales=Q, ldo=32)
    a.update(change)
    assert lib.dnb_mx4_gated_dev(*(a[n] for n in ("ctx", "act", "xc", "xs", "gc", "gs", "uc", "us", "nt", "k", "n", "ty", "out", "out_scales", "ldo"))) == want


@pytest.mark.parametrize("want,change", [
    (ERR, dict(ctx=None)), (ERR, dict(act=5)), (ERR, dict(nt=-1)), (ERR, dict(n=0)), (ERR, dict(x=None)), (ERR, dict(g=None)), (ERR, dict(out=None)),
    (ERR, dict(ldx=8)), (ERR, dict(ldo=8)), (DECLINED, dict(ty=F32)), (DECLINED, dict(ty=MX)), (DECLINED, dict(k=20, ldx=24)), (DECLINED, dict(n=12)), (DECLINED, dict(n=(1 << 30) + 8, ldo=1 << 31)),
    (DECLINED, dict(x=ODD)), (DECLINED, dict(ldx=20)), (DECLINED, dict(u=ODD)), (DECLINED, dict(pre=ODD)), (DECLINED, dict(out=P + 1)),
])
def test_gated(lib, ctx, want, change):
    a = dict(ctx=ctx, act=0, ty=BF16, x=P, ldx=16, g=P, u=Q, nt=3, k=16, n=24, out=P, ldo=24, pre=Q)
    a.update(change)
    assert lib.dnb_gated_dev(*(a[n] for n in ("ctx", "act", "ty", "x", "ldx", "g", "u", "nt", "k", "n", "out", "ldo", "pre"))) == want


@pytest.mark.parametrize("want,change", [
    (ERR, dict(ctx=None)), (ERR, dict(act=5)), (ERR, dict(pre=None)), (ERR, dict(dout=None)), (ERR, dict(dpre=None)), (ERR, dict(dg=None)), (ERR, dict(du=None)),
    (ERR, dict(x=None)), (ERR, dict(g=None)), (ERR, dict(ldd=8)), (ERR, dict(lddx=8)), (DECLINED, dict(ty=F32)), (DECLINED, dict(ldd=28)), (DECLINED, dict(n=28, ldd=32)),
    (DECLINED, dict(dpre=ODD)), (DECLINED, dict(dout=ODD)), (DECLINED, dict(pre=ODD)), (DECLINED, dict(dx=P + 1)), (DECLINED, dict(dg=P + 1)),
])
def test_gated_backward(lib, ctx, want, change):
    a = dict(ctx=ctx, act=0, ty=F16, x=P, ldx=16, g=P, u=Q, pre=P, dout=Q, ldd=24, nt=3, k=16, n=24, dpre=P, dx=P, lddx=16, dg=P, du=Q)
    a.update(change)
    names = ("ctx", "act", "ty", "x", "ldx", "g", "u", "pre", "dout", "ldd", "nt", "k", "n", "dpre", "dx", "lddx", "dg", "du")
    assert lib.dnb_gated_backward_dev(*(a[n] for n in names)) == want
