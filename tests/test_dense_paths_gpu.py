"""Paths of the dense products that a device's size leads to: tiles split among the pairs of a cluster (4 bits), and several tiles a block of few rows.
That these sizes take them is asserted without a GPU (test_dense_plan)."""
import pytest
import torch

import dense_helpers as dh
import dense_sizes as sizes

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def cu():
    from denno_beta_b200 import cuda

    return cuda


@pytest.fixture()
def ctx(cu):
    c = cu.CudaCtx(0)
    c.set_stream(1)  # torch's default stream
    yield c
    assert c.device_status() == 0
    c.close()


def check(got, want, off):
    bad = (got.double() - want).abs() > off
    assert not bad.any(), "%d of %d, first %s: %r for %r (may be %r off)" % (
        bad.sum(), bad.numel(), bad.nonzero()[0].tolist(), got[bad][0].item(), want[bad][0].item(), off[bad][0].item())


def operands(gen, *shapes, lo=119, hi=123):
    """Per shape ((codes, scales) on the device, their 64-bit values)."""
    made = []
    for rows, k in shapes:
        m = dh.random_codes(gen, rows, k, lo, hi)
        made.append((dh.pack(*m, dirty=255), dh.values(*m).cuda()))
    return made


def pointers(*matrices):
    return [t.data_ptr() for (m, _) in matrices for t in m]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("nt,k,n", sizes.SPLIT_PRODUCTS + sizes.SEVERAL_A_BLOCK_PRODUCTS)
def test_product(cu, ctx, nt, k, n, name):
    """Rows with and without a gap (stores of their own each), every time the same bits."""
    t = TYPES[name]
    ty = {"f32": cu.F32, "f16": cu.F16, "bf16": cu.BF16}[name]
    x, w = operands(torch.Generator().manual_seed(nt + k + n), (nt, k), (n, k))
    want = x[1] @ w[1].T
    off = dh.sum_error(k, x[1].abs() @ w[1].abs().T)
    off = off + (0 if name == "f32" else dh.half_step(t) * (want.abs() + off) + dh.floor_of(t))
    first = None
    for ld in (n, n + 3, n):
        out = torch.full((nt, ld), 77.0, dtype=t, device="cuda")
        assert ctx.mx4_gemm_dev(*pointers(x, w), nt, k, n, ty, out.data_ptr(), ld)
        torch.cuda.synchronize()
        check(out[:, :n], want, off)
        assert bool((out[:, n:] == 77).all())
        first = out[:, :n].clone() if first is None else first
        assert torch.equal(out[:, :n], first)


def gated_bounds(act, k, x, g, u):
    wg, wu = x @ g.T, x @ u.T
    want = dh.act(act, wg) * wu
    off_g, off_u = dh.sum_error(k, x.abs() @ g.abs().T), dh.sum_error(k, x.abs() @ u.abs().T)
    return want, (dh.SLOPE * off_g + 2.0 ** -20 * wg.abs()) * (wu.abs() + off_u) + dh.act(act, wg).abs() * off_u


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("nt,k,n", sizes.SPLIT_GATED + sizes.SEVERAL_A_BLOCK_GATED)
def test_gated(cu, ctx, nt, k, n, act):
    """In 32 and 16 bits, with and without a gap; in 4 bits what quantising the 32-bit result gives, zeros past a row's end; every time the same bits."""
    ids = {"silu": cu.ACT_SILU, "gelu": cu.ACT_GELU}[act]
    x, g, u = operands(torch.Generator().manual_seed(nt + k + n), (nt, k), (n, k), (n, k), lo=120, hi=122)
    want, off = gated_bounds(act, k, x[1], g[1], u[1])
    ptrs, first = pointers(x, g, u), {}
    for name, ld in (("f32", n), ("f32", n + 5), ("bf16", n), ("bf16", n + 1), ("f32", n), ("bf16", n)):
        t = TYPES[name]
        out = torch.full((nt, ld), 77.0, dtype=t, device="cuda")
        assert ctx.mx4_gated_dev(ids, *ptrs, nt, k, n, {"f32": cu.F32, "bf16": cu.BF16}[name], out.data_ptr(), None, ld)
        torch.cuda.synchronize()
        check(out[:, :n], want, off + dh.half_step(t) * (want.abs() + off) + dh.floor_of(t))
        assert bool((out[:, n:] == 77).all())
        assert torch.equal(out[:, :n], first.setdefault(name, out[:, :n].clone()))
    nc, ns = cu.mx4_bytes(nt, n)
    again = [torch.full((b,), 0xEE, dtype=torch.uint8, device="cuda") for b in (nc, ns)]
    plain = first["f32"].contiguous()
    assert ctx.mx4_quantize_dev(cu.F32, plain.data_ptr(), nt, n, *(m.data_ptr() for m in again))
    for _ in range(3):
        four = [torch.full((b,), 0xEE, dtype=torch.uint8, device="cuda") for b in (nc, ns)]
        assert ctx.mx4_gated_dev(ids, *ptrs, nt, k, n, cu.MXFP4, *(m.data_ptr() for m in four))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(four, again))  # rows past the last: as they were in both


@pytest.mark.parametrize("nt,k,n", sizes.SEVERAL_A_BLOCK_GATED)
def test_gated_of_16_bits(cu, ctx, nt, k, n):
    gen = torch.Generator().manual_seed(nt + k + n)
    x, g, u = ((torch.randn(*s, generator=gen) / s[1] ** 0.25).bfloat16().cuda() for s in ((nt, k), (n, k), (n, k)))
    want, off = gated_bounds("silu", k, x.double(), g.double(), u.double())
    first = None
    for _ in range(3):
        out, pre = torch.full((nt, n), 77.0, dtype=torch.bfloat16, device="cuda"), torch.full((2, nt, n), 77.0, device="cuda")
        assert ctx.gated_dev(cu.ACT_SILU, cu.BF16, x.data_ptr(), g.data_ptr(), u.data_ptr(), nt, k, n, out.data_ptr(), pre.data_ptr())
        torch.cuda.synchronize()
        check(out, want, off + dh.half_step(torch.bfloat16) * (want.abs() + off) + dh.floor_of(torch.bfloat16))
        for got, w in ((pre[0], g), (pre[1], u)):
            check(got, x.double() @ w.double().T, dh.sum_error(k, x.double().abs() @ w.double().abs().T))
        first = first or (out, pre)
        assert torch.equal(out, first[0]) and torch.equal(pre, first[1])
