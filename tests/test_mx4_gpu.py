"""Microscaled 4-bit matrices on the GPU: quantisation, its inverse and the products against plain 64-bit forms."""
import numpy as np
import pytest
import torch

import dense_helpers as dh

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


def ids(cu):
    return {"f32": cu.F32, "f16": cu.F16, "bf16": cu.BF16}


def buffers(cu, rows, k, fill=0xEE):
    nc, ns = cu.mx4_bytes(rows, k)
    return torch.full((max(nc, 1),), fill, dtype=torch.uint8, device="cuda"), torch.full((max(ns, 1),), fill, dtype=torch.uint8, device="cuda")


def quantised(cu, ctx, x, name, ldx=0):
    rows, k = x.shape
    codes, scales = buffers(cu, rows, k)
    assert ctx.mx4_quantize_dev(ids(cu)[name], x.data_ptr(), rows, k, codes.data_ptr(), scales.data_ptr(), ldx)
    torch.cuda.synchronize()
    return codes, scales


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 96), (129, 128), (70, 2080), (300, 4096)])
def test_quantise(cu, ctx, name, rows, k):
    gen = torch.Generator().manual_seed(rows * k)
    x = torch.randn(rows, k, generator=gen) * torch.exp2(torch.randint(-20, 14, (rows, 1), generator=gen).float())
    # halves and quarters of powers of two: ties and borders of the grid
    x[:, ::3] = torch.round(x[:, ::3] * 8) / 8
    x[0, :32] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.5] * 4) * torch.tensor([1, -1] * 16)
    x = x.to(TYPES[name]).cuda()
    codes, scales = quantised(cu, ctx, x, name)
    code, e = dh.unpack(codes, scales, rows, k)
    want, want_e = dh.quantise(x)
    assert torch.equal(e, want_e)
    assert torch.equal(code, want)
    # scales past a row's end are zero, rows past the last as they were
    full, nkb = scales.cpu(), -(-k // 128)
    for j in range(k // 32, nkb * 4):
        assert all(full[dh.place(r, j, k)] == 0 for r in range(rows))
    if rows % 128:
        assert all(full[dh.place(rows, j, k)] == 0xEE for j in range(nkb * 4))


@pytest.mark.parametrize("name", TYPES)
def test_quantise_edges(cu, ctx, name):
    """Zeros, the least and the largest numbers, infinities, NaN and signs; a block of each."""
    t = TYPES[name]
    info = torch.finfo(t)
    x = torch.zeros(10, 64)
    x[1] = info.tiny * info.eps  # the least subnormal number
    x[2] = info.tiny
    x[3] = info.max
    x[4] = -info.max
    x[5, 3] = float("inf")
    x[6, 40] = float("nan")
    x[7, 0], x[7, 1] = 1.0, -0.0
    x[8, ::2] = -info.tiny
    x[9] = torch.linspace(-6.4, 6.4, 64)
    x = x.to(t).cuda()
    codes, scales = quantised(cu, ctx, x, name)
    code, e = dh.unpack(codes, scales, 10, 64)
    want, want_e = dh.quantise(x)
    assert torch.equal(e, want_e)
    assert torch.equal(code, want)
    out = torch.empty(10, 64, device="cuda")
    assert ctx.mx4_dequantize_dev(codes.data_ptr(), scales.data_ptr(), 10, 64, cu.F32, out.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(out.isnan().cpu(), dh.values(code, e).isnan())


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("shift", [0, 1])
def test_rows_apart(cu, ctx, name, shift):
    """Rows with gaps, on and off 16-byte boundaries, in and out; gaps of the output stay as they were."""
    rows, k, ld = 37, 160, 173 + shift * 11
    flat = torch.randn(rows * ld + 8, generator=torch.Generator().manual_seed(5)).to(TYPES[name]).cuda()
    x = flat[shift:shift + rows * ld].reshape(rows, ld)
    codes, scales = buffers(cu, rows, k)
    assert ctx.mx4_quantize_dev(ids(cu)[name], x.data_ptr(), rows, k, codes.data_ptr(), scales.data_ptr(), ld)
    back = torch.full((rows * ld + 8,), 99.0, dtype=TYPES[name], device="cuda")
    o = back[shift:shift + rows * ld].reshape(rows, ld)
    assert ctx.mx4_dequantize_dev(codes.data_ptr(), scales.data_ptr(), rows, k, ids(cu)[name], o.data_ptr(), ld)
    torch.cuda.synchronize()
    code, e = dh.quantise(x[:, :k])
    assert torch.equal(o[:, :k].cpu(), dh.values(code, e).to(TYPES[name]))
    assert bool((o[:, k:] == 99).all())


def test_every_code_and_scale_comes_back(cu, ctx):
    """All 16 codes under all 256 scales: exact in F32 and BF16 (infinite beyond them), rounded in F16."""
    code = torch.arange(16, dtype=torch.uint8).repeat(256, 2)
    e = torch.arange(256, dtype=torch.uint8).reshape(256, 1)
    codes, scales = dh.pack(code, e)
    want = dh.values(code, e)
    for name, t in TYPES.items():
        out = torch.empty(256, 32, dtype=t, device="cuda")
        assert ctx.mx4_dequantize_dev(codes.data_ptr(), scales.data_ptr(), 256, 32, ids(cu)[name], out.data_ptr())
        torch.cuda.synchronize()
        got, w = out.cpu(), want.to(torch.float32).to(t)
        assert torch.equal(got.isnan(), w.isnan())
        assert torch.equal(got[~w.isnan()], w[~w.isnan()])


def test_blocks_of_a_file(cu, ctx):
    """17-byte blocks: the scale, then elements 0 to 15 in the low halves of 16 bytes and 16 to 31 in the high ones."""
    gen = torch.Generator().manual_seed(3)
    rows, k, ld = 131, 224, 256
    blocks = torch.randint(0, 256, (rows, ld // 32, 17), generator=gen, dtype=torch.uint8)
    lo, hi = blocks[:, :k // 32, 1:] & 15, blocks[:, :k // 32, 1:] >> 4
    code, e = torch.cat([lo, hi], -1).reshape(rows, k), blocks[:, :k // 32, 0]
    codes, scales = buffers(cu, rows, k)
    dev = blocks.cuda()
    assert ctx.mx4_quantize_dev(cu.MXFP4, dev.data_ptr(), rows, k, codes.data_ptr(), scales.data_ptr(), ld)
    torch.cuda.synchronize()
    got, got_e = dh.unpack(codes, scales, rows, k)
    assert torch.equal(got, code) and torch.equal(got_e, e)


def check(got, want, off):
    bad = (got.double().cpu() - want).abs() > off
    assert not bad.any(), "%d of %d, first %s: %r for %r (may be %r off)" % (
        bad.sum(), bad.numel(), bad.nonzero()[0].tolist(), got.cpu()[bad][0].item(), want[bad][0].item(), off[bad][0].item())


@pytest.mark.parametrize("nt,k,n,name", [
    (1, 32, 1, "f32"), (1, 4096, 300, "f32"), (2, 64, 128, "bf16"), (16, 96, 129, "f16"), (17, 512, 640, "f32"), (33, 2080, 257, "bf16"),
    (64, 256, 100, "f32"), (65, 1056, 384, "f16"), (128, 4000, 131, "f32"), (129, 288, 1000, "f32"), (257, 1024, 513, "bf16"), (700, 2016, 1111, "f32"),
    (2500, 160, 2053, "bf16"),
])
def test_product(cu, ctx, nt, k, n, name):
    gen = torch.Generator().manual_seed(nt + k + n)
    x, w = dh.random_codes(gen, nt, k), dh.random_codes(gen, n, k)
    (xc, xs), (wc, ws) = dh.pack(*x, dirty=255), dh.pack(*w, dirty=255)
    vx, vw = dh.values(*x), dh.values(*w)
    want, size = vx @ vw.T, vx.abs() @ vw.abs().T
    ld = n + 5
    out = torch.full((nt, ld), 77.0, dtype=TYPES[name], device="cuda")
    assert ctx.mx4_gemm_dev(xc.data_ptr(), xs.data_ptr(), wc.data_ptr(), ws.data_ptr(), nt, k, n, ids(cu)[name], out.data_ptr(), ld)
    torch.cuda.synchronize()
    assert bool((out[:, n:] == 77).all())
    want = want.clamp(-torch.finfo(TYPES[name]).max, torch.finfo(TYPES[name]).max) if name == "f16" else want
    got = out[:, :n].clamp(-65504, 65504) if name == "f16" else out[:, :n]
    check(got, want, dh.sum_error(k, size) + dh.half_step(TYPES[name]) * want.abs() + dh.floor_of(TYPES[name]))


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("nt,k,n", [(3000, 64, 4100), (5000, 256, 2048), (2600, 544, 5003), (90, 96, 70000)])
def test_product_of_many_tiles(cu, ctx, nt, k, n, name):
    """Several tiles for every SM, with next to nothing between them: each tile's results are its own, every time."""
    gen = torch.Generator().manual_seed(nt + k + n)
    x, w = dh.random_codes(gen, nt, k, 120, 125), dh.random_codes(gen, n, k, 120, 125)
    (xc, xs), (wc, ws) = dh.pack(*x), dh.pack(*w)
    vx, vw = dh.values(*x).cuda(), dh.values(*w).cuda()
    want = vx @ vw.T
    off = dh.sum_error(k, vx.abs() @ vw.abs().T) + dh.half_step(TYPES[name]) * want.abs() + dh.floor_of(TYPES[name])
    for _ in range(4):
        out = torch.full((nt, n), 77.0, dtype=TYPES[name], device="cuda")
        assert ctx.mx4_gemm_dev(xc.data_ptr(), xs.data_ptr(), wc.data_ptr(), ws.data_ptr(), nt, k, n, ids(cu)[name], out.data_ptr())
        torch.cuda.synchronize()
        assert int(((out.double() - want).abs() > off).sum()) == 0


@pytest.mark.parametrize("nt,k,n", [(3000, 64, 4128), (2600, 256, 4096)])
def test_gated_of_many_tiles(cu, ctx, nt, k, n):
    gen = torch.Generator().manual_seed(nt + k + n)
    x, g, u = dh.random_codes(gen, nt, k, 124, 128), dh.random_codes(gen, n, k, 119, 123), dh.random_codes(gen, n, k, 119, 123)
    (xc, xs), (gc, gs), (uc, us) = (dh.pack(*m) for m in (x, g, u))
    vx, vg, vu = (dh.values(*m).cuda() for m in (x, g, u))
    wg, wu = vx @ vg.T, vx @ vu.T
    want = dh.act("silu", wg) * wu
    off_g, off_u = dh.sum_error(k, vx.abs() @ vg.abs().T), dh.sum_error(k, vx.abs() @ vu.abs().T)
    off = (dh.SLOPE * off_g + 2.0 ** -20 * wg.abs()) * (wu.abs() + off_u) + dh.act("silu", wg).abs() * off_u
    ptrs = [t.data_ptr() for t in (xc, xs, gc, gs, uc, us)]
    for _ in range(4):
        out = torch.full((nt, n), 77.0, device="cuda")
        assert ctx.mx4_gated_dev(cu.ACT_SILU, *ptrs, nt, k, n, cu.F32, out.data_ptr())
        codes, scales = buffers(cu, nt, n)
        assert ctx.mx4_gated_dev(cu.ACT_SILU, *ptrs, nt, k, n, cu.MXFP4, codes.data_ptr(), scales.data_ptr())
        again, again_s = quantised(cu, ctx, out, "f32")
        torch.cuda.synchronize()
        assert int(((out.double() - want).abs() > off + dh.half_step(torch.float32) * want.abs()).sum()) == 0
        assert torch.equal(codes, again)
        code, e = dh.unpack(codes, scales, nt, n)
        assert torch.equal(e, dh.unpack(again, again_s, nt, n)[1])


def test_product_nan_and_far_scales(cu, ctx):
    """A NaN scale makes its row's results NaN and no other's; scales at both ends of their range meet."""
    gen = torch.Generator().manual_seed(8)
    nt, k, n = 40, 320, 200
    x, w = dh.random_codes(gen, nt, k, 0, 40), dh.random_codes(gen, n, k, 214, 254)
    x[1][7, 3] = 255
    w[1][11, 9] = 255
    (xc, xs), (wc, ws) = dh.pack(*x, dirty=255), dh.pack(*w, dirty=255)
    vx, vw = dh.values(*x), dh.values(*w)
    want, size = vx @ vw.T, vx.abs() @ vw.abs().T
    out = torch.empty(nt, n, device="cuda")
    assert ctx.mx4_gemm_dev(xc.data_ptr(), xs.data_ptr(), wc.data_ptr(), ws.data_ptr(), nt, k, n, cu.F32, out.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(out.isnan().cpu(), want.isnan())
    fine = ~want.isnan()
    check(out.cpu()[fine], want[fine], dh.sum_error(k, size)[fine])


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("nt,k,n,name", [
    (1, 32, 8, "f32"), (1, 2048, 1000, "bf16"), (5, 160, 129, "f32"), (31, 544, 96, "f16"), (64, 1024, 256, "f32"), (100, 96, 320, "f32"),
    (130, 2048, 640, "bf16"), (900, 288, 1030, "f32"),
])
def test_gated(cu, ctx, act, nt, k, n, name):
    gen = torch.Generator().manual_seed(nt + k + n)
    x, g, u = dh.random_codes(gen, nt, k, 124, 128), dh.random_codes(gen, n, k, 119, 123), dh.random_codes(gen, n, k, 119, 123)
    (xc, xs), (gc, gs), (uc, us) = (dh.pack(*m, dirty=255) for m in (x, g, u))
    vx, vg, vu = dh.values(*x), dh.values(*g), dh.values(*u)
    wg, wu = vx @ vg.T, vx @ vu.T
    want = dh.act(act, wg) * wu
    off_g, off_u = dh.sum_error(k, vx.abs() @ vg.abs().T), dh.sum_error(k, vx.abs() @ vu.abs().T)
    # the activation itself: a few steps of 32 bits of its value and of its argument's
    off = (dh.SLOPE * off_g + 2.0 ** -20 * wg.abs()) * (wu.abs() + off_u) + dh.act(act, wg).abs() * off_u
    ld = n + 3
    out = torch.full((nt, ld), 77.0, dtype=TYPES[name], device="cuda")
    ids_act = {"silu": cu.ACT_SILU, "gelu": cu.ACT_GELU}[act]
    assert ctx.mx4_gated_dev(ids_act, xc.data_ptr(), xs.data_ptr(), gc.data_ptr(), gs.data_ptr(), uc.data_ptr(), us.data_ptr(), nt, k, n, ids(cu)[name],
                             out.data_ptr(), None, ld)
    torch.cuda.synchronize()
    assert bool((out[:, n:] == 77).all())
    check(out[:, :n], want, off + dh.half_step(TYPES[name]) * (want.abs() + off) + dh.floor_of(TYPES[name]))


@pytest.mark.parametrize("nt,k,n", [(1, 64, 32), (3, 2048, 160), (20, 96, 224), (70, 512, 1056), (128, 320, 96), (300, 512, 512)])
def test_gated_to_four_bits(cu, ctx, nt, k, n):
    """The result in 4 bits is what quantising the 32-bit result gives: codes, scales, zeros past a row's end."""
    gen = torch.Generator().manual_seed(nt + k + n)
    x, g, u = dh.random_codes(gen, nt, k, 124, 128), dh.random_codes(gen, n, k, 119, 123), dh.random_codes(gen, n, k, 119, 123)
    g[1][n // 2, 0] = 255  # a feature that is NaN
    (xc, xs), (gc, gs), (uc, us) = (dh.pack(*m) for m in (x, g, u))
    ptrs = [t.data_ptr() for t in (xc, xs, gc, gs, uc, us)]
    plain = torch.empty(nt, n, device="cuda")
    assert ctx.mx4_gated_dev(cu.ACT_SILU, *ptrs, nt, k, n, cu.F32, plain.data_ptr())
    codes, scales = buffers(cu, nt, n)
    assert ctx.mx4_gated_dev(cu.ACT_SILU, *ptrs, nt, k, n, cu.MXFP4, codes.data_ptr(), scales.data_ptr())
    torch.cuda.synchronize()
    want, want_e = dh.quantise(plain)
    code, e = dh.unpack(codes, scales, nt, n)
    assert torch.equal(e, want_e) and torch.equal(code, want)
    assert int((e == 255).sum()) == nt
    for j in range(n // 32, -(-n // 128) * 4):
        assert all(scales.cpu()[dh.place(r, j, n)] == 0 for r in range(nt))


def test_a_whole_block_runs_together(cu, ctx):
    """Weights laid out once from rows, activations quantised, gated result in 4 bits, product: twice, and replayed from a graph; the same bits."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    nt, k, n = 45, 512, 704
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x = rnd(nt, k).bfloat16()
    weights = [quantised(cu, ctx, (rnd(n, k) * k ** -0.5), "f32") for _ in range(2)] + [quantised(cu, ctx, rnd(k, n) * n ** -0.5, "f32")]
    (gc, gs), (uc, us), (dc, ds) = weights
    x4, h4 = buffers(cu, nt, k), buffers(cu, nt, n)
    out = torch.empty(nt, k, device="cuda")

    def block():
        assert ctx.mx4_quantize_dev(cu.BF16, x.data_ptr(), nt, k, x4[0].data_ptr(), x4[1].data_ptr())
        assert ctx.mx4_gated_dev(cu.ACT_SILU, x4[0].data_ptr(), x4[1].data_ptr(), gc.data_ptr(), gs.data_ptr(), uc.data_ptr(), us.data_ptr(), nt, k, n, cu.MXFP4,
                                 h4[0].data_ptr(), h4[1].data_ptr())
        assert ctx.mx4_gemm_dev(h4[0].data_ptr(), h4[1].data_ptr(), dc.data_ptr(), ds.data_ptr(), nt, n, k, cu.F32, out.data_ptr())

    block()
    torch.cuda.synchronize()
    first = out.clone()
    vx = dh.values(*dh.quantise(x))
    vg, vu, vd = (dh.values(*dh.unpack(c, s, r, q)) for (c, s), r, q in zip(weights, (n, n, k), (k, k, n)))
    h = dh.act("silu", vx @ vg.T) * (vx @ vu.T)
    want = dh.values(*dh.quantise(h)) @ vd.T
    # an element that lies next to a border of the grid may fall on its other side: few do
    assert float((first.cpu().double() - want).norm() / want.norm()) < 1e-2
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        block()
    out.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    del graph
    ctx.set_stream(1)


def test_no_rows(cu, ctx):
    codes, scales = buffers(cu, 128, 64)
    out = torch.full((64,), 5.0, device="cuda")
    p = codes.data_ptr(), scales.data_ptr()
    before = ctx.launch_count()
    assert ctx.mx4_quantize_dev(cu.F32, None, 0, 64, None, None)
    assert ctx.mx4_dequantize_dev(None, None, 0, 64, cu.F32, None)
    assert ctx.mx4_gemm_dev(None, None, *p, 0, 64, 128, cu.F32, out.data_ptr())
    assert ctx.mx4_gated_dev(cu.ACT_SILU, None, None, *p, *p, 0, 64, 128, cu.F32, out.data_ptr())
    assert ctx.launch_count() == before
    torch.cuda.synchronize()
    assert bool((out == 5).all())


def test_two_contexts_at_once(cu):
    """Two contexts, each on a stream of its own, with products of both sizes in flight together: each gives what it gives alone."""
    gen = torch.Generator().manual_seed(6)
    work = []
    for i, shapes in enumerate((((2000, 512, 2100), (7, 2048, 3000)), ((1500, 768, 1800), (100, 1024, 2000)))):
        c, stream, jobs = cu.CudaCtx(0), torch.cuda.Stream(), []
        c.set_stream(stream.cuda_stream)
        for nt, k, n in shapes:
            x, w = dh.pack(*dh.random_codes(gen, nt, k)), dh.pack(*dh.random_codes(gen, n, k))
            jobs.append((nt, k, n, x, w, torch.empty(nt, n, device="cuda")))
        work.append((c, stream, jobs))

    def enqueue(c, jobs):
        for nt, k, n, x, w, out in jobs:
            assert c.mx4_gemm_dev(x[0].data_ptr(), x[1].data_ptr(), w[0].data_ptr(), w[1].data_ptr(), nt, k, n, cu.F32, out.data_ptr())

    torch.cuda.synchronize()
    alone = []
    for c, _, jobs in work:
        enqueue(c, jobs)
        torch.cuda.synchronize()
        alone.append([j[-1].clone() for j in jobs])
        for j in jobs:
            j[-1].zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for c, _, jobs in work:
            enqueue(c, jobs)
    torch.cuda.synchronize()
    for (c, _, jobs), want in zip(work, alone):
        assert c.device_status() == 0
        assert all(torch.equal(j[-1], v) for j, v in zip(jobs, want))
        c.close()


def test_waits_for_what_is_before_it_on_its_stream(cu, ctx):
    """An operand that a long kernel writes just before, on the same stream that is not torch's own, is the one that is used."""
    gen = torch.Generator().manual_seed(2)
    nt, k, n = 200, 256, 300
    x, w = dh.pack(*dh.random_codes(gen, nt, k)), dh.pack(*dh.random_codes(gen, n, k))
    want, out = torch.empty(nt, n, device="cuda"), torch.empty(nt, n, device="cuda")
    args = lambda o, c, s: (c.data_ptr(), s.data_ptr(), w[0].data_ptr(), w[1].data_ptr(), nt, k, n, cu.F32, o.data_ptr())  # noqa: E731
    assert ctx.mx4_gemm_dev(*args(want, *x))
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    late = torch.zeros_like(x[0]), torch.zeros_like(x[1])
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        ctx.stall(3.0)
        late[0].copy_(x[0])
        late[1].copy_(x[1])
        assert ctx.mx4_gemm_dev(*args(out, *late))
        late[0].zero_()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    ctx.set_stream(1)


def test_first_calls_inside_a_capture():
    """In a process that has not launched any of them: kernels are loaded and devices asked while the stream is being captured."""
    import subprocess
    import sys

    text = """
import sys
sys.path[:0] = %r
import torch
from denno_beta_b200 import cuda as cu
c, stream = cu.CudaCtx(0), torch.cuda.Stream()
c.set_stream(stream.cuda_stream)
x, w = torch.randn(300, 256, device="cuda"), torch.randn(400, 256, device="cuda")
m = lambda rows: [torch.empty(n, dtype=torch.uint8, device="cuda") for n in cu.mx4_bytes(rows, 256)]
xm, wm = m(300), m(400)
many, few = torch.empty(300, 400, device="cuda"), torch.empty(3, 400, device="cuda")
p = lambda v: [t.data_ptr() for t in v]
def calls():
    assert c.mx4_quantize_dev(cu.F32, x.data_ptr(), 300, 256, *p(xm)) and c.mx4_quantize_dev(cu.F32, w.data_ptr(), 400, 256, *p(wm))
    assert c.mx4_gemm_dev(*p(xm), *p(wm), 300, 256, 400, cu.F32, many.data_ptr())
    assert c.mx4_gemm_dev(*p(xm), *p(wm), 3, 256, 400, cu.F32, few.data_ptr())
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=stream):
    calls()
g.replay()
torch.cuda.synchronize()
a, b = many.clone(), few.clone()
many.zero_(), few.zero_()
calls()
torch.cuda.synchronize()
assert torch.equal(a, many) and torch.equal(b, few) and bool(a.any()) and torch.equal(a[:3], b)
print("same")
""" % (sys.path,)
    got = subprocess.run([sys.executable, "-c", text], capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and "same" in got.stdout, got.stderr[-2000:]
