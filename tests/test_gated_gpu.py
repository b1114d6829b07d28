"""The gated feed-forward block on 16-bit operands, forward and backward, against plain 64-bit forms and against differences."""
import pytest
import torch

import dense_helpers as dh

pytestmark = pytest.mark.gpu
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
SHAPES = [(1, 8, 8), (1, 2048, 1000), (2, 64, 128), (15, 136, 264), (17, 520, 96), (33, 1024, 136), (64, 72, 640), (77, 2056, 1128), (128, 256, 384),
          (129, 512, 200), (300, 264, 1032), (1000, 640, 520)]


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


class Block:
    """Operands, results and 64-bit references of one shape."""

    def __init__(self, cu, act, name, nt, k, n, gap=0, seed=0):
        gen = torch.Generator().manual_seed(nt + k + n + seed)
        self.cu, self.act, self.name, self.t, self.nt, self.k, self.n, self.gap = cu, act, name, TYPES[name], nt, k, n, gap
        rnd = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
        rows = lambda r, c: rnd(r, c + gap).to(self.t).cuda()  # noqa: E731
        self.x, self.dout = rows(nt, k), rows(nt, n)
        self.g, self.u = (rnd(n, k) * (2.0 / k ** 0.5)).to(self.t).cuda(), (rnd(n, k) / k ** 0.5).to(self.t).cuda()
        self.out = torch.full((nt, n + gap), 7.0, dtype=self.t, device="cuda")
        self.dx = torch.full((nt, k + gap), 7.0, dtype=self.t, device="cuda")
        self.pre = torch.empty(2, nt, n, device="cuda")
        self.dpre = torch.empty(2, nt, n, dtype=self.t, device="cuda")
        self.dg, self.du = torch.empty(n, k, dtype=self.t, device="cuda"), torch.empty(n, k, dtype=self.t, device="cuda")
        self.ids = {"silu": cu.ACT_SILU, "gelu": cu.ACT_GELU}[act], {"f16": cu.F16, "bf16": cu.BF16}[name]

    def forward(self, ctx, keep=True):
        return ctx.gated_dev(*self.ids, self.x.data_ptr(), self.g.data_ptr(), self.u.data_ptr(), self.nt, self.k, self.n, self.out.data_ptr(),
                             self.pre.data_ptr() if keep else None, self.k + self.gap, self.n + self.gap)

    def backward(self, ctx, dx=True, dw=True):
        return ctx.gated_backward_dev(*self.ids, self.x.data_ptr() if dw else None, self.g.data_ptr() if dx else None, self.u.data_ptr() if dx else None,
                                      self.pre.data_ptr(), self.dout.data_ptr(), self.nt, self.k, self.n, self.dpre.data_ptr(),
                                      self.dx.data_ptr() if dx else None, self.dg.data_ptr() if dw else None, self.du.data_ptr() if dw else None,
                                      self.k + self.gap, self.n + self.gap, self.k + self.gap)

    def wide(self):
        x, dout = self.x[:, :self.k], self.dout[:, :self.n]
        return [v.double().cpu() for v in (x, self.g, self.u, dout)]


def check(what, got, want, off):
    bad = (got.double().cpu() - want).abs() > off
    assert not bad.any(), "%s: %d of %d, first %s: %r for %r (may be %r off)" % (
        what, bad.sum(), bad.numel(), bad.nonzero()[0].tolist(), got.cpu()[bad][0].item(), want[bad][0].item(), off[bad][0].item())


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("nt,k,n", SHAPES)
def test_both_directions(cu, ctx, act, name, nt, k, n):
    b = Block(cu, act, name, nt, k, n, gap=8 if nt % 2 else 0)
    assert b.forward(ctx)
    assert b.backward(ctx)
    torch.cuda.synchronize()
    x, wg, wu, dout = b.wide()
    half, least = dh.half_step(b.t), dh.floor_of(b.t)
    g, u = (x @ wg.T).requires_grad_(), x @ wu.T
    a = dh.act(act, g)
    slope, = torch.autograd.grad(a.sum(), g)
    g, a = g.detach(), a.detach()
    off_g, off_u = dh.sum_error(k, x.abs() @ wg.abs().T), dh.sum_error(k, x.abs() @ wu.abs().T)
    off_a = dh.SLOPE * off_g + 2.0 ** -20 * g.abs()  # the activation in 32 bits: a few steps
    off_s = dh.BEND * off_g + 2.0 ** -19 * (1 + g.abs())
    want = a * u
    off = off_a * (u.abs() + off_u) + a.abs() * off_u
    check("out", b.out[:, :n], want, off + half * (want.abs() + off) + least)
    check("gate", b.pre[0], g, off_g)
    check("up", b.pre[1], u, off_u)
    dg, du = dout * u * slope, dout * a
    off_dg = dout.abs() * (off_u * (slope.abs() + off_s) + u.abs() * off_s)
    off_du = dout.abs() * off_a
    off_dg = off_dg + (half + 2.0 ** -22) * (dg.abs() + off_dg) + least
    off_du = off_du + (half + 2.0 ** -22) * (du.abs() + off_du) + least
    check("dgate before", b.dpre[0], dg, off_dg)
    check("dup before", b.dpre[1], du, off_du)
    want = dg @ wg + du @ wu
    size = (dg.abs() + off_dg) @ wg.abs() + (du.abs() + off_du) @ wu.abs()
    off = off_dg @ wg.abs() + off_du @ wu.abs() + dh.sum_error(2 * n, size)
    check("dx", b.dx[:, :k], want, off + half * (want.abs() + off) + least)
    for what, d, off_d, got in (("dgate", dg, off_dg, b.dg), ("dup", du, off_du, b.du)):
        want, off = d.T @ x, off_d.T @ x.abs() + dh.sum_error(nt, (d.abs() + off_d).T @ x.abs())
        check(what, got, want, off + half * (want.abs() + off) + least)
    if b.gap:
        assert bool((b.out[:, n:] == 7).all()) and bool((b.dx[:, k:] == 7).all())


@pytest.mark.parametrize("nt,k,n", [(77, 2056, 5640), (3000, 72, 2056), (8, 4096, 4096), (2000, 2048, 136), (2900, 2048, 264), (2600, 2304, 1408), (4700, 640, 1032)])
def test_many_tiles(cu, ctx, nt, k, n):
    """Several tiles for every SM, with next to nothing between them: sums of the kernel's own 16-bit operands, every time the same bits."""
    b = Block(cu, "silu", "bf16", nt, k, n)
    first = None
    for _ in range(4):
        for t in (b.out, b.dx, b.dg, b.du):
            t.fill_(7)
        assert b.forward(ctx) and b.backward(ctx)
        torch.cuda.synchronize()
        got = [t.clone() for t in (b.out, b.pre, b.dx, b.dg, b.du)]
        first = first or got
        assert all(torch.equal(p, q) for p, q in zip(got, first))
    x, wg, wu, _ = (v.cuda() for v in b.wide())
    dg, du, half = b.dpre[0].double(), b.dpre[1].double(), dh.half_step(b.t)
    for got, want, off in ((b.pre[0], x @ wg.T, dh.sum_error(k, x.abs() @ wg.abs().T)), (b.pre[1], x @ wu.T, dh.sum_error(k, x.abs() @ wu.abs().T)),
                           (b.dg, dg.T @ x, dh.sum_error(nt, dg.abs().T @ x.abs())), (b.du, du.T @ x, dh.sum_error(nt, du.abs().T @ x.abs())),
                           (b.dx, dg @ wg + du @ wu, dh.sum_error(2 * n, dg.abs() @ wg.abs() + du.abs() @ wu.abs()))):
        off = off + (half * (want.abs() + off) if got.dtype is b.t else 0)
        assert int(((got.double() - want).abs() > off + dh.floor_of(b.t)).sum()) == 0


@pytest.mark.parametrize("nt,k,n", [(3000, 64, 1032), (20, 1024, 264), (700, 2048, 136)])
def test_results_off_their_alignment(cu, ctx, nt, k, n):
    """out and dx at odd addresses with rows of odd distances, beside pre in 32 bits: the bits of the aligned call."""
    b = Block(cu, "gelu", "bf16", nt, k, n)
    assert b.forward(ctx) and b.backward(ctx)
    torch.cuda.synchronize()
    want = [t.clone() for t in (b.out, b.pre, b.dx, b.dg, b.du)]
    for _ in range(3):
        out, dx = (torch.full((nt * (w + 5) + 1,), 9.0, dtype=b.t, device="cuda") for w in (n, k))
        dg, du = (torch.full((n * k + 1,), 9.0, dtype=b.t, device="cuda") for _ in range(2))
        b.pre.fill_(0)
        assert ctx.gated_dev(*b.ids, b.x.data_ptr(), b.g.data_ptr(), b.u.data_ptr(), nt, k, n, out.data_ptr() + 2, b.pre.data_ptr(), 0, n + 5)
        assert ctx.gated_backward_dev(*b.ids, b.x.data_ptr(), b.g.data_ptr(), b.u.data_ptr(), b.pre.data_ptr(), b.dout.data_ptr(), nt, k, n, b.dpre.data_ptr(),
                                      dx.data_ptr() + 2, dg.data_ptr() + 2, du.data_ptr() + 2, 0, 0, k + 5)
        torch.cuda.synchronize()
        for got, w, width in ((out[1:].reshape(nt, n + 5), want[0], n), (dx[1:].reshape(nt, k + 5), want[2], k)):
            assert torch.equal(got[:, :width], w) and bool((got[:, width:] == 9).all())
        assert torch.equal(b.pre, want[1]) and torch.equal(dg[1:].reshape(n, k), want[3]) and torch.equal(du[1:].reshape(n, k), want[4])
        assert all(float(t[0]) == 9 for t in (out, dx, dg, du))


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gradients_against_differences(cu, ctx, act):
    """Along random directions: (f(p + h d) - f(p - h d)) / 2 h in 64 bits against the kernel's gradients."""
    b = Block(cu, act, "f16", 21, 136, 264)
    assert b.forward(ctx) and b.backward(ctx)
    torch.cuda.synchronize()
    x, wg, wu, dout = b.wide()
    f = lambda x, wg, wu: float((dh.act(act, x @ wg.T) * (x @ wu.T) * dout).sum())  # noqa: E731
    gen = torch.Generator().manual_seed(9)
    for at, grad in ((0, b.dx), (1, b.dg), (2, b.du)):
        grad = grad.double().cpu()
        d = torch.randn(grad.shape, generator=gen, dtype=torch.float64) + grad.sign()  # partly along the gradient: the sum does not cancel
        p = [x, wg, wu]
        p[at] = p[at] + 1e-5 * d
        up = f(*p)
        p[at] = p[at] - 2e-5 * d
        got, want = float((grad * d).sum()), (up - f(*p)) / 2e-5
        # every element within three roundings of 2^-11 of its terms; the sum of magnitudes bounds what they add up to
        assert abs(got - want) <= 4 * 2.0 ** -11 * float((grad.abs() * d.abs()).sum()) * 3


@pytest.mark.parametrize("dx,dw", [(True, False), (False, True), (False, False)])
def test_parts_of_the_backward_pass(cu, ctx, dx, dw):
    b, whole = Block(cu, "silu", "bf16", 50, 264, 136), Block(cu, "silu", "bf16", 50, 264, 136)
    for v, parts in ((whole, (True, True)), (b, (dx, dw))):
        for t in (v.dx, v.dg, v.du):
            t.fill_(3)
        assert v.forward(ctx) and v.backward(ctx, *parts)
    torch.cuda.synchronize()
    assert torch.equal(b.dpre, whole.dpre)
    for part, ran, names in ((b, dx, ("dx",)), (b, dw, ("dg", "du"))):
        for name in names:
            got = getattr(part, name)
            assert torch.equal(got, getattr(whole, name)) if ran else bool((got == 3).all())


def test_nothing_kept_without_a_backward_pass(cu, ctx):
    b, kept = Block(cu, "gelu", "bf16", 30, 72, 136), Block(cu, "gelu", "bf16", 30, 72, 136)
    b.pre.fill_(5)
    assert b.forward(ctx, keep=False) and kept.forward(ctx)
    torch.cuda.synchronize()
    assert torch.equal(b.out, kept.out) and bool((b.pre == 5).all())


def test_far_arguments(cu, ctx):
    """Pre-activations far beyond where the activations saturate: finite results, and zero slope on the far side."""
    for act in ("silu", "gelu"):
        b = Block(cu, act, "bf16", 4, 64, 64)
        b.x.fill_(1)
        b.g.copy_(torch.linspace(-40, 40, 64).reshape(64, 1).expand(64, 64))
        b.u.fill_(1 / 64)
        b.dout.fill_(1)
        assert b.forward(ctx) and b.backward(ctx)
        torch.cuda.synchronize()
        x, wg, wu, _ = b.wide()
        g = x @ wg.T
        assert torch.isfinite(b.out.float()).all() and torch.isfinite(b.dx.float()).all() and torch.isfinite(b.dg.float()).all()
        assert bool((b.out[g.cuda() < -200].float().abs() <= 1e-30).all())
        hi = g.cuda() > 200
        assert torch.equal(b.out[hi].float(), g.cuda().bfloat16().float()[hi])


def test_captured_and_replayed(cu, ctx):
    """A training step in a graph, replayed on changed inputs: what direct calls on them give."""
    b = Block(cu, "silu", "bf16", 90, 136, 264)
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    assert b.forward(ctx) and b.backward(ctx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        assert b.forward(ctx) and b.backward(ctx)
    b.x.mul_(-0.5)
    b.dout.mul_(2)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    got = [v.clone() for v in (b.out, b.dx, b.dg, b.du)]
    assert b.forward(ctx) and b.backward(ctx)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, (b.out, b.dx, b.dg, b.du)))
    del graph
    ctx.set_stream(1)


def test_no_tokens(cu, ctx):
    b = Block(cu, "silu", "bf16", 1, 64, 72)
    b.nt = 0
    for t in (b.dg, b.du, b.out, b.dx):
        t.fill_(3)
    assert b.forward(ctx) and b.backward(ctx)
    torch.cuda.synchronize()
    assert not b.dg.any() and not b.du.any()
    assert bool((b.out == 3).all()) and bool((b.dx == 3).all())


def test_four_bit_weights_by_their_values(cu, ctx):
    """Weights quantised, brought back to BF16 (exact) and used by the 16-bit block: the 4-bit block's values on the same rows, to rounding."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    nt, k, n = 24, 256, 320
    x = (torch.randn(nt, k, generator=gen, device="cuda")).bfloat16()
    four, wide, alive = [], [], []
    for m in (x, torch.randn(n, k, generator=gen, device="cuda") / 16, torch.randn(n, k, generator=gen, device="cuda") / 16):
        nc, ns = cu.mx4_bytes(*m.shape)
        codes, scales = torch.empty(nc, dtype=torch.uint8, device="cuda"), torch.empty(ns, dtype=torch.uint8, device="cuda")
        ty = cu.BF16 if m.dtype is torch.bfloat16 else cu.F32
        assert ctx.mx4_quantize_dev(ty, m.data_ptr(), *m.shape, codes.data_ptr(), scales.data_ptr())
        back = torch.empty(m.shape, dtype=torch.bfloat16, device="cuda")
        assert ctx.mx4_dequantize_dev(codes.data_ptr(), scales.data_ptr(), *m.shape, cu.BF16, back.data_ptr())
        four += [codes.data_ptr(), scales.data_ptr()]
        wide += [back]
        torch.cuda.synchronize()
        alive.append((codes, scales))
    a, b = torch.empty(nt, n, dtype=torch.bfloat16, device="cuda"), torch.empty(nt, n, dtype=torch.bfloat16, device="cuda")
    assert ctx.mx4_gated_dev(cu.ACT_SILU, *four, nt, k, n, cu.BF16, a.data_ptr())
    assert ctx.gated_dev(cu.ACT_SILU, cu.BF16, *(w.data_ptr() for w in wide), nt, k, n, b.data_ptr())
    torch.cuda.synchronize()
    off = 2.0 ** -7 * b.float().abs() + 1e-5  # a rounding each, and sums of 256 products in 32 bits
    assert bool(((a.float() - b.float()).abs() <= off).all())
