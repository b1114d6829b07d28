"""Activations far from zero: what a call returns there is right relative to its own size, down to the least 32-bit numbers.  Operands are such that g and u are
exact, so that nothing but the activation, its slope and the product is rounded."""
import pytest
import torch

import dense_helpers as dh

pytestmark = pytest.mark.gpu
GRID = [6.0, 4.0, 3.0, 2.0, 1.5, 1.0, 0.5]
CODE = {0.0: 0, 0.5: 1, 1.0: 2, 1.5: 3, 2.0: 4, 3.0: 5, 4.0: 6, 6.0: 7}
N = 448
G = (torch.arange(N, dtype=torch.float64) - N // 2) / 2  # -112 to 111.5: beyond where exp(g) leaves the 32-bit numbers


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


def exponent(act, g):
    """(z, its slope) with act(g) = g / (1 + exp(-z)): tanh's form would cancel to nothing."""
    if act == "silu":
        return g, torch.ones_like(g)
    c = 2 * (2 / torch.pi) ** 0.5
    return c * (g + 0.044715 * g ** 3), c * (1 + 3 * 0.044715 * g ** 2)


def relative(act, z):
    """Of act, or of its product with an exact number, which is g / (1 + e), for negative g times e = h^2: the power of two h is off by 2^-22 (2 steps of 2^-23), so e by
    4, which the quotient takes over at most whole; the reciprocal by 1; five other operations by half a one each.  h's argument carries its constant's
    and its own rounding, 2^-24 of itself each, and gelu's three more (second constant, square, sum); h^2 is off by as much as z is."""
    return 7.5 * 2.0 ** -23 + {"silu": 2, "gelu": 5}[act] * 2.0 ** -24 * z.abs()


def as_codes(v):
    """A row of 32 grid elements that sum to v, a multiple of a half."""
    left, row = abs(v), []
    for _ in range(32):
        piece = next((p for p in GRID if p <= left), 0.0)
        left -= piece
        row.append(CODE[piece] + (8 if v < 0 and piece else 0))
    assert left == 0
    return row


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("nt", [1, 7, 40, 128, 200])
def test_four_bit_operands(cu, ctx, act, nt):
    k = 32
    one = torch.full((nt, k), CODE[1.0], dtype=torch.uint8), (127 - torch.arange(nt).reshape(nt, 1) % 4).to(torch.uint8)  # 1, 1/2, 1/4, 1/8
    gate = torch.tensor([as_codes(float(v)) for v in G], dtype=torch.uint8), torch.full((N, 1), 127, dtype=torch.uint8)
    up = torch.zeros(N, k, dtype=torch.uint8), torch.full((N, 1), 127, dtype=torch.uint8)
    up[0][:, 0] = CODE[1.0]
    packed = [t for m in (one, gate, up) for t in dh.pack(*m)]
    x = torch.pow(2.0, -(torch.arange(nt, dtype=torch.float64).reshape(nt, 1) % 4))
    g, u = x * G, x.expand(nt, N)
    z, _ = exponent(act, g)
    want = g * torch.sigmoid(z) * u
    least = (2 + 4 * g.abs()) * 2.0 ** -149
    ids = {"silu": cu.ACT_SILU, "gelu": cu.ACT_GELU}[act]
    for ty, dtype, half in ((cu.F32, torch.float32, 0.0), (cu.BF16, torch.bfloat16, 2.0 ** -8)):
        out = torch.full((nt, N), 7.0, dtype=dtype, device="cuda")
        assert ctx.mx4_gated_dev(ids, *(t.data_ptr() for t in packed), nt, k, N, ty, out.data_ptr())
        torch.cuda.synchronize()
        off = want.abs() * (relative(act, z) * (1 + half) + half) + least + (2.0 ** -134 if half else 0)
        bad = (out.cpu().double() - want).abs() > off
        assert not bad.any(), (int(bad.sum()), g[bad][0].item(), out.cpu()[bad][0].item(), want[bad][0].item())
        if half == 0:
            plain = out.clone()
    # and the 4-bit result is that of the 32-bit one
    nc, ns = cu.mx4_bytes(nt, N)
    codes, scales = torch.empty(nc, dtype=torch.uint8, device="cuda"), torch.empty(ns, dtype=torch.uint8, device="cuda")
    assert ctx.mx4_gated_dev(ids, *(t.data_ptr() for t in packed), nt, k, N, cu.MXFP4, codes.data_ptr(), scales.data_ptr())
    torch.cuda.synchronize()
    code, e = dh.unpack(codes, scales, nt, N)
    want_code, want_e = dh.quantise(plain)
    assert torch.equal(e, want_e) and torch.equal(code, want_code)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("nt", [3, 50, 140])
def test_sixteen_bit_operands_and_slopes(cu, ctx, act, nt):
    """dout and u are 1: dpre holds act'(g) and act(g) themselves."""
    k, t = 8, torch.bfloat16
    x, gate, up = torch.zeros(nt, k, dtype=t), torch.zeros(N, k, dtype=t), torch.zeros(N, k, dtype=t)
    x[:, 0], gate[:, 0], up[:, 0] = 1, G.to(t), 1
    x, gate, up, dout = x.cuda(), gate.cuda(), up.cuda(), torch.ones(nt, N, dtype=t, device="cuda")
    out, pre, dpre = torch.empty(nt, N, dtype=t, device="cuda"), torch.empty(2, nt, N, device="cuda"), torch.empty(2, nt, N, dtype=t, device="cuda")
    ids = {"silu": cu.ACT_SILU, "gelu": cu.ACT_GELU}[act], cu.BF16
    assert ctx.gated_dev(*ids, x.data_ptr(), gate.data_ptr(), up.data_ptr(), nt, k, N, out.data_ptr(), pre.data_ptr())
    assert ctx.gated_backward_dev(*ids, None, None, None, pre.data_ptr(), dout.data_ptr(), nt, k, N, dpre.data_ptr())
    torch.cuda.synchronize()
    g = G.expand(nt, N)
    assert torch.equal(pre[0].cpu().double(), g) and bool((pre[1] == 1).all())
    z, rise = exponent(act, g)
    p, rest = torch.sigmoid(z), torch.sigmoid(-z)
    value, slope, terms = g * p, p + g * p * rest * rise, p + (g * p * rest * rise).abs()
    half, least = 2.0 ** -8, (2 + 4 * g.abs()) * 2.0 ** -149 + 2.0 ** -134
    off = value.abs() * (relative(act, z) * (1 + half) + half) + least
    # the slope's second term has the other of p and 1 - p (the reciprocal again, and 3 operations) and z' (2 constants, square, sum, product) as factors, and
    # two operations join them; where it is 1 - p that has e, p has not, so that e counts once
    off_s = terms * (relative(act, z) + 6 * 2.0 ** -23) * (1 + half) + half * slope.abs() + least * (1 + rise)
    for what, got, want, o in (("out", out, value, off), ("act", dpre[1], value, off), ("slope", dpre[0], slope, off_s)):
        bad = (got.cpu().double() - want).abs() > o
        assert not bad.any(), (what, int(bad.sum()), g[bad][0].item(), got.cpu()[bad][0].item(), want[bad][0].item())
