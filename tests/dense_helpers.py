"""Plain forms, in 64 bits, of the dense operators (microscaled 4-bit matrices, the gated feed-forward block), and how far a kernel may be off."""
import math

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantise(x):
    """x [rows][k] -> (codes [rows][k] 0..15, scale bytes [rows][k / 32]), on the CPU, element by element from the definition."""
    b = x.detach().cpu().double().reshape(x.shape[0], -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    finite = torch.isfinite(amax)
    _, ex = torch.frexp(torch.where(finite, amax, 1.0))  # amax = m * 2^ex, m in [0.5, 1)
    e = torch.where(amax > 0, (ex - 1 - 2).clamp(min=-127), -127)
    a = torch.where(finite, b, 0.0) * torch.pow(torch.tensor(2.0, dtype=torch.float64), -e.double())
    dist = (a.abs().unsqueeze(-1) - GRID).abs()
    near = dist.min(-1, keepdim=True).values
    code = torch.arange(8).expand_as(dist)
    tied = torch.where(dist == near, code, 99)  # ties (two neighbours, one of them even): to the even code
    lo, hi = tied.min(-1).values, torch.where(tied == 99, -1, tied).max(-1).values
    code = torch.where(lo % 2 == 0, lo, hi)
    code = code + 8 * torch.signbit(b).long()
    code = torch.where(finite, code, 0)
    e = torch.where(finite, e + 127, 255)
    return code.reshape(x.shape).to(torch.uint8), e.squeeze(-1).to(torch.uint8)


def values(code, e):
    v = GRID[(code & 7).long()] * torch.where(code >= 8, -1.0, 1.0).double()
    s = torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double() - 127)
    s = torch.where(e == 255, math.nan, s)
    return (v.reshape(e.shape[0], -1, 32) * s.unsqueeze(-1)).reshape(code.shape)


def place(r, j, k):
    """Byte of scale j of row r."""
    return ((r // 128) * -(-k // 128) + j // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + j % 4


def pack(code, e, dirty=0):
    """(codes, scales) as they lie in memory, on the GPU; bytes of rows beyond the matrix are `dirty`."""
    rows, k = code.shape
    packed = (code[:, 0::2] | code[:, 1::2] << 4).contiguous()
    nkb, nrb = -(-k // 128), -(-rows // 128)
    full = torch.full((nrb * 128, nkb * 4), dirty, dtype=torch.uint8)
    full[:rows] = 0
    full[:rows, :k // 32] = e
    r, j = torch.meshgrid(torch.arange(nrb * 128), torch.arange(nkb * 4), indexing="ij")
    scales = torch.empty(nrb * nkb * 512, dtype=torch.uint8)
    scales[place(r, j, k).reshape(-1)] = full.reshape(-1)
    return packed.cuda(), scales.cuda()


def unpack(codes, scales, rows, k):
    codes, scales = codes.cpu(), scales.cpu()
    code = torch.stack([codes & 15, codes >> 4], -1).reshape(rows, k)
    r, j = torch.meshgrid(torch.arange(rows), torch.arange(k // 32), indexing="ij")
    return code, scales[place(r, j, k)]


def random_codes(gen, rows, k, lo=120, hi=134):
    code = torch.randint(0, 16, (rows, k), generator=gen, dtype=torch.uint8)
    e = torch.randint(lo, hi, (rows, k // 32), generator=gen, dtype=torch.uint8)
    return code, e


def act(name, g):
    return g * torch.sigmoid(g) if name == "silu" else torch.nn.functional.gelu(g, approximate="tanh")


# Largest |act'| and |act''| of either activation, for what an error of its argument can do.
SLOPE, BEND = 1.13, 1.0


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def floor_of(dtype):
    """The least step of a type: results below its normal numbers are off by at most this."""
    return torch.finfo(dtype).tiny * (torch.finfo(dtype).eps if dtype is torch.float16 else 1)


def sum_error(k, size):
    """A sum of k exact products, kept in 32 bits by the tensor core, which truncates (a step of the running sum, 2^-23, for each 16 of k at least),
    and split eight ways at most: k / 16 + 16 steps of the sum of magnitudes."""
    return (k / 16 + 16) * 2.0 ** -23 * size
