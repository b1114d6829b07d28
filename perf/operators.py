"""Operators of dense layers as cases that can be timed: microscaled 4-bit matrices and the gated feed-forward block.

A microscaled matrix holds 4-bit floating point numbers (sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6)
with a power of two for each 32 of a row.  In memory it is two arrays: codes [rows][k / 2], element 2 i in the low half of
byte i, and scales (2^(byte - 127)) in tiles of 128 rows x 4 scales, scale j of row r at byte
    ((r / 128) * ceil(k / 128) + j / 4) * 512 + (r % 32) * 16 + (r % 128) / 32 * 4 + j % 4,
zeros where a tile reaches beyond the matrix.  Quantisation: the scale's exponent is floor(log2(largest magnitude)) - 2, at least
-127; elements are rounded to nearest, ties to even, and beyond 6 to 6.

    quantise   rows -> 4 bits (-> the values they stand for)
    product    out[t][r] = sum_i X[t][i] W[r][i], both in 4 bits: a linear layer's
    gated4     out = act(X G^T) * (X U^T), all three in 4 bits
    ffn4       a feed-forward block in 4 bits: quantise, gated4 (result in 4 bits), product
    gated      act(x G^T) * (x U^T) with 16-bit operands
    train      the same, and the gradients of x, G and U

    listed()  the cases            draw(rng)  one more of the same ranges
    prepare(case, seed)            operands and output buffers, as a program keeps them
    run(state)                     one pass; returns its outputs
    exact(case, seed)              the same in 64 bits
    work(case)                     what a pass cannot do without
"""
import math

import torch

own = False

TYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # The input of one decoded token's layer, the smallest call: latency.
        dict(name="quantise, one row of 2048", kind="quantise", nt=1, k=2048, ty="f32"),
        # A long prompt's activations, or a layer's weights as they are loaded.
        dict(name="quantise, 14018 rows of 4096", kind="quantise", nt=14018, k=4096, ty="bf16"),
        # One decoded token through a square projection.
        dict(name="product, one token, 4096 x 4096", kind="product", nt=1, k=4096, n=4096, ty="f32"),
        # Eight sequences at the output head: the weights' bytes count.
        dict(name="product, 8 tokens, 65536 x 4096", kind="product", nt=8, k=4096, n=65536, ty="f32"),
        # A prompt chunk through a projection of odd sizes.
        dict(name="product, 500 tokens, 4064 -> 5003", kind="product", nt=500, k=4064, n=5003, ty="bf16"),
        # A long prompt, or a batch of them: the tensor cores' rate counts.
        dict(name="product, 8192 tokens, 4096 -> 8192", kind="product", nt=8192, k=4096, n=8192, ty="bf16"),
        # One decoded token through both projections of a feed-forward block.
        dict(name="4-bit gated, one token, 2048 -> 8192", kind="gated4", nt=1, k=2048, n=8192, ty="bf16", act="silu"),
        # A prompt chunk through a whole feed-forward block in 4 bits.
        dict(name="4-bit block, 512 tokens, 4096 -> 12288", kind="ffn4", nt=512, k=4096, n=12288, ty="bf16", act="silu"),
        # 16-bit weights (a leading dense layer, a shared expert): four sequences, and a chunk.
        dict(name="gated, 4 tokens, 4096 -> 10240", kind="gated", nt=4, k=4096, n=10240, ty="bf16", act="silu"),
        dict(name="gated, 512 tokens, 2560 -> 9728, gelu", kind="gated", nt=512, k=2560, n=9728, ty="f16", act="gelu"),
        # Fine-tuning such a block: a short text at odd sizes, and a full batch.
        dict(name="training step, 77 tokens, 2056 -> 5640", kind="train", nt=77, k=2056, n=5640, ty="f16", act="gelu"),
        dict(name="training step, 4096 tokens, 4096 -> 10240", kind="train", nt=4096, k=4096, n=10240, ty="bf16", act="silu"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantise", "product", "product", "gated4", "ffn4", "gated", "train", "train"])
    if kind == "quantise":
        return dict(kind=kind, nt=_log(rng, 1, 8000), k=32 * _log(rng, 4, 220), ty=rng.choice(["f32", "bf16", "f16"]))
    nt = _log(rng, 1, 6000)
    if kind == "product":
        return dict(kind=kind, nt=nt, k=32 * _log(rng, 4, 300), n=_log(rng, 100, 9000), ty=rng.choice(["f32", "bf16", "f16"]))
    if kind in ("gated4", "ffn4"):
        return dict(kind=kind, nt=nt, k=32 * _log(rng, 8, 140), n=32 * _log(rng, 8, 380), ty=rng.choice(["bf16", "f16"]), act=rng.choice(["silu", "gelu"]))
    return dict(kind=kind, nt=min(nt, 4096), k=8 * _log(rng, 16, 512), n=8 * _log(rng, 16, 1280), ty=rng.choice(["bf16", "f16"]), act=rng.choice(["silu", "gelu"]))


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _normal(gen, sigma, *shape):
    return torch.randn(*shape, generator=gen, device="cuda") * sigma


def _activations(gen, nt, k, ty):
    """Normal, with one channel in 64 ten times as large, as a network's residual stream has them."""
    x = _normal(gen, 1.0, nt, k)
    return (x * torch.where(torch.rand(k, generator=gen, device="cuda") < 1 / 64, 10.0, 1.0)).to(TYPE[ty])


def _inputs(case, seed):
    """The numbers of a case before any of them is held in 4 bits."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, nt, k = case["kind"], case["nt"], case["k"]
    if kind == "quantise":
        return {"x": _activations(gen, nt, k, case["ty"])}
    n, ty = case["n"], TYPE[case["ty"]]
    if kind == "product":
        return {"x": _activations(gen, nt, k, "f32"), "w": _normal(gen, k ** -0.5, n, k)}
    if kind in ("gated4", "ffn4"):
        made = {"x": _activations(gen, nt, k, "bf16"), "g": _normal(gen, k ** -0.5, n, k), "u": _normal(gen, k ** -0.5, n, k)}
        return dict(made, d=_normal(gen, n ** -0.5, k, n)) if kind == "ffn4" else made
    made = {"x": _normal(gen, 1.0, nt, k).to(ty), "g": _normal(gen, k ** -0.5, n, k).to(ty), "u": _normal(gen, k ** -0.5, n, k).to(ty)}
    return dict(made, dout=_normal(gen, 1.0, nt, n).to(ty)) if kind == "train" else made


# ---- 4 bits, in elementary operations -------------------------------------------------------------------------------------

def _quantise(x):
    """(codes [rows][k], exponents [rows][k / 32] + 127): a number per element."""
    x = x.float().reshape(x.shape[0], -1, 32)
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.where(amax > 0, torch.frexp(amax).exponent + (127 - 3), 0).clamp(min=0)
    a = (x.abs() * torch.exp2((127 - e).double())).float()  # by a power of two: exact, or far below the least step
    code = ((a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).byte()
    code = code + 8 * torch.signbit(x).byte()
    return code.reshape(x.shape[0], -1), e.squeeze(-1).byte()


def _values(code, e):
    """The fp32 numbers that codes and exponents stand for."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=code.device)
    v = table[(code & 7).int()] * torch.where(code >= 8, -1.0, 1.0)
    scale = torch.exp2(e.double() - 127).float()
    return (v.reshape(*e.shape, 32) * scale.unsqueeze(-1)).reshape(code.shape)


def _tiled(e):
    """Scales [rows][k / 32] as they lie in memory."""
    rows, kb = e.shape
    r, t = -(-rows // 128), -(-kb // 4)
    full = torch.zeros(r * 128, t * 4, dtype=torch.uint8, device=e.device)
    full[:rows, :kb] = e
    return full.reshape(r, 4, 32, t, 4).permute(0, 3, 2, 1, 4).contiguous().reshape(-1)


def _untiled(scales, rows, k):
    r, t = -(-rows // 128), -(-k // 128)
    return scales.reshape(r, t, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(r * 128, t * 4)[:rows, :k // 32]


def _packed(x):
    code, e = _quantise(x)
    return code[:, 0::2] | code[:, 1::2] << 4, _tiled(e)


def _unpacked(m):
    codes, scales = m
    code = torch.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)
    return _values(code, _untiled(scales, *code.shape))


# ---- preparation ------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    kind, nt, k, n, ty = case["kind"], case["nt"], case["k"], case.get("n"), TYPE[case["ty"]]
    made = _inputs(case, seed)
    empty = lambda *shape, dtype=torch.uint8: torch.empty(*shape, dtype=dtype, device="cuda")  # noqa: E731
    tiles = lambda rows, k: -(-rows // 128) * -(-k // 128) * 512  # noqa: E731
    s = {"case": case}
    for name, m in made.items():
        s[name] = _packed(m) if kind in ("product", "gated4") or (kind == "ffn4" and name != "x") else m
    if kind in ("quantise", "ffn4"):
        s["x4"] = empty(nt, k // 2), empty(tiles(nt, k))
    if kind == "quantise":
        s["out"] = empty(nt, k, dtype=torch.bfloat16)
    elif kind == "ffn4":
        s["h4"] = empty(nt, n // 2), empty(tiles(nt, n))
        s["out"] = empty(nt, k, dtype=ty)
    else:
        s["out"] = empty(nt, n, dtype=ty)
    if kind == "train":
        s["pre"], s["dpre"] = empty(2, nt, n, dtype=torch.float32), empty(2, nt, n, dtype=ty)
        s["dx"], s["dg"], s["du"] = empty(nt, k, dtype=ty), empty(n, k, dtype=ty), empty(n, k, dtype=ty)
    torch.cuda.synchronize()
    return s


# ---- a pass ------------------------------------------------------------------------------------------------------------------

_contexts = {}


def _context():
    """The framework and its context for the current device and the stream that torch works on there, now: a context works on one stream.
    Asked by torch's raw calls: a Stream object takes as long as a small call."""
    device = torch._C._cuda_getDevice()
    stream = torch._C._cuda_getCurrentRawStream(device)
    found = _contexts.get((device, stream))
    if found is None:
        from denno_beta_b200 import cuda as cu
        found = _contexts[device, stream] = cu, cu.CudaCtx(device)
        found[1].set_stream(stream or 1)  # 1: the default stream by its handle
    return found


def _done(ok):
    if not ok:
        raise RuntimeError("the library declined the call")


def _ptrs(m):
    return m[0].data_ptr(), m[1].data_ptr()


def run(s):
    if own:
        cu, ctx = _context()
        return OWN[s["case"]["kind"]](s, s["case"], cu, ctx)
    return PLAIN[s["case"]["kind"]](s, s["case"])


def _own_type(cu, case):
    return {"f32": cu.F32, "f16": cu.F16, "bf16": cu.BF16}[case["ty"]]


def _own_act(cu, case):
    return {"silu": cu.ACT_SILU, "gelu": cu.ACT_GELU}[case["act"]]


def _own_quantise(s, case, cu, ctx):
    _done(ctx.mx4_quantize_dev(_own_type(cu, case), s["x"].data_ptr(), case["nt"], case["k"], *_ptrs(s["x4"])))
    _done(ctx.mx4_dequantize_dev(*_ptrs(s["x4"]), case["nt"], case["k"], cu.BF16, s["out"].data_ptr()))
    return s["out"]


def _own_product(s, case, cu, ctx):
    _done(ctx.mx4_gemm_dev(*_ptrs(s["x"]), *_ptrs(s["w"]), case["nt"], case["k"], case["n"], _own_type(cu, case), s["out"].data_ptr()))
    return s["out"]


def _own_gated4(s, case, cu, ctx):
    _done(ctx.mx4_gated_dev(_own_act(cu, case), *_ptrs(s["x"]), *_ptrs(s["g"]), *_ptrs(s["u"]), case["nt"], case["k"], case["n"], _own_type(cu, case),
                            s["out"].data_ptr()))
    return s["out"]


def _own_ffn4(s, case, cu, ctx):
    nt, k, n = case["nt"], case["k"], case["n"]
    _done(ctx.mx4_quantize_dev(cu.BF16, s["x"].data_ptr(), nt, k, *_ptrs(s["x4"])))
    _done(ctx.mx4_gated_dev(_own_act(cu, case), *_ptrs(s["x4"]), *_ptrs(s["g"]), *_ptrs(s["u"]), nt, k, n, cu.MXFP4, *_ptrs(s["h4"])))
    _done(ctx.mx4_gemm_dev(*_ptrs(s["h4"]), *_ptrs(s["d"]), nt, n, k, _own_type(cu, case), s["out"].data_ptr()))
    return s["out"]


def _own_gated(s, case, cu, ctx, pre=None):
    _done(ctx.gated_dev(_own_act(cu, case), _own_type(cu, case), s["x"].data_ptr(), s["g"].data_ptr(), s["u"].data_ptr(), case["nt"], case["k"], case["n"],
                        s["out"].data_ptr(), pre))
    return s["out"]


def _own_train(s, case, cu, ctx):
    _own_gated(s, case, cu, ctx, s["pre"].data_ptr())
    _done(ctx.gated_backward_dev(_own_act(cu, case), _own_type(cu, case), s["x"].data_ptr(), s["g"].data_ptr(), s["u"].data_ptr(), s["pre"].data_ptr(),
                                 s["dout"].data_ptr(), case["nt"], case["k"], case["n"], s["dpre"].data_ptr(), s["dx"].data_ptr(), s["dg"].data_ptr(),
                                 s["du"].data_ptr()))
    return {"out": s["out"], "dx": s["dx"], "dg": s["dg"], "du": s["du"]}


OWN = {"quantise": _own_quantise, "product": _own_product, "gated4": _own_gated4, "ffn4": _own_ffn4, "gated": _own_gated, "train": _own_train}


def _act(name, g):
    if name == "silu":
        return g / (1 + torch.exp(-g))
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))


def _act_slope(name, g):
    if name == "silu":
        p = 1 / (1 + torch.exp(-g))
        return p * (1 + g * (1 - p))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


def _plain_quantise(s, case):
    return _values(*_quantise(s["x"])).to(torch.bfloat16)


def _plain_product(s, case):
    return (_unpacked(s["x"]) @ _unpacked(s["w"]).T).to(TYPE[case["ty"]])


def _plain_gated4(s, case):
    x = _unpacked(s["x"])
    return (_act(case["act"], x @ _unpacked(s["g"]).T) * (x @ _unpacked(s["u"]).T)).to(TYPE[case["ty"]])


def _plain_ffn4(s, case):
    x = _values(*_quantise(s["x"]))
    h = _act(case["act"], x @ _unpacked(s["g"]).T) * (x @ _unpacked(s["u"]).T)
    return (_values(*_quantise(h)) @ _unpacked(s["d"]).T).to(TYPE[case["ty"]])


def _plain_gated(s, case):
    x = s["x"].float()
    return (_act(case["act"], x @ s["g"].float().T) * (x @ s["u"].float().T)).to(TYPE[case["ty"]])


def _plain_train(s, case):
    x, wg, wu, dout, act = s["x"].float(), s["g"].float(), s["u"].float(), s["dout"].float(), case["act"]
    g, u = x @ wg.T, x @ wu.T
    a = _act(act, g)
    dg, du = dout * u * _act_slope(act, g), dout * a
    found = {"out": a * u, "dx": dg @ wg + du @ wu, "dg": dg.T @ x, "du": du.T @ x}
    return {name: v.to(TYPE[case["ty"]]) for name, v in found.items()}


PLAIN = {"quantise": _plain_quantise, "product": _plain_product, "gated4": _plain_gated4, "ffn4": _plain_ffn4, "gated": _plain_gated, "train": _plain_train}


# ---- in 64 bits --------------------------------------------------------------------------------------------------------------

def _exact4(x):
    """What x stands for once it is held in 4 bits: by the step of the grid between two powers of two."""
    b = x.double().unflatten(-1, (-1, 32))
    largest = b.abs().amax(-1, keepdim=True)
    unit = torch.pow(2.0, (torch.frexp(largest)[1].double() - 3).clamp(min=-127)).double()  # frexp: a logarithm may fall short of a power of two
    a = b / unit
    step = torch.where(a.abs() < 2, 0.5, torch.where(a.abs() < 4, 1.0, 2.0))
    return ((torch.round(a / step) * step).clamp(-6, 6) * unit).flatten(-2)


def exact(case, seed):
    made, kind = _inputs(case, seed), case["kind"]
    if kind == "quantise":
        return _exact4(made["x"])
    if kind == "product":
        return _exact4(made["x"]) @ _exact4(made["w"]).T
    smooth = {"silu": lambda v: v * torch.sigmoid(v), "gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[case["act"]]
    if kind in ("gated4", "ffn4"):
        x = _exact4(made["x"])
        h = smooth(x @ _exact4(made["g"]).T) * (x @ _exact4(made["u"]).T)
        return h if kind == "gated4" else _exact4(h) @ _exact4(made["d"]).T
    x, g, u = (made[name].double().requires_grad_(kind == "train") for name in ("x", "g", "u"))
    out = smooth(x @ g.T) * (x @ u.T)
    if kind == "gated":
        return out
    dx, dg, du = torch.autograd.grad(out, (x, g, u), made["dout"].double())
    return {"out": out.detach(), "dx": dx, "dg": dg, "du": du}


# ---- what a pass needs ---------------------------------------------------------------------------------------------------------

def _bytes4(rows, k):
    return rows * (k // 2 + k // 32)


def work(case):
    kind, nt, k, n, size = case["kind"], case["nt"], case["k"], case.get("n", 0), 4 if case["ty"] == "f32" else 2
    if kind == "quantise":  # in, 4 bits out, and the values that they stand for
        return {"bytes": nt * k * (size + 2) + _bytes4(nt, k), "flops": 3 * nt * k}
    if kind == "product":
        return {"bytes": _bytes4(nt, k) + _bytes4(n, k) + size * nt * n, "flops": 2 * nt * k * n}
    if kind == "gated4":
        return {"bytes": _bytes4(nt, k) + 2 * _bytes4(n, k) + size * nt * n, "flops": 4 * nt * k * n}
    if kind == "ffn4":
        return {"bytes": 4 * nt * k + 2 * _bytes4(n, k) + _bytes4(k, n), "flops": 6 * nt * k * n}
    if kind == "gated":
        return {"bytes": 2 * (nt * k + 2 * n * k + nt * n), "flops": 4 * nt * k * n}
    # x, both weights and the output's gradient in; the output and three gradients out
    return {"bytes": 2 * (2 * nt * k + 4 * n * k + 2 * nt * n), "flops": 12 * nt * k * n}
