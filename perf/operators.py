"""The operators of a feed-forward layer, as cases to measure: the gated product with its gradients, the gradients of
the plain "rc" product, and the microscaled 4-bit (MXFP4) quantisation and product.

Each case runs either in its plain form (elementary torch operations in 32 bits) or, with `own` set, through the calls
that a user of the `beam` package makes.  Layouts are those of the package: activations [rows, K], weights [N, K], both
row-major; 4-bit matrices as packed bytes [rows, K / 2] (element 2 i in the low half of byte i) with one power-of-two
scale byte for every 32 elements of a row, the scales in blocks of 128 rows x 4 scales (see `tile_scales`).
"""
import math
import os
import sys

import torch

own = False

if os.path.join(os.getcwd(), "general-nvgpu-testing_b200") not in sys.path:
    sys.path.insert(0, os.path.join(os.getcwd(), "general-nvgpu-testing_b200"))  # where the package lies in the repository

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ACTIVATIONS = ("silu", "gelu", "gelu_tanh", "relu")
LARGEST_FLOPS = 8.0 * 8192 * 4096 * 16384


# ---------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one token of a served sequence through the gated projections: bound by reading both weights
        {"name": "gated 1 token", "op": "gated", "m": 1, "k": 4096, "f": 16384, "type": "bf16", "act": "silu", "keep": False},
        # a small batch of served sequences, odd sizes throughout, the exact Gaussian activation
        {"name": "gated 77 rows odd", "op": "gated", "m": 77, "k": 2056, "f": 5464, "type": "fp16", "act": "gelu", "keep": False},
        # a training step's forward pass: the projections are kept for the backward pass
        {"name": "gated 4096 rows kept", "op": "gated", "m": 4096, "k": 4096, "f": 16384, "type": "bf16", "act": "silu", "keep": True},
        # the gradients of a small model's gated projections on a ragged batch
        {"name": "gated gradient odd", "op": "gated_backward", "m": 333, "k": 1000, "f": 2744, "type": "fp16", "act": "gelu_tanh"},
        # the gradients of a large training step: the costliest case
        {"name": "gated gradient 8192 rows", "op": "gated_backward", "m": 8192, "k": 4096, "f": 16384, "type": "bf16", "act": "silu"},
        # the gradients of a projection back to the model's width, ragged
        {"name": "product gradient odd", "op": "backward", "m": 1111, "n": 1048, "k": 2728, "type": "fp16"},
        # ... and of a training step
        {"name": "product gradient 8192 rows", "op": "backward", "m": 8192, "n": 4096, "k": 8192, "type": "bf16"},
        # activations to 4 bits and back, small and odd
        {"name": "mxfp4 round trip odd", "op": "quantize", "m": 333, "k": 1056, "type": "fp16"},
        # a large weight to 4 bits and back
        {"name": "mxfp4 round trip 16384 rows", "op": "quantize", "m": 16384, "k": 8192, "type": "bf16"},
        # one token through a projection whose weights were laid out in 4 bits beforehand
        {"name": "mxfp4 product 1 token", "op": "mx_linear", "m": 1, "n": 16384, "k": 8192, "type": "bf16"},
        # a ragged batch through a small projection
        {"name": "mxfp4 product odd", "op": "mx_linear", "m": 205, "n": 2072, "k": 1376, "type": "fp16"},
        # a long prompt through a large projection
        {"name": "mxfp4 product 8192 rows", "op": "mx_linear", "m": 8192, "n": 8192, "k": 8192, "type": "bf16"},
    ]


def _spread(rng, low, high, step):
    """A size between low and high, even over the logarithm, a multiple of step."""
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high))) / step + 0.5) * step))


def draw(rng):
    op = rng.choice(("gated", "gated", "gated_backward", "backward", "quantize", "mx_linear", "mx_linear"))
    case = {"op": op, "type": rng.choice(("bf16", "fp16"))}
    if op == "gated":
        case.update(m=_spread(rng, 1, 8192, 1), k=_spread(rng, 256, 8192, 8), f=_spread(rng, 256, 16384, 8),
                    act=rng.choice(ACTIVATIONS), keep=rng.random() < 0.5)
    elif op == "gated_backward":
        case.update(m=_spread(rng, 16, 8192, 1), k=_spread(rng, 256, 8192, 8), f=_spread(rng, 256, 16384, 8),
                    act=rng.choice(ACTIVATIONS))
    elif op == "backward":
        case.update(m=_spread(rng, 16, 16384, 1), n=_spread(rng, 256, 8192, 8), k=_spread(rng, 256, 8192, 8))
    elif op == "quantize":
        case.update(m=_spread(rng, 1, 16384, 1), k=_spread(rng, 64, 8192, 32))
    else:
        case.update(m=_spread(rng, 1, 8192, 1), n=_spread(rng, 256, 16384, 8), k=_spread(rng, 256, 8192, 32))
    while work(case)["flops"] > LARGEST_FLOPS:
        case["m"] = case["m"] // 2 + 1
    return case


def work(case):
    m, k = case["m"], case["k"]
    op = case["op"]
    if op == "gated":
        f = case["f"]
        return {"bytes": 2 * (m * k + 2 * f * k + m * f * (3 if case["keep"] else 1)), "flops": 4 * m * f * k}
    if op == "gated_backward":
        f = case["f"]
        return {"bytes": 2 * (3 * m * f + 2 * m * k + 4 * f * k), "flops": 8 * m * f * k}
    if op == "backward":
        n = case["n"]
        return {"bytes": 2 * (m * n + 2 * m * k + 2 * n * k), "flops": 4 * m * n * k}
    if op == "quantize":  # the values in, the packed bytes and scales, the values out
        return {"bytes": m * k * 2 + m * k // 2 + m * k // 32 + m * k * 2, "flops": 2 * m * k}
    n = case["n"]
    return {"bytes": 2 * m * k + n * k // 2 + n * k // 32 + 2 * m * n, "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------------ MXFP4 in elementary steps
def tile_scales(s):
    """Scale bytes [rows, K / 32] in the package's layout: blocks of 128 rows x 4 scales (128 elements of K), 512 bytes
    each, row r and scale c of a block at byte (r % 32) * 16 + (r // 32) * 4 + c; what lies outside the matrix is 0."""
    rows, cols = s.shape
    rb, cb = -(-rows // 128), -(-cols // 4)
    whole = torch.zeros(rb * 128, cb * 4, dtype=torch.uint8, device=s.device)
    whole[:rows, :cols] = s
    return whole.view(rb, 4, 32, cb, 4).permute(0, 3, 2, 1, 4).reshape(rb, cb, 512).contiguous()


def untile_scales(t, rows, cols):
    rb, cb, _ = t.shape
    return t.view(rb, cb, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rb * 128, cb * 4)[:rows, :cols]


def encode(x):
    """(codes [rows, K] of 4 bits, scale bytes [rows, K / 32]) of a finite x: the scale is 2 to the exponent of the
    block's largest magnitude, less 2; elements are rounded to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6, ties to even
    codes, and what lies above 6 becomes 6."""
    b = x.float().view(x.shape[0], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    _, e = torch.frexp(top)  # top = m 2^e, 0.5 <= m < 1
    e = torch.where(top > 0, (e - 3).clamp(min=-127), torch.full_like(e, -127))
    v = torch.ldexp(b, -e)
    a = v.abs()
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int()
            + (a >= 3.5).int() + (a > 5.0).int())
    code = code + 8 * (v < 0).int()
    return code.view(x.shape).to(torch.uint8), (e.squeeze(-1) + 127).to(torch.uint8)


def decode(code, scale):
    """The values of codes and scale bytes, in 32 bits (every product here is exact)."""
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=code.device)
    v = table[code.int()].view(code.shape[0], -1, 32)
    return torch.ldexp(v, scale.int().unsqueeze(-1) - 127).view(code.shape)


def pack(code):
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous()


def unpack(q):
    return torch.stack((q & 15, q >> 4), -1).view(q.shape[0], -1)


# ----------------------------------------------------------------------------------------------------------- the inputs
def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t, op, m, k = TYPES[case["type"]], case["op"], case["m"], case["k"]
    s = dict(case)
    if op in ("gated", "gated_backward"):
        f = case["f"]
        s["a"] = _normal(g, (m, k), t)
        s["b_gate"], s["b_up"] = _normal(g, (f, k), t, k ** -0.5), _normal(g, (f, k), t, k ** -0.5)
        if op == "gated_backward":  # what the forward pass kept, and the gradient that arrives
            s["gate"], s["up"] = torch.matmul(s["a"], s["b_gate"].t()), torch.matmul(s["a"], s["b_up"].t())
            s["dc"] = _normal(g, (m, f), t)
    elif op == "backward":
        n = case["n"]
        s["a"], s["b"], s["dc"] = _normal(g, (m, k), t), _normal(g, (n, k), t, k ** -0.5), _normal(g, (m, n), t)
    else:
        # activations: channels of unlike sizes, as they come out of a norm with learned gains
        s["x"] = (_normal(g, (m, k), torch.float32) * torch.exp(0.5 * _normal(g, (k,), torch.float32))).to(t)
        if op == "mx_linear":  # the weights are laid out in 4 bits once, when a model is loaded
            code, scale = encode(_normal(g, (case["n"], k), t, k ** -0.5))
            s["w"], s["w_scales"] = pack(code), tile_scales(scale)
    return s


# ------------------------------------------------------------------------------------------------------- one pass each
def run(state):
    return {"gated": _gated, "gated_backward": _gated_backward, "backward": _backward, "quantize": _quantize,
            "mx_linear": _mx_linear}[state["op"]](state)


def _act(name, g):
    """(act(g), its derivative)"""
    if name == "silu":
        p = 1 / (1 + torch.exp(-g))
        return g * p, p * (1 + g * (1 - p))
    if name == "gelu":
        p = 0.5 * torch.erfc(g * -math.sqrt(0.5))
        return g * p, p + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        p = 1 / (1 + torch.exp(-2 * c * (g + 0.044715 * g * g * g)))
        return g * p, p + 2 * c * g * p * (1 - p) * (1 + 3 * 0.044715 * g * g)
    return torch.where(g > 0, g, 0 * g), (g > 0).to(g.dtype)


def _gated(s):
    a, m, f = s["a"], s["m"], s["f"]
    if own:
        import beam
        c = torch.empty(m, f, dtype=a.dtype, device=a.device)
        if not s["keep"]:
            beam.gated_gemmrc(a, s["b_gate"], s["b_up"], c, activation=s["act"])
            return {"c": c}
        gate, up = torch.empty_like(c), torch.empty_like(c)
        beam.gated_gemmrc(a, s["b_gate"], s["b_up"], c, activation=s["act"], gate=gate, up=up)
        return {"c": c, "gate": gate, "up": up}
    x = a.float()
    gate, up = torch.matmul(x, s["b_gate"].float().t()), torch.matmul(x, s["b_up"].float().t())
    c = (_act(s["act"], gate)[0] * up).to(a.dtype)
    return {"c": c, "gate": gate.to(a.dtype), "up": up.to(a.dtype)} if s["keep"] else {"c": c}


def _gated_backward(s):
    a = s["a"]
    if own:
        import beam
        da, dg, du = torch.empty_like(a), torch.empty_like(s["b_gate"]), torch.empty_like(s["b_up"])
        beam.gated_gemmrc_backward(s["dc"], a, s["b_gate"], s["b_up"], s["gate"], s["up"], da=da, db_gate=dg, db_up=du,
                                   activation=s["act"])
        return {"da": da, "db_gate": dg, "db_up": du}
    d, gate, up, x = s["dc"].float(), s["gate"].float(), s["up"].float(), a.float()
    act, slope = _act(s["act"], gate)
    dgate, dup = d * up * slope, d * act
    da = torch.matmul(dgate, s["b_gate"].float()) + torch.matmul(dup, s["b_up"].float())
    return {"da": da.to(a.dtype), "db_gate": torch.matmul(dgate.t(), x).to(a.dtype),
            "db_up": torch.matmul(dup.t(), x).to(a.dtype)}


def _backward(s):
    a, b = s["a"], s["b"]
    if own:
        import beam
        da, db = torch.empty_like(a), torch.empty_like(b)
        beam.gemmrc_backward(s["dc"], a, b, da=da, db=db)
        return {"da": da, "db": db}
    d = s["dc"].float()
    return {"da": torch.matmul(d, b.float()).to(a.dtype), "db": torch.matmul(d.t(), a.float()).to(b.dtype)}


def _quantize(s):
    x = s["x"]
    if own:
        import beam
        q, scales = beam.mxfp4_empty(s["m"], s["k"], x.device)
        beam.mxfp4_quantize(x, q, scales)
        y = torch.empty_like(x)
        beam.mxfp4_dequantize(q, scales, y)
        return {"values": y}
    return {"values": decode(*encode(x)).to(x.dtype)}


def _mx_linear(s):
    x, m, n = s["x"], s["m"], s["n"]
    if own:
        import beam
        q, scales = beam.mxfp4_empty(m, s["k"], x.device)
        beam.mxfp4_quantize(x, q, scales)
        c = torch.empty(m, n, dtype=x.dtype, device=x.device)
        beam.mxfp4_gemmrc(q, scales, s["w"], s["w_scales"], c)
        return {"c": c}
    w = decode(unpack(s["w"]), untile_scales(s["w_scales"], n, s["k"] // 32))
    return {"c": torch.matmul(decode(*encode(x)), w.t()).to(x.dtype)}


# -------------------------------------------------------------------------------- the definitions, in 64 bits throughout
def _mx_round(x):
    """The values that a finite x has after quantisation, by the spacing of the 4-bit numbers in each binade."""
    b = x.double().reshape(-1, 32)
    top = b.abs().max(1, keepdim=True).values
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -140)))
    e = torch.where(torch.exp2(e) > top.clamp(min=2.0 ** -140), e - 1, e)  # a logarithm rounded up at a border
    e = torch.where(torch.exp2(e + 1) <= top, e + 1, e)
    unit = torch.exp2((e - 2).clamp(min=-127.0))
    v = b / unit
    step = 0.5 * torch.exp2((v.abs() >= 2).double() + (v.abs() >= 4).double())
    return ((torch.round(v / step) * step).clamp(-6, 6) * unit).reshape(x.shape)


def _slope(name, g):
    """(act(g), act'(g)), from the definitions."""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    if name == "gelu":
        s = torch.special.ndtr(g)
        return g * s, s + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        h = torch.tanh(c * (g + 0.044715 * g ** 3))
        return 0.5 * g * (1 + h), 0.5 * (1 + h) + 0.5 * g * (1 - h * h) * c * (1 + 3 * 0.044715 * g * g)
    return g.clamp(min=0), torch.sign(g).clamp(min=0)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return {"values": _mx_round(s["x"])}
    if op == "mx_linear":
        n, k = case["n"], case["k"]
        low, high = (s["w"] & 15).long(), (s["w"] >> 4).long()
        v = torch.empty(n, k, dtype=torch.float64, device="cuda")
        for part, c in ((0, low), (1, high)):
            e, h = (c >> 1) & 3, (c & 1).double()
            size = torch.where(e == 0, 0.5 * h, torch.exp2(e.double() - 1) * (1 + 0.5 * h))
            v[:, part::2] = torch.where(c >= 8, -size, size)
        r, c = torch.arange(n, device="cuda")[:, None], torch.arange(k // 32, device="cuda")[None]
        flat = ((r // 128) * s["w_scales"].shape[1] + c // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + c % 4
        unit = torch.exp2(s["w_scales"].reshape(-1)[flat].double() - 127)
        return {"c": _mx_round(s["x"]) @ (v.view(n, -1, 32) * unit[..., None]).view(n, k).t()}
    a = s["a"].double()
    if op == "gated":
        gate, up = a @ s["b_gate"].double().t(), a @ s["b_up"].double().t()
        c = _slope(case["act"], gate)[0] * up
        return {"c": c, "gate": gate, "up": up} if case["keep"] else {"c": c}
    d = s["dc"].double()
    if op == "backward":
        return {"da": d @ s["b"].double(), "db": d.t() @ a}
    act, slope = _slope(case["act"], s["gate"].double())
    dgate, dup = d * s["up"].double() * slope, d * act
    return {"da": dgate @ s["b_gate"].double() + dup @ s["b_up"].double(), "db_gate": dgate.t() @ a, "db_up": dup.t() @ a}
