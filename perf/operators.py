"""Microscaled formats (blocks of 32 values that share a power of two): what is measured of them.

Three operators and the two paths that a user's program takes through them:

  quant   ``quant.QuantizeMX`` and ``quant.DequantizeMX``: a tensor into codes and scales, and the values they stand for
  norm    ``quant.AddRMSNormMX``: the residual's addition, the root-mean-square norm and the quantised rows; the sum goes on
  matmul  ``quant.MatMulMX``: the product of two quantised matrices
  linear  ``quant.LinearMX``: a layer with quantised weights on 16-bit rows (the rows are quantised within the call)
  train   ``quant.TrainLinearMX``: such a layer forward and backward, gradients of input, weight and bias

Formats (OCP Microscaling 1.0): a block's scale is 2^e, e = floor(log2(largest magnitude)) - E, held as e + 127 in 8 bits; its
values are rounded to nearest even and saturate.  mxfp8: E4M3 (E = 8, largest 448); mxfp4: E2M1 (E = 2, largest 6), two to a
byte, the first in the lower half.  Scales lie in pieces of 128 rows by 4 blocks: row r of a piece at 16 (r % 32) + 4 (r // 32).
"""
import math

import torch

own = False

BLOCK = 32
#: mantissa bits, least exponent, exponent of the largest number, the largest number
FORMATS = {"mxfp8": (3, -6, 8, 448.0), "mxfp4": (1, 0, 2, 6.0)}
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # the norm before a block's products while one sequence is generated, token by token (1.3 B model, width 2048)
        {"name": "norm, one token", "op": "norm", "format": "mxfp8", "dtype": "bf16", "rows": 1, "width": 2048},
        # a training-sized batch through the norm of the 12-layer model
        {"name": "norm, 16 x 1024 tokens", "op": "norm", "format": "mxfp8", "dtype": "bf16", "rows": 16384, "width": 768},
        # fp32 rows of a width that no vector or block divides
        {"name": "norm, ragged fp32", "op": "norm", "format": "mxfp4", "dtype": "f32", "rows": 5003, "width": 1003},
        # the vocabulary head's weights once, after loading
        {"name": "quant, vocabulary head", "op": "quant", "format": "mxfp4", "dtype": "bf16", "rows": 50304, "width": 2048},
        # the rows of a small odd batch
        {"name": "quant, ragged fp16", "op": "quant", "format": "mxfp8", "dtype": "f16", "rows": 1001, "width": 1000},
        # four sequences generated together through a feed-forward layer: the weights' bytes are what counts
        {"name": "matmul, 4 tokens", "op": "matmul", "format": "mxfp4", "dtype": "bf16", "rows": 4, "width": 2048, "features": 8192, "bias": True},
        # the square product of the kernel benchmark
        {"name": "matmul, 8192 cubed", "op": "matmul", "format": "mxfp8", "dtype": "bf16", "rows": 8192, "width": 8192, "features": 8192, "bias": False},
        # a long prompt batch through a feed-forward layer of the 1.3 B model
        {"name": "matmul, 16384 tokens fp4", "op": "matmul", "format": "mxfp4", "dtype": "bf16", "rows": 16384, "width": 2048, "features": 8192, "bias": True},
        # one token through the second feed-forward layer
        {"name": "linear, one token", "op": "linear", "format": "mxfp4", "dtype": "bf16", "rows": 1, "width": 8192, "features": 2048, "act": "none"},
        # a short prompt through the joint projection of the 12-layer model
        {"name": "linear, 77 tokens", "op": "linear", "format": "mxfp8", "dtype": "bf16", "rows": 77, "width": 768, "features": 2304, "act": "gelu"},
        # the joint projection in training: 16 sequences of 1024 tokens
        {"name": "train, 16 x 1024 tokens", "op": "train", "format": "mxfp8", "dtype": "bf16", "rows": 16384, "width": 768, "features": 2304},
        # a last, smaller batch through a layer of odd sizes
        {"name": "train, ragged fp16", "op": "train", "format": "mxfp8", "dtype": "f16", "rows": 1001, "width": 1000, "features": 520},
    ]


def draw(rng):
    def size(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    op = rng.choice(["norm", "quant", "matmul", "linear", "train"])
    case = {"op": op, "format": rng.choice(["mxfp8", "mxfp4"]), "dtype": rng.choice(["bf16", "f16"])}
    if op in ("norm", "quant"):
        case["dtype"] = rng.choice(["bf16", "f16", "f32"])
        case["width"] = size(32, 8192)
        case["rows"] = size(1, min(65536, 2 ** 26 // case["width"]))
        return case
    case["width"], case["features"] = size(32, 8192), size(16, 8192)
    case["rows"] = size(1, min(16384, 2 ** 37 // (case["width"] * case["features"])))
    if op == "matmul":
        case["bias"] = rng.random() < 0.5
    elif op == "linear":
        case["act"] = rng.choice(["none", "gelu", "relu"])
    else:
        case["format"] = "mxfp8"
    return case


def work(case):
    rows, width, size = case["rows"], case["width"], TYPES[case["dtype"]].itemsize
    per = (1.0 if case["format"] == "mxfp8" else 0.5) + 1.0 / BLOCK     # bytes of a quantised value and its part of the scale
    n = rows * width
    if case["op"] == "quant":       # read, packed; packed values read, values
        return {"bytes": n * (size + 2 * per + 2), "flops": 4 * n}
    if case["op"] == "norm":        # two tensors and the weight read, the sum and packed values written; packed values read, values
        return {"bytes": n * (3 * size + 2 * per + 2) + width * size, "flops": 8 * n}
    f = case["features"]
    if case["op"] == "matmul":
        return {"bytes": (n + f * width) * per + rows * f * size + (f * size if case["bias"] else 0), "flops": 2 * n * f}
    if case["op"] == "linear":
        return {"bytes": n * size + f * width * per + (rows * f + f) * size, "flops": 2 * n * f}
    # x, w, b and dy read; y, dx, dw and db written; three products
    return {"bytes": 2 * (n + f * width + f + rows * f) * size, "flops": 6 * n * f}


# ---------------------------------------------------------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------------------------------------------------------
def _two(e):
    """2^e in 64 bits, exactly (powers by a library's function are off by a last bit, which decides ties)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _blocks(x, format):
    """(values / scale rounded to the format, exponents of the scales): (rows, blocks, 32) and (rows, blocks), in 32 bits."""
    mant, least, top, largest = FORMATS[format]
    x = torch.nn.functional.pad(x.float(), (0, -x.shape[-1] % BLOCK)).unflatten(-1, (-1, BLOCK))
    big = x.abs().amax(-1)
    e = (torch.frexp(big).exponent - 1 - top).clamp(-127, 127)
    e = torch.where(big == 0, torch.full_like(e, -127), e)
    v = x * _two(-e.unsqueeze(-1)).float()
    step = _two((torch.frexp(v).exponent - 1).clamp(min=least) - mant).float()
    v = (torch.round(v / step) * step).clamp(-largest, largest)
    return v, e


def _rounded(x, format):
    """The values that the quantised x stands for, in 32 bits."""
    v, e = _blocks(x, format)
    return (v * _two(e.unsqueeze(-1)).float()).flatten(-2)[:, : x.shape[-1]]


def _numbers(format, device):
    """The number that each code stands for, in 32 bits."""
    mant, least, _, _ = FORMATS[format]
    bits = 8 if format == "mxfp8" else 4
    code = torch.arange(2 ** bits, device=device)
    exp, frac = (code >> mant) % 2 ** (bits - 1 - mant), (code % 2 ** mant).float() / 2 ** mant
    v = torch.where(exp == 0, frac * 2.0 ** least, (1 + frac) * 2.0 ** (exp - 1 + least).float())
    return torch.where(code >= 2 ** (bits - 1), -v, v)


def _values(data, scales, width, format):
    """The same from codes and scales as they are kept."""
    rows, blocks = data.shape[0], -(-width // BLOCK)
    code = data if format == "mxfp8" else torch.stack((data & 15, data >> 4), -1).flatten(-2)
    v = _numbers(format, data.device)[code.long()].unflatten(-1, (-1, BLOCK))
    s = scales.view(-(-rows // 128), -1, 32, 4, 4).permute(0, 3, 2, 1, 4).flatten(3).flatten(0, 2)[:rows, :blocks]
    return (v * _two(s.long().unsqueeze(-1) - 127).float()).flatten(-2)[:, :width]


def _activated(y, act):
    if act == "gelu":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return y.clamp(min=0) if act == "relu" else y


# ---------------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------------
def _packed(x, format):
    """Codes and scales as they are kept."""
    v, e = _blocks(x, format)
    v = v.flatten(-2)
    if format == "mxfp8":
        data = v.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        half = torch.searchsorted(_numbers(format, v.device)[:8].contiguous(), v.abs().contiguous()) + 8 * (v < 0)
        data = (half[:, 0::2] + 16 * half[:, 1::2]).to(torch.uint8)
    rows, blocks = e.shape
    per = 4 if format == "mxfp8" else 8                        # blocks of a 128-byte piece of a row
    e = torch.nn.functional.pad((e + 127).to(torch.uint8), (0, -blocks % per, 0, -rows % 128))
    scales = e.view(e.shape[0] // 128, 4, 32, -1, 4).permute(0, 3, 2, 1, 4).reshape(-1)
    return data.contiguous(), scales.contiguous()


def _inputs(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    rows, width, dtype = case["rows"], case["width"], TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    # activations: a few channels of a model are much larger than the others
    loud = 1 + 15 * (torch.rand(width, generator=g, device="cuda") < 0.01)
    made = {"x": (normal(rows, width) * loud).to(dtype)}
    if case["op"] == "norm":
        made |= {"residual": normal(rows, width).to(dtype), "weight": (1 + 0.2 * normal(width)).to(dtype)}
    elif case["op"] != "quant":
        f = case["features"]
        made["w"] = (normal(f, width) / math.sqrt(width)).to(dtype)
        made["bias"] = None if case.get("bias") is False else (0.1 * normal(f)).to(dtype)
        made["dy"] = normal(rows, f).to(dtype) if case["op"] == "train" else None
    return made


def prepare(case, seed):
    state = dict(case, **_inputs(case, seed), type=TYPES[case["dtype"]])
    if case["op"] in ("matmul", "linear"):
        state["w"] = _packed(state["w"], case["format"])
    if case["op"] == "matmul":
        state["x"] = _packed(state["x"], case["format"])
    return state


# ---------------------------------------------------------------------------------------------------------------------------
# a pass
# ---------------------------------------------------------------------------------------------------------------------------
def _plain(s):
    op, format, x, dtype = s["op"], s["format"], s["x"], s["type"]
    if op == "quant":
        return _rounded(x, format).to(torch.bfloat16)
    if op == "norm":
        h = x.float() + s["residual"].float()
        y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["weight"].float()
        return _rounded(y, format).to(torch.bfloat16), h.to(dtype)
    bias = 0.0 if s["bias"] is None else s["bias"].float()
    if op == "train":
        w, dy = s["w"], s["dy"]
        y = _rounded(x, format) @ _rounded(w, format).T + bias
        dx = _rounded(dy, format) @ _rounded(w.T, format).T
        dw = _rounded(dy.T, format) @ _rounded(x.T, format).T
        return y.to(dtype), dx.to(dtype), dw.to(dtype), dy.float().sum(0).to(dtype)
    a = _values(*x, s["width"], format) if op == "matmul" else _rounded(x, format)
    y = a @ _values(*s["w"], s["width"], format).T + bias
    return _activated(y, s.get("act")).to(dtype)


def _own(s):
    from gonn_b200 import quant

    op, format, x, dtype = s["op"], s["format"], s["x"], s["type"]
    if op == "quant":
        return quant.DequantizeMX(quant.QuantizeMX(x, format), torch.bfloat16)
    if op == "norm":
        q, h = quant.AddRMSNormMX(x, s["residual"], s["weight"], EPS, format)
        return quant.DequantizeMX(q, torch.bfloat16), h
    if op == "train":
        x, w, b = (t.detach().requires_grad_() for t in (x, s["w"], s["bias"]))
        y = quant.TrainLinearMX(x, w, b)
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), s["dy"]))
    w = quant.QTensorMX(*s["w"], format, (s["features"], s["width"]))
    if op == "matmul":
        return quant.MatMulMX(quant.QTensorMX(*x, format, (s["rows"], s["width"])), w, s["bias"], dtype)
    return quant.LinearMX(x, w, s["bias"], s["act"])


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------------
def _nearest(x, format):
    """The values that x (in 64 bits) stands for once it is quantised: the nearest number of a list, ties to the even code."""
    bits, frac, E, bias = (8, 8, 8, 7) if format == "mxfp8" else (4, 2, 2, 1)
    numbers = [(c % frac / frac) * 2.0 ** (1 - bias) if c < frac else (1 + c % frac / frac) * 2.0 ** (c // frac - bias) for c in range(2 ** (bits - 1))]
    numbers = torch.tensor(numbers[: 127 if bits == 8 else 8], dtype=torch.float64, device=x.device)
    between = (numbers[1:] + numbers[:-1]) / 2
    rows, width = x.shape
    padded = torch.zeros(rows, (width + 31) // 32 * 32, dtype=torch.float64, device=x.device)
    padded[:, :width] = x
    v = padded.view(rows, -1, 32)
    big = v.abs().max(-1, keepdim=True).values
    powers = torch.tensor([2.0 ** k for k in range(-149, 129)], dtype=torch.float64, device=x.device)
    e = (torch.searchsorted(powers, big, right=True) - 1 - 149 - E).clamp(-127, 127)       # 0: below all of them
    scale = powers[e + 149]
    m = v.abs() / scale
    low, high = torch.bucketize(m, between), torch.bucketize(m, between, right=True)      # differ on a tie: one of the two is even
    code = torch.where(low % 2 == 0, low, high)
    return (torch.sign(v) * numbers[code] * scale).view(rows, -1)[:, :width]


def exact(case, seed):
    made = {k: None if v is None else v.double() for k, v in _inputs(case, seed).items()}
    x, format, op = made["x"], case["format"], case["op"]
    if op == "quant":
        return _nearest(x, format)
    if op == "norm":
        h = x + made["residual"]
        return _nearest(h / torch.sqrt((h ** 2).sum(1, keepdim=True) / h.shape[1] + EPS) * made["weight"], format), h
    w, dy = made["w"], made["dy"]
    y = torch.mm(_nearest(x, format), _nearest(w, format).t())
    if made["bias"] is not None:
        y += made["bias"]
    if op == "train":
        return (y, torch.mm(_nearest(dy, format), _nearest(w.t(), format).t()),
                torch.mm(_nearest(dy.t(), format), _nearest(x.t(), format).t()), torch.ones_like(dy[:, 0]) @ dy)
    if case.get("act") == "gelu":
        return y / 2 * (1 + torch.tanh((y + 0.044715 * y ** 3) * (2 / math.pi) ** 0.5))
    return torch.relu(y) if case.get("act") == "relu" else y
