"""Microscaled formats (OCP Microscaling 1.0): quantised tensors, their products, and layers that compute with them.

A block of 32 consecutive values along the last dimension shares a scale 2^e, e = clamp(floor(log2(largest magnitude)) - E,
-127, 127), held as ``e + 127`` in a byte; its values are ``v / 2^e`` rounded to nearest even, and saturate:

    "mxfp8"   E4M3 codes, a byte each; E = 8, largest number 448
    "mxfp4"   E2M1 codes, two to a byte, the first in the lower half; E = 2, largest number 6

A block of zeros has e = -127.  A block that holds an infinity or a NaN gets scale code 255: all of its values are NaN, and so is
every product with them.  Sums of products are kept in fp32 by the tensor core, which truncates each sum at the accumulator's last bit.

CUDA tensors run on ``csrc/mx_quant.cu`` and ``csrc/mx_gemm.cu`` (tcgen05 with block scales), CPU tensors on the same formulas
with tensor operations.  ``QuantizeMX``, ``AddRMSNormMX``, ``MatMulMX`` and ``LinearMX`` serve evaluation, like the int8 layers of
this package; ``TrainLinearMX`` is differentiable.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch

from .. import lib as _l
from ..nn.linear import Linear
from ..nn.module import Module
from ..nn.norm import RMSNorm
from ..ops.gemm import ACT, _act_ref

MXBlock = 32
_FMT = {"mxfp8": 0, "mxfp4": 1}
_TYPES = (torch.bfloat16, torch.float16, torch.float32)


@dataclass
class QTensorMX:
    """Codes and scales of a tensor of ``Shape``, quantised along its last dimension.

    ``Data``: uint8 (rows, row bytes): rows of codes, padded with zeros to whole blocks.  ``Scales``: uint8, in pieces of 512 bytes for
    128 rows by four blocks, the order in which the tensor core takes them: the pieces of 128 rows behind one another, row
    r of a piece at byte 16 (r % 32) + 4 (r // 32).  MXFP4 has an even number of pieces in a row of pieces.  Scales behind the
    last block of a row are zeros; those of rows behind the last one are never read into a result."""
    Data: torch.Tensor
    Scales: torch.Tensor
    Format: str
    Shape: tuple

    def Numel(self) -> int:
        n = 1
        for s in self.Shape:
            n *= s
        return n

    def ScaleCodes(self) -> torch.Tensor:
        """The scale codes as (rows, blocks)."""
        rows, blocks = self.Data.shape[0], -(-self.Shape[-1] // MXBlock)
        if rows == 0:
            return self.Scales.new_empty((0, blocks))
        s = self.Scales.view(-(-rows // 128), -1, 32, 4, 4).permute(0, 3, 2, 1, 4)
        return s.reshape(s.shape[0] * 128, -1)[:rows, :blocks]


def _format(format: str) -> int:
    try:
        return _FMT[format]
    except KeyError:
        raise ValueError(f"quant: microscaled formats are 'mxfp8' and 'mxfp4', not {format!r}") from None


def _row_bytes(K: int, fmt: int) -> int:
    return -(-K // MXBlock) * (32 >> fmt)


def _pieces(K: int, fmt: int) -> int:
    return -(-K // 128) if fmt == 0 else 2 * -(-K // 256)


def _empty(rows: int, shape: tuple, fmt: int, device) -> QTensorMX:
    K = shape[-1]
    data = torch.empty((rows, _row_bytes(K, fmt)), dtype=torch.uint8, device=device)
    scales = torch.empty(-(-rows // 128) * _pieces(K, fmt) * 512, dtype=torch.uint8, device=device)
    return QTensorMX(data, scales, "mxfp4" if fmt else "mxfp8", shape)


def _rows(t: torch.Tensor, what: str) -> torch.Tensor:
    """``t`` as a matrix of its last dimension: a view where its rows lie evenly spaced and its elements side by side."""
    if t.dim() == 0 or t.shape[-1] == 0:
        raise ValueError(f"{what}: a last dimension of at least one value is needed, got shape {tuple(t.shape)}")
    if not t.is_floating_point():
        raise TypeError(f"{what}: a floating point tensor is needed, got {t.dtype}")
    if t.is_cuda and t.dtype not in _TYPES:
        raise TypeError(f"{what}: no CUDA kernel for dtype {t.dtype}")
    t = t.detach()
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 and (t.stride(0) >= t.shape[1] or t.shape[0] <= 1) or t.shape[1] == 1 and t.stride(0) >= 1 else t.contiguous()


def _call(device, name: str, *args) -> None:
    """A native call on ``device``'s current stream, whichever device is the current one."""
    if device.index is None or device.index == torch.cuda.current_device():
        _l.call(name, *args, _l.stream_ptr())
    else:
        with torch.cuda.device(device):
            _l.call(name, *args, _l.stream_ptr())


# ---------------------------------------------------------------------------------------
# the oracle: the same on CPU tensors
# ---------------------------------------------------------------------------------------
def _numbers(fmt: int) -> torch.Tensor:
    """The number that each code stands for (NaN for E4M3's code 127)."""
    mant, bias, codes = (3, 7, 128) if fmt == 0 else (1, 1, 8)
    c = torch.arange(codes, dtype=torch.float64)
    e, f = torch.floor(c / 2 ** mant), torch.remainder(c, 2 ** mant) / 2 ** mant
    v = torch.where(e == 0, f * 2.0 ** (1 - bias), (1 + f) * torch.pow(2.0, e - bias))
    if fmt == 0:
        v[127] = float("nan")
    return torch.cat((v, -v))


def _pack_scales(codes: torch.Tensor, fmt: int) -> torch.Tensor:
    rows, blocks = codes.shape
    per = 8 if fmt else 4
    s = torch.zeros((-(-rows // 128) * 128, -(-blocks // per) * per), dtype=torch.uint8)
    s[:rows, :blocks] = codes
    return s.view(-1, 4, 32, s.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).reshape(-1)


def _quantize_ref(t: torch.Tensor, fmt: int, shape: tuple) -> QTensorMX:
    rows, K = t.shape
    blocks, top, largest = -(-K // MXBlock), (2 if fmt else 8), (6.0 if fmt else 448.0)
    v = torch.zeros((rows, blocks * MXBlock), dtype=torch.float64)
    v[:, :K] = t.double()
    v = v.view(rows, blocks, MXBlock)
    big = v.abs().amax(2)
    odd = ~torch.isfinite(v).all(2)
    e = (torch.frexp(big).exponent - 1 - top).clamp(-127, 127)
    e = torch.where((big == 0) | odd, torch.full_like(e, -127), e)
    v = torch.ldexp(v, -e[..., None].double())
    numbers = _numbers(fmt)[: 8 if fmt else 127]
    m = v.abs().clamp(max=largest)
    mid = (numbers[1:] + numbers[:-1]) / 2
    low, high = torch.bucketize(m, mid), torch.bucketize(m, mid, right=True)
    code = torch.where(low % 2 == 0, low, high) + torch.signbit(v) * (8 if fmt else 128)
    code = torch.where(odd[..., None], torch.where(torch.isnan(v) | torch.isinf(v), 7 if fmt else 127, 0), code)
    code = code.flatten(1).to(torch.uint8)
    data = (code[:, 0::2] | code[:, 1::2] << 4) if fmt else code
    return QTensorMX(data.contiguous(), _pack_scales(torch.where(odd, 255, e + 127).to(torch.uint8), fmt), "mxfp4" if fmt else "mxfp8", shape)


def _values_ref(q: QTensorMX) -> torch.Tensor:
    """(rows, K) in fp64."""
    fmt, K = _FMT[q.Format], q.Shape[-1]
    code = torch.stack((q.Data & 15, q.Data >> 4), -1).flatten(1) if fmt else q.Data
    v = _numbers(fmt)[code.long()].view(code.shape[0], code.shape[1] // MXBlock, MXBlock)
    s = q.ScaleCodes()
    e = torch.where(s == 255, torch.full(s.shape, float("nan"), dtype=torch.float64), torch.pow(2.0, s.double() - 127))
    return (v * e[..., None]).flatten(1)[:, :K]


# ---------------------------------------------------------------------------------------
# operators
# ---------------------------------------------------------------------------------------
def QuantizeMX(t: torch.Tensor, format: str = "mxfp8") -> QTensorMX:
    """Codes and scales of ``t`` (bf16, fp16 or fp32 on CUDA) along its last dimension, of any length."""
    fmt, shape = _format(format), tuple(t.shape)
    x = _rows(t, "QuantizeMX")
    if not x.is_cuda:
        return _quantize_ref(x, fmt, shape)
    rows, K = x.shape
    q = _empty(rows, shape, fmt, x.device)
    if rows:
        _call(x.device, "gb_mx_quantize", _l.I(_l.dtype_code(x.dtype)), _l.I(fmt), _l.ptr(x), _l.L(x.stride(0)), _l.ptr(q.Data), _l.ptr(q.Scales),
              _l.L(rows), _l.L(K))
    return q


def QuantizeMXPair(t: torch.Tensor) -> Tuple[QTensorMX, QTensorMX]:
    """MXFP8 codes and scales of the matrix ``t`` (leading dimensions are flattened) along its rows' last dimension, and of its
    transpose along the other one, from one reading: what a layer's forward and its gradients multiply."""
    shape = tuple(t.shape)
    x = _rows(t, "QuantizeMXPair")
    rows, K = x.shape
    if rows == 0:
        raise ValueError("QuantizeMXPair: at least one row is needed")
    if not x.is_cuda:
        return _quantize_ref(x, 0, shape), _quantize_ref(x.t(), 0, (K, rows))
    q, qt = _empty(rows, shape, 0, x.device), _empty(K, (K, rows), 0, x.device)
    _call(x.device, "gb_mx_quantize_both", _l.I(_l.dtype_code(x.dtype)), _l.ptr(x), _l.L(x.stride(0)), _l.ptr(q.Data), _l.ptr(q.Scales), _l.ptr(qt.Data),
          _l.ptr(qt.Scales), _l.L(rows), _l.L(K))
    return q, qt


def _checked(q: QTensorMX, what: str) -> int:
    """The format's code, once codes and scales fit the shape."""
    fmt = _format(q.Format)
    if len(q.Shape) == 0 or q.Shape[-1] < 1:
        raise ValueError(f"{what}: a quantised tensor of shape {tuple(q.Shape)}")
    rows, K = 1, q.Shape[-1]
    for s in q.Shape[:-1]:
        rows *= s
    d, s = q.Data, q.Scales
    if d.dtype != torch.uint8 or s.dtype != torch.uint8 or d.device != s.device:
        raise TypeError(f"{what}: codes and scales are uint8 tensors of one device")
    if tuple(d.shape) != (rows, _row_bytes(K, fmt)) or s.numel() != -(-rows // 128) * _pieces(K, fmt) * 512:
        raise ValueError(f"{what}: codes {tuple(d.shape)} and {s.numel()} scales do not belong to shape {tuple(q.Shape)} in {q.Format}")
    if not (d.is_contiguous() and s.is_contiguous()):
        raise ValueError(f"{what}: codes and scales must be contiguous")
    if d.is_cuda and (d.data_ptr() | s.data_ptr()) & 15:
        raise ValueError(f"{what}: codes and scales must be 16-byte aligned")
    return fmt


def DequantizeMX(q: QTensorMX, dtype=torch.float32) -> torch.Tensor:
    """The values that ``q`` stands for, rounded to ``dtype`` (exact in fp32, but for MXFP8 values below 2^-149)."""
    fmt = _checked(q, "DequantizeMX")
    if not q.Data.is_cuda:
        return _values_ref(q).to(dtype).reshape(q.Shape)
    if dtype not in _TYPES:
        raise TypeError(f"DequantizeMX: no CUDA kernel for dtype {dtype}")
    y = torch.empty(q.Shape, dtype=dtype, device=q.Data.device)
    if y.numel():
        _call(y.device, "gb_mx_dequantize", _l.I(_l.dtype_code(dtype)), _l.I(fmt), _l.ptr(q.Data), _l.ptr(q.Scales), _l.ptr(y), _l.L(q.Data.shape[0]),
              _l.L(q.Shape[-1]))
    return y


def AddRMSNormMX(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-6,
                 format: str = "mxfp8") -> Tuple[QTensorMX, torch.Tensor]:
    """``h = x + residual`` and the quantised ``h / sqrt(mean(h^2) + eps) * weight``: what a pre-norm block hands to its next
    products, and the stream that goes on beside them.  Returns (codes and scales, h); the norm takes the sum in fp32, before it is
    rounded to h's type.  Without a residual h is x itself."""
    fmt, shape = _format(format), tuple(x.shape)
    a = _rows(x, "AddRMSNormMX")
    rows, K = a.shape
    r = None
    if residual is not None:
        if tuple(residual.shape) != shape or residual.dtype != x.dtype or residual.device != x.device:
            raise ValueError(f"AddRMSNormMX: the residual must be like x ({shape}, {x.dtype}, {x.device})")
        r = _rows(residual, "AddRMSNormMX")
    if tuple(weight.shape) != (K,) or weight.device != x.device:
        raise ValueError(f"AddRMSNormMX: weight must have shape ({K},) on {x.device}")
    if weight.dtype not in (x.dtype, torch.float32):
        raise TypeError("AddRMSNormMX: weight dtype must equal the input dtype or be float32")
    if not x.is_cuda:
        ct = torch.float64 if x.dtype == torch.float64 else torch.float32
        h = a.to(ct) if r is None else a.to(ct) + r.to(ct)
        y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps) * weight.detach().to(ct)
        return _quantize_ref(y, fmt, shape), (x if r is None else h.to(x.dtype).reshape(shape))
    w = weight.detach().contiguous()
    q = _empty(rows, shape, fmt, x.device)
    h = None if r is None else torch.empty(shape, dtype=x.dtype, device=x.device)
    if rows:
        _call(x.device, "gb_mx_add_rms_norm", _l.I(_l.dtype_code(x.dtype)), _l.I(fmt), _l.ptr(a), _l.L(a.stride(0)), _l.ptr(r),
              _l.L(K if r is None else r.stride(0)), _l.ptr(w), _l.I(int(w.dtype == torch.float32)), _l.ptr(h), _l.ptr(q.Data), _l.ptr(q.Scales),
              _l.L(rows), _l.L(K), _l.F(eps))
    return q, (x if h is None else h)


def MatMulMX(a: QTensorMX, b: QTensorMX, bias: Optional[torch.Tensor] = None, dtype=torch.bfloat16, act: Optional[str] = None) -> torch.Tensor:
    """``act(A B^T + bias)`` in ``dtype`` (bf16, fp16 or fp32) for A (..., K) and B (N, K), both quantised along K in one format.
    ``act``: relu, gelu or geluexact, as ``nn.Linear`` takes it."""
    fmt = _checked(a, "MatMulMX")
    if _checked(b, "MatMulMX") != fmt:
        raise ValueError(f"MatMulMX: both operands have one format, got {a.Format} and {b.Format}")
    if len(b.Shape) != 2 or a.Shape[-1] != b.Shape[-1]:
        raise ValueError(f"MatMulMX: shapes {tuple(a.Shape)} and {tuple(b.Shape)} do not match (..., K) and (N, K)")
    if a.Data.device != b.Data.device:
        raise ValueError(f"MatMulMX: operands on {a.Data.device} and {b.Data.device}")
    if act not in ACT:
        raise ValueError(f"MatMulMX: unknown activation {act!r}")
    N, K = b.Shape
    M, dev = a.Data.shape[0], a.Data.device
    if bias is not None:
        if tuple(bias.shape) != (N,) or bias.device != dev:
            raise ValueError(f"MatMulMX: bias must have shape ({N},) on {dev}")
        bias = bias.detach()
    shape = (*a.Shape[:-1], N)
    if not a.Data.is_cuda:
        y = _values_ref(a) @ _values_ref(b).t()
        if bias is not None:
            y = y + bias.double()
        return _act_ref(y, act).to(dtype).reshape(shape)
    if dtype not in _TYPES:
        raise TypeError(f"MatMulMX: no CUDA kernel for dtype {dtype}")
    if bias is not None:
        bias = (bias if bias.dtype in (dtype, torch.float32) else bias.float()).contiguous()
    y = torch.empty(shape, dtype=dtype, device=dev)
    if y.numel() == 0:
        return y
    need = _workspace(M, N, K, fmt)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _call(dev, "gb_mx_matmul", _l.I(fmt), _l.ptr(a.Data), _l.ptr(a.Scales), _l.ptr(b.Data), _l.ptr(b.Scales), _l.ptr(y), _l.L(N), _l.ptr(bias),
          _l.I(int(bias is not None and bias.dtype == torch.float32)), _l.L(M), _l.L(N), _l.L(K), _l.I(_l.dtype_code(dtype)), _l.I(ACT[act]), _l.ptr(ws),
          _l.L(need))
    return y


def _workspace(M: int, N: int, K: int, fmt: int) -> int:
    out = (_l.L * 4)()
    _l.check(_l.lib().gb_mx_plan(_l.L(M), _l.L(N), _l.L(K), _l.I(fmt), out), "gb_mx_plan")
    return out[3]


def LinearMX(x: Union[torch.Tensor, QTensorMX], weight: QTensorMX, bias: Optional[torch.Tensor] = None, act: Optional[str] = None,
             dtype=None) -> torch.Tensor:
    """``act(Q(x) W^T + bias)`` with quantised weights (out, in).  ``x``: a tensor, quantised here in the weights' format, or what
    ``AddRMSNormMX`` returned.  ``dtype``: of the result; x's own, or bf16 for a quantised x.  Evaluation only, no gradients."""
    if isinstance(x, QTensorMX):
        return MatMulMX(x, weight, bias, dtype or torch.bfloat16, act)
    return MatMulMX(QuantizeMX(x, weight.Format), weight, bias, dtype or x.dtype, act)


class _TrainLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        N, K = weight.shape
        ctx.xshape, ctx.params, ctx.xdtype = x.shape, (weight, bias), x.dtype
        ctx.saved = ()
        if x.numel() == 0:
            ctx.empty = True
            return x.new_empty((*x.shape[:-1], N))
        ctx.empty = False
        xq, xt = QuantizeMXPair(x) if need_w else (QuantizeMX(x), None)
        wq, wt = QuantizeMXPair(weight) if need_x else (QuantizeMX(weight), None)
        ctx.save_for_backward(*(t for q in (xt, wt) if q is not None for t in (q.Data, q.Scales)))
        ctx.kept = (xt is not None, wt is not None)
        return MatMulMX(xq, wq, bias, x.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        from ..ops.linear import emit_grad, emit_vector_grad
        weight, bias = ctx.params
        N, K = weight.shape
        dx = dw = db = None
        if ctx.empty:
            z = torch.zeros
            dx = z(ctx.xshape, dtype=ctx.xdtype, device=dy.device) if ctx.needs_input_grad[0] else None
            dw = emit_grad(weight, torch.zeros_like(weight)) if ctx.needs_input_grad[1] else None
            db = emit_grad(bias, torch.zeros_like(bias)) if bias is not None and ctx.needs_input_grad[2] else None
            return dx, dw, db
        saved = list(ctx.saved_tensors)
        rows = dy.numel() // N
        xt = QTensorMX(saved.pop(0), saved.pop(0), "mxfp8", (K, rows)) if ctx.kept[0] else None
        wt = QTensorMX(saved.pop(0), saved.pop(0), "mxfp8", (K, N)) if ctx.kept[1] else None
        g = _rows(dy, "TrainLinearMX")
        gq, gt = QuantizeMXPair(g) if xt is not None else (QuantizeMX(g) if wt is not None else None, None)
        if wt is not None:
            dx = MatMulMX(gq, wt, None, ctx.xdtype).reshape(ctx.xshape)
        if xt is not None:
            dw = emit_grad(weight, MatMulMX(gt, xt, None, weight.dtype))
        if bias is not None and ctx.needs_input_grad[2]:
            db = emit_vector_grad(bias, g)
        return dx, dw, db


def TrainLinearMX(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``Q(x) Q(W)^T + b`` in MXFP8 with gradients that go straight through the rounding; every product's operands are quantised
    along its contraction: dx = Q(dy) Q(W^T)^T, dW = Q(dy^T) Q(x^T)^T, db = column sums of dy.  For the backward pass the layer
    keeps the codes of x^T and W^T, a byte a value."""
    if weight.dim() != 2 or x.dim() == 0 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"TrainLinearMX: shapes {tuple(x.shape)} and {tuple(weight.shape)} do not match (..., K) and (N, K)")
    if weight.device != x.device:
        raise ValueError(f"TrainLinearMX: x on {x.device}, weight on {weight.device}")
    return _TrainLinear.apply(x, weight, bias)


# ---------------------------------------------------------------------------------------
# layers
# ---------------------------------------------------------------------------------------
class MXLinear(Module):
    """A ``Linear`` whose weights are quantised once; its rows are quantised per call, or come quantised from ``MXRMSNorm``.
    Bias and activation run in the product's epilogue.  Inference only."""

    def __init__(self, linear: Linear, format: str = "mxfp8"):
        super().__init__()
        q = QuantizeMX(linear.weight, format)
        self.format, self.activation = format, linear.activation
        self.in_features, self.out_features = linear.in_features, linear.out_features
        self.register_buffer("codes", q.Data)
        self.register_buffer("scales", q.Scales)
        self.register_buffer("bias", None if linear.bias is None else linear.bias.detach().clone())

    def Weight(self) -> QTensorMX:
        return QTensorMX(self.codes, self.scales, self.format, (self.out_features, self.in_features))

    @torch.no_grad()
    def forward(self, x, dtype=None):
        return LinearMX(x, self.Weight(), self.bias, self.activation, dtype)


class MXRMSNorm(Module):
    """``RMSNorm`` with a quantised result: ``(codes and scales, h)`` of ``h = x + residual``.  Inference only."""

    def __init__(self, norm: RMSNorm, format: str = "mxfp8"):
        super().__init__()
        _format(format)
        self.format, self.eps = format, norm.eps
        self.register_buffer("weight", norm.weight.detach().clone())

    @torch.no_grad()
    def forward(self, x, residual=None):
        return AddRMSNormMX(x, residual, self.weight, self.eps, self.format)


class MXTrainLinear(Module):
    """A ``Linear`` that trains in MXFP8 (``TrainLinearMX``); child ``linear`` holds the parameters.  ``Convert()`` produces the
    ``MXLinear`` that evaluates with the weights as they are then."""

    def __init__(self, linear: Linear):
        super().__init__()
        if linear.activation not in (None, "none"):
            raise ValueError("MXTrainLinear: a Linear without a fused activation is needed")
        self.linear = linear

    def forward(self, x):
        return TrainLinearMX(x, self.linear.weight, self.linear.bias)

    def Convert(self, format: str = "mxfp8") -> MXLinear:
        return MXLinear(self.linear, format)


def NewMXLinearFrom(l: Linear, format: str = "mxfp8") -> MXLinear:
    return MXLinear(l, format)


def NewMXTrainLinearFrom(l: Linear) -> MXTrainLinear:
    return MXTrainLinear(l)
