"""Microscaled formats (OCP Microscaling 1.0): quantised tensors, their products, and layers that compute with them.

A block of 32 consecutive values along the last dimension shares a scale 2^e, e = clamp(floor(log2(largest magnitude)) - E,
-127, 127), held as ``e + 127`` in a byte; its values are ``v / 2^e`` rounded to nearest even, and saturate:

    "mxfp8"   E4M3 codes, a byte each; E = 8, largest number 448
    "mxfp4"   E2M1 codes, two to a byte, the first in the lower half; E = 2, largest number 6

A block of zeros has e = -127.  A block that holds an infinity or a NaN gets scale code 255: all of its values are NaN, and so is
every product with them.  Sums of products are kept in fp32 by the tensor core, which truncates each sum at the accumulator's last bit.

CUDA tensors run on ``csrc/mx_quant.cu`` and ``csrc/mx_gemm.cu`` (tcgen05 with block scales), CPU tensors on the same formulas
with tensor operations.  ``QuantizeMX``, ``AddRMSNormMX``, ``MatMulMX`` and ``LinearMX`` serve evaluation, like the int8 layers of
this package; ``TrainLinearMX`` is differentiable.  The modules stand wherever a module is called; the blocks of ``models`` and ``nn.Transformer``
read the parameters of their ``Linear`` layers for fused kernels and take neither these nor the int8 layers in their place.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from .. import lib as _l
from ..nn.linear import Linear
from ..nn.module import Module
from ..nn.norm import RMSNorm
from ..ops.gemm import ACT, _act_ref
from ..ops.linear import emit_grad, emit_vector_grad
from ..ops.reduce import column_sum

MXBlock = 32
_FMT = {"mxfp8": 0, "mxfp4": 1}
_NAMES = ("mxfp8", "mxfp4")
_TYPES = {torch.bfloat16: _l.DT_BF16, torch.float16: _l.DT_F16, torch.float32: _l.DT_F32}


class QTensorMX:
    """Codes and scales of a tensor of ``Shape``, quantised along its last dimension.

    ``Data``: uint8 (rows, row bytes): rows of codes, padded with zeros to whole blocks.  ``Scales``: uint8, in pieces of 512 bytes for
    128 rows by four blocks, the order in which the tensor core takes them: the pieces of 128 rows behind one another, row
    r of a piece at byte 16 (r % 32) + 4 (r // 32).  MXFP4 has an even number of pieces in a row of pieces.  Scales behind the
    last block of a row are zeros; those of rows behind the last one are never read into a result."""

    __slots__ = ("_format", "_shape", "_data", "_scales", "_whole", "_rows")

    def __init__(self, Data: torch.Tensor, Scales: torch.Tensor, Format: str, Shape: tuple):
        self._format, self._shape = Format, tuple(Shape)
        self._data, self._scales, self._whole, self._rows = Data, Scales, None, None

    Format = property(lambda self: self._format)
    Shape = property(lambda self: self._shape)

    @classmethod
    def _of(cls, whole: torch.Tensor, rows: int, fmt: int, shape: tuple) -> "QTensorMX":
        """Codes and scales in one allocation, which the operators address as it is; ``Data`` and ``Scales`` become views of it when they are
        asked for (two allocations and their checks are 5 of the 15 us that the host takes for a product)."""
        q = cls(None, None, _NAMES[fmt], shape)
        q._whole, q._rows = whole, rows
        return q

    def _views(self):
        w, rows = self._whole, self._rows
        if w is not None:
            per = _row_bytes(self._shape[-1], _FMT[self._format])
            self._data, self._scales = w[:rows * per].view(rows, per), w[_up16(rows * per):]
            self._whole = None
        return self._data, self._scales

    Data = property(lambda self: self._views()[0])
    Scales = property(lambda self: self._views()[1])

    def __repr__(self) -> str:
        return f"QTensorMX({self.Format}, {tuple(self.Shape)})"

    def Numel(self) -> int:
        return math.prod(self.Shape)

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


def _up16(n: int) -> int:
    return (n + 15) & ~15


def _empty(rows: int, shape: tuple, fmt: int, like: torch.Tensor):
    """(an unwritten quantised tensor, the addresses of its codes and scales)."""
    K = shape[-1]
    n = _up16(rows * _row_bytes(K, fmt))
    whole = like.new_empty(n + -(-rows // 128) * _pieces(K, fmt) * 512, dtype=torch.uint8)
    at = whole.data_ptr()
    return QTensorMX._of(whole, rows, fmt, shape), at, at + n


def _rows(t: torch.Tensor, what: str) -> torch.Tensor:
    """``t`` as a matrix of its last dimension: a view where its rows lie evenly spaced and its elements side by side."""
    shape = t.shape
    if not shape or shape[-1] == 0:
        raise ValueError(f"{what}: a last dimension of at least one value is needed, got shape {tuple(shape)}")
    if t.is_cuda:
        if t.dtype not in _TYPES:
            raise TypeError(f"{what}: no CUDA kernel for dtype {t.dtype}")
    elif not t.is_floating_point():
        raise TypeError(f"{what}: a floating point tensor is needed, got {t.dtype}")
    if len(shape) != 2:
        t = t.reshape(-1, shape[-1])
    s0, s1 = t.stride()
    if (s1 != 1 and shape[-1] > 1) or (s0 < shape[-1] and t.shape[0] > 1):
        t = t.contiguous()
    return t if t.is_cuda else t.detach()


def _call(device: int, name: str, *args) -> None:
    """A native call on the current stream of a device, whichever is the current one."""
    if device == _device():
        _l.call(name, *args, _l.current_stream_handle())
    else:
        with torch.cuda.device(device):
            _l.call(name, *args, _l.current_stream_handle())


def _device() -> int:
    return _l._raw_device() if _l._raw_device is not None else torch.cuda.current_device()


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
    q, codes, scales = _empty(rows, shape, fmt, x)
    if rows:
        _call(x.get_device(), "gb_mx_quantize", _TYPES[x.dtype], fmt, x.data_ptr(), x.stride(0), codes, scales, rows, K)
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
    (q, codes, scales), (qt, codes_t, scales_t) = _empty(rows, shape, 0, x), _empty(K, (K, rows), 0, x)
    _call(x.get_device(), "gb_mx_quantize_both", _TYPES[x.dtype], x.data_ptr(), x.stride(0), codes, scales, codes_t, scales_t, None, None, 0, rows, K)
    return q, qt


def _checked(q: QTensorMX, what: str):
    """(format's code, rows, K, a tensor of the device, address of the codes, of the scales), once codes and scales fit the shape."""
    whole = q._whole
    if whole is not None:
        fmt, rows, K = _FMT[q._format], q._rows, q._shape[-1]
        at = whole.data_ptr()
        return fmt, rows, K, whole, at, at + _up16(rows * _row_bytes(K, fmt))
    fmt, shape, d, s = _format(q._format), q._shape, q._data, q._scales
    if not shape or shape[-1] < 1:
        raise ValueError(f"{what}: a quantised tensor of shape {tuple(shape)}")
    rows, K = math.prod(shape[:-1]), shape[-1]
    if d.dtype != torch.uint8 or s.dtype != torch.uint8 or d.get_device() != s.get_device():
        raise TypeError(f"{what}: codes and scales are uint8 tensors of one device")
    if d.shape != (rows, _row_bytes(K, fmt)) or s.numel() != -(-rows // 128) * _pieces(K, fmt) * 512:
        raise ValueError(f"{what}: codes {tuple(d.shape)} and {s.numel()} scales do not belong to shape {tuple(shape)} in {q.Format}")
    if not (d.is_contiguous() and s.is_contiguous()):
        raise ValueError(f"{what}: codes and scales must be contiguous")
    codes, scales = d.data_ptr(), s.data_ptr()
    if d.is_cuda and (codes | scales) & 15:
        raise ValueError(f"{what}: codes and scales must be 16-byte aligned")
    return fmt, rows, K, d, codes, scales


def DequantizeMX(q: QTensorMX, dtype=torch.float32) -> torch.Tensor:
    """The values that ``q`` stands for, rounded to ``dtype`` (exact in fp32)."""
    fmt, rows, K, like, codes, scales = _checked(q, "DequantizeMX")
    if not like.is_cuda:
        return _values_ref(q).to(dtype).reshape(q.Shape)
    if dtype not in _TYPES:
        raise TypeError(f"DequantizeMX: no CUDA kernel for dtype {dtype}")
    y = like.new_empty(q.Shape, dtype=dtype)
    if rows:
        _call(like.get_device(), "gb_mx_dequantize", _TYPES[dtype], fmt, codes, scales, y.data_ptr(), rows, K)
    return y


class _OnTape(torch.autograd.Function):
    """h, which a kernel wrote, as the sum of x and the residual.  (In a list: a tensor that went in would come out as a view, which nothing may be
    added to in place.)"""

    @staticmethod
    def forward(ctx, x, residual, h):
        return h[0]

    @staticmethod
    def backward(ctx, dh):
        need_x, need_r, _ = ctx.needs_input_grad
        return dh if need_x else None, dh if need_r else None, None


def AddRMSNormMX(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-6,
                 format: str = "mxfp8") -> Tuple[QTensorMX, torch.Tensor]:
    """``h = x + residual`` and the quantised ``h / sqrt(mean(h^2) + eps) * weight``: what a pre-norm block hands to its next
    products, and the stream that goes on beside them.  Returns (codes and scales, h).  The norm takes the sum before it is rounded to
    h's type; a value is rounded once, to its code: none of the arithmetic before moves one that lies next to the border between two
    codes to the other (for weights up to 2^27).  Without a residual h is x itself.  Gradients go through the sum alone: the quantised rows
    have none, like all that is computed from them here."""
    fmt, shape = _format(format), tuple(x.shape)
    a = _rows(x, "AddRMSNormMX")
    rows, K = a.shape
    r = None
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device:
            raise ValueError(f"AddRMSNormMX: the residual must be like x ({shape}, {x.dtype}, {x.device})")
        r = _rows(residual, "AddRMSNormMX")
    if weight.shape != (K,) or weight.device != x.device:
        raise ValueError(f"AddRMSNormMX: weight must have shape ({K},) on {x.device}")
    if weight.dtype not in (x.dtype, torch.float32):
        raise TypeError("AddRMSNormMX: weight dtype must equal the input dtype or be float32")
    if not x.is_cuda:
        h = a.double() if r is None else a.double() + r.double()
        y = h / torch.sqrt(h.square().sum(-1, keepdim=True) / K + eps) * weight.detach().double()
        return _quantize_ref(y, fmt, shape), _sum_of(x, residual, None if r is None else h.reshape(shape).to(x.dtype, copy=True))
    w = weight if weight.is_contiguous() else weight.contiguous()
    q, codes, scales = _empty(rows, shape, fmt, a)
    h = None if r is None else a.new_empty(shape)
    if rows:
        _call(a.get_device(), "gb_mx_add_rms_norm", _TYPES[x.dtype], fmt, a.data_ptr(), a.stride(0), None if r is None else r.data_ptr(),
              K if r is None else r.stride(0), w.data_ptr(), w.dtype == torch.float32, None if h is None else h.data_ptr(), codes, scales, rows, K, eps)
    return q, _sum_of(x, residual, h)


def _sum_of(x, residual, h):
    if h is None:
        return x
    if torch.is_grad_enabled() and (x.requires_grad or residual.requires_grad):
        return _OnTape.apply(x, residual, [h])
    return h


def _epilogue(bias, N: int, device, dtype, act, what: str):
    """(bias, its address, whether it is fp32, the activation's code) of a product in ``dtype``."""
    code = ACT.get(act)
    if code is None:
        raise ValueError(f"{what}: unknown activation {act!r}")
    if bias is None:
        return None, None, False, code
    if bias.shape != (N,) or bias.device != device:
        raise ValueError(f"{what}: bias must have shape ({N},) on {device}")
    if bias.is_cuda:
        if bias.dtype != dtype and bias.dtype != torch.float32:
            bias = bias.float()
        bias = bias.contiguous()
    return bias, bias.data_ptr(), bias.dtype == torch.float32, code


def MatMulMX(a: QTensorMX, b: QTensorMX, bias: Optional[torch.Tensor] = None, dtype=torch.bfloat16, act: Optional[str] = None) -> torch.Tensor:
    """``act(A B^T + bias)`` in ``dtype`` (bf16, fp16 or fp32) for A (..., K) and B (N, K), both quantised along K in one format.
    ``act``: relu, gelu or geluexact, as ``nn.Linear`` takes it.  No gradients."""
    fmt, M, K, like, codes, scales = _checked(a, "MatMulMX")
    fmt_b, N, K_b, like_b, codes_b, scales_b = _checked(b, "MatMulMX")
    if fmt != fmt_b:
        raise ValueError(f"MatMulMX: both operands have one format, got {a.Format} and {b.Format}")
    if len(b.Shape) != 2 or K != K_b:
        raise ValueError(f"MatMulMX: shapes {tuple(a.Shape)} and {tuple(b.Shape)} do not match (..., K) and (N, K)")
    if like.device != like_b.device:
        raise ValueError(f"MatMulMX: operands on {like.device} and {like_b.device}")
    bias, bias_at, bias_f32, code = _epilogue(bias, N, like.device, dtype, act, "MatMulMX")
    shape = (*a.Shape[:-1], N)
    if not like.is_cuda:
        y = _values_ref(a) @ _values_ref(b).t()
        if bias is not None:
            y = y + bias.detach().double()
        return _act_ref(y, act).to(dtype).reshape(shape)
    if dtype not in _TYPES:
        raise TypeError(f"MatMulMX: no CUDA kernel for dtype {dtype}")
    y = like.new_empty(shape, dtype=dtype)
    if M == 0 or N == 0:
        return y
    _call(like.get_device(), "gb_mx_matmul", fmt, codes, scales, codes_b, scales_b, y.data_ptr(), N, bias_at, bias_f32, M, N, K, _TYPES[dtype], code)
    return y


def LinearMX(x: Union[torch.Tensor, QTensorMX], weight: QTensorMX, bias: Optional[torch.Tensor] = None, act: Optional[str] = None,
             dtype=None) -> torch.Tensor:
    """``act(Q(x) W^T + bias)`` with quantised weights (out, in).  ``x``: a tensor, quantised here in the weights' format, or what
    ``AddRMSNormMX`` returned.  ``dtype``: of the result; x's own, or bf16 for a quantised x.  No gradients."""
    if isinstance(x, QTensorMX):
        return MatMulMX(x, weight, bias, dtype or torch.bfloat16, act)
    if not x.is_cuda:
        return MatMulMX(QuantizeMX(x, weight.Format), weight, bias, dtype or x.dtype, act)
    fmt, N, K, like, codes, scales = _checked(weight, "LinearMX")
    a = _rows(x, "LinearMX")
    M = a.shape[0]
    if len(weight.Shape) != 2 or a.shape[1] != K:
        raise ValueError(f"LinearMX: shapes {tuple(x.shape)} and {tuple(weight.Shape)} do not match (..., K) and (N, K)")
    if a.device != like.device:
        raise ValueError(f"LinearMX: x on {a.device}, weights on {like.device}")
    dtype = dtype or x.dtype
    if dtype not in _TYPES:
        raise TypeError(f"LinearMX: no CUDA kernel for dtype {dtype}")
    bias, bias_at, bias_f32, code = _epilogue(bias, N, a.device, dtype, act, "LinearMX")
    y = like.new_empty((*x.shape[:-1], N), dtype=dtype)
    if M == 0 or N == 0:
        return y
    need, scratch = 0, None
    if M > 16:                   # (up to 16 rows are quantised within the product's kernel)
        need = _l.lib().gb_mx_linear_bytes(M, N, K, fmt)
        scratch = like.new_empty(need, dtype=torch.uint8)
    _call(like.get_device(), "gb_mx_linear", _TYPES[x.dtype], fmt, a.data_ptr(), a.stride(0), codes, scales, y.data_ptr(), bias_at, bias_f32, M, N, K,
          _TYPES[dtype], code, None if scratch is None else scratch.data_ptr(), need)
    return y


class _TrainLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, taped):
        N, K = weight.shape
        need_x, need_w = (taped and n for n in ctx.needs_input_grad[:2])      # (parameters ask for gradients without a tape too)
        a, w = _rows(x, "TrainLinearMX"), _rows(weight, "TrainLinearMX")
        M = a.shape[0]
        ctx.meta = (x.shape, x.dtype, M, N, K, need_x, need_w)
        ctx.params = (weight, bias)
        y = x.new_empty((*x.shape[:-1], N))
        if M == 0:
            return y
        if not x.is_cuda:
            (xq, xt), (wq, wt) = (QuantizeMXPair(t) if need else (QuantizeMX(t), None) for t, need in ((a, need_w), (w, need_x)))
            ctx.save_for_backward(*(v for t in (xt, wt) for v in ((None, None) if t is None else (t.Data, t.Scales))))
            return y.copy_(MatMulMX(xq, wq, bias, x.dtype).view(y.shape))
        sizes = _l.lib().gb_mx_train_bytes
        kept = scratch = None
        n_kept, n_scratch = sizes(M, N, K, need_x, need_w, 0), sizes(M, N, K, need_x, need_w, 1)
        if n_kept:
            kept = x.new_empty(n_kept, dtype=torch.uint8)
        scratch = x.new_empty(n_scratch, dtype=torch.uint8)
        _, bias_at, bias_f32, _ = keep = _epilogue(bias, N, x.device, x.dtype, None, "TrainLinearMX")
        _call(x.get_device(), "gb_mx_train_forward", _TYPES[x.dtype], _TYPES[weight.dtype], a.data_ptr(), a.stride(0), w.data_ptr(), w.stride(0), y.data_ptr(),
              bias_at, bias_f32, M, N, K, need_x, need_w, None if kept is None else kept.data_ptr(), n_kept, scratch.data_ptr(), n_scratch)
        del keep
        ctx.save_for_backward(kept)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        xshape, xdtype, M, N, K, need_x, need_w = ctx.meta
        weight, bias = ctx.params
        need_b = bias is not None and ctx.needs_input_grad[2]
        dx = dw = db = None
        if M == 0:
            return (dy.new_zeros(xshape, dtype=xdtype) if need_x else None, emit_grad(weight, torch.zeros_like(weight)) if need_w else None,
                    emit_grad(bias, torch.zeros_like(bias)) if need_b else None, None)
        g = _rows(dy, "TrainLinearMX")
        if not dy.is_cuda:
            xt, xs, wt, ws = ctx.saved_tensors
            gq, gt = QuantizeMXPair(g)
            if need_x:
                dx = MatMulMX(gq, QTensorMX(wt, ws, "mxfp8", (K, N)), None, xdtype).reshape(xshape)
            if need_w:
                dw = MatMulMX(gt, QTensorMX(xt, xs, "mxfp8", (K, M)), None, weight.dtype)
        elif need_x or need_w:
            (kept,) = ctx.saved_tensors
            n_scratch = _l.lib().gb_mx_train_bytes(M, N, K, need_x, need_w, 2)
            scratch = dy.new_empty(n_scratch, dtype=torch.uint8)
            if need_x:
                dx = dy.new_empty(xshape, dtype=xdtype)
            if need_w:
                dw = torch.empty_like(weight, memory_format=torch.contiguous_format)
                if need_b and bias.dtype in _TYPES:
                    db = torch.empty_like(bias)
            _call(dy.get_device(), "gb_mx_train_backward", _TYPES[dy.dtype], g.data_ptr(), g.stride(0), kept.data_ptr(), None if dx is None else dx.data_ptr(),
                  _TYPES[xdtype], None if dw is None else dw.data_ptr(), _TYPES[weight.dtype], None if db is None else db.data_ptr(),
                  0 if db is None else _TYPES[db.dtype], M, N, K, scratch.data_ptr(), n_scratch)
        # gradients go to their sinks last: a sink may start a step that rewrites the parameters
        if need_b:
            if db is None and bias.dtype in (g.dtype, torch.float32):
                db = emit_vector_grad(bias, g)
            else:                   # (summed beside dW's codes; or a bias of a type of its own)
                db = emit_grad(bias, column_sum(g, out_dtype=torch.float32).to(bias.dtype) if db is None else db)
        if dw is not None:
            dw = emit_grad(weight, dw)
        return dx, dw, db, None


def TrainLinearMX(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``Q(x) Q(W)^T + b`` in MXFP8 with gradients that go straight through the rounding; every product's operands are quantised
    along its contraction: dx = Q(dy) Q(W^T)^T, dW = Q(dy^T) Q(x^T)^T, db = column sums of dy.  For the backward pass the layer
    keeps the codes of x^T and W^T, a byte a value; without a tape it neither makes nor keeps them.  Into a CUDA graph, capture it with ``torch.autograd.grad`` or ``GraphedStep``
    (``backward()`` adds to gradients on the stream that saw a parameter first, which a capture cannot follow)."""
    if weight.dim() != 2 or x.dim() == 0 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"TrainLinearMX: shapes {tuple(x.shape)} and {tuple(weight.shape)} do not match (..., K) and (N, K)")
    if weight.device != x.device:
        raise ValueError(f"TrainLinearMX: x on {x.device}, weight on {weight.device}")
    if weight.shape[0] == 0:
        raise ValueError("TrainLinearMX: a layer needs outputs")
    if bias is not None and (bias.shape != weight.shape[:1] or bias.device != x.device):
        raise ValueError(f"TrainLinearMX: bias must have shape ({weight.shape[0]},) on {x.device}")
    return _TrainLinear.apply(x, weight, bias, torch.is_grad_enabled())


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
