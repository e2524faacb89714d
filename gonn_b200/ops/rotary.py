"""Rotary positions: pairs of a head's columns turned by an angle that grows with the token's position.

CUDA: ``csrc/rotary.cu``, where angles come from 64 bits of fixed point: up to position 2^27 they are off by 2.4e-8 for fp32 rows, by 9.4e-8 for
16-bit ones, whatever the position; behind it p w / 2 pi in fp64 is off by more.  CPU: the same formulas with tensor operations, angles in fp64."""
from __future__ import annotations

import math
from ctypes import c_longlong
from functools import lru_cache
from typing import Optional, Sequence

import torch

from .. import lib as _l

_fwd_ad = torch.autograd.forward_ad

_TYPES = {torch.bfloat16: _l.DT_BF16, torch.float16: _l.DT_F16, torch.float32: _l.DT_F32}


def frequencies(dim: int, base: float, scaling: str = "none", factor: float = 1.0, original: int = 0, low: float = 1.0,
                high: float = 32.0) -> Sequence[float]:
    """The angle w_i that pair i < dim / 2 is turned by a position (see ``nn.RotaryEmbedding``)."""
    if scaling == "base":
        base = base * factor ** (dim / (dim - 2))
    w = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    if scaling == "linear":
        w = [f / factor for f in w]
    elif scaling == "bands":
        def part(f):
            g = min(1.0, max(0.0, (original * f / (2 * math.pi) - low) / (high - low)))
            return f * (g + (1.0 - g) / factor)
        w = [part(f) for f in w]
    return w


def turns_of(w: Sequence[float]) -> torch.Tensor:
    """Fractions of a turn in 64 bits of fixed point, as int64; off by 2^-55 for frequencies up to 1, as their quotients in fp64 are."""
    t = torch.tensor(w, dtype=torch.float64) / (2 * math.pi)
    t = t - torch.floor(t + 0.5)                      # whole turns go; exact, like the power of two
    return torch.round(t * 2.0 ** 64).to(torch.int64)


def rotate_ref(x: torch.Tensor, positions: torch.Tensor, w: Sequence[float], interleaved: bool, amplitude: float, back: bool = False):
    """Oracle: x (batch, tokens, heads, width), positions (batch, tokens) or (tokens,); in fp32 (fp64 for fp64)."""
    ct = torch.float64 if x.dtype == torch.float64 else torch.float32
    half = len(w)
    angle = positions.to(torch.float64)[..., None] * torch.tensor(w, dtype=torch.float64, device=x.device)
    cos, sin = ((amplitude * f(angle)).to(ct)[..., None, :] for f in (torch.cos, torch.sin))
    if back:
        sin = -sin
    y = x.to(ct)
    part, rest = y[..., :2 * half], y[..., 2 * half:]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :half], part[..., half:])
    u, v = a * cos - b * sin, a * sin + b * cos
    part = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((part, rest), -1).to(x.dtype)


@lru_cache(maxsize=4096)
def words(*sizes: int):
    """Sizes and strides as the native library takes them.  (A call of eight arguments with such an array takes the host 3 us less than one of 24.)"""
    return (c_longlong * len(sizes))(*sizes)


def _launch(x, positions, turns, interleaved, amplitude, back, out=None):
    shape = x.shape
    batch, tokens, heads, width = shape
    if x.stride(3) != 1 and width > 1:
        x = x.contiguous()
    y = out if out is not None else torch.empty_like(x) if x.is_contiguous() else x.new_empty(shape)
    at, wide, pb, pt = None, 0, 0, 0
    if positions is not None:
        at, wide = positions.data_ptr(), positions.dtype is torch.int64
        pb, pt = positions.stride() if positions.dim() == 2 else (0, positions.stride(0))
    sb, st, sh, _ = x.stride()
    yb, yt, yh, _ = y.stride()
    _l.call_on(x.get_device(), "gb_rotary", _TYPES[x.dtype], x.data_ptr(), y.data_ptr(),
               words(sb, st, sh, yb, yt, yh, batch, tokens, heads, width, 2 * turns.shape[0], interleaved, back, wide, pb, pt), turns.data_ptr(), at, amplitude)
    return y


def rotate_in_place(x: torch.Tensor, plan, back: bool = False) -> None:
    """Turns a (batch, tokens, heads, width) view of a CUDA buffer where it lies, positions 0, 1, ...; ``plan``: of a RotaryEmbedding.  For buffers
    that their caller owns: no tape."""
    _, turns, interleaved, amplitude = plan
    if turns.get_device() != x.get_device():
        raise ValueError(f"rotary: the frequencies are on {turns.device}, x on {x.device}; move the module there")
    _launch(x, None, turns, interleaved, amplitude, back, x)


class _Rotary(torch.autograd.Function):
    """A turn; its gradient is the turn back (with a gradient of its own)."""

    @staticmethod
    def forward(ctx, x, positions, turns, interleaved, amplitude, back):
        ctx.rest = positions, turns, interleaved, amplitude, not back
        ctx.written = _writes(positions)        # (compared by hand: two saved tensors take the host 3 us more a step)
        return _launch(x, positions, turns, interleaved, amplitude, back)

    @staticmethod
    def backward(ctx, dy):
        if _writes(ctx.rest[0]) != ctx.written:
            raise RuntimeError("rotary: the positions have been written over since the forward pass, whose gradient needs them")
        dx = _Rotary.apply(dy, *ctx.rest) if torch.is_grad_enabled() else _launch(dy, *ctx.rest)
        return dx, None, None, None, None, None

    @staticmethod
    def jvp(ctx, dx, *_):
        *rest, back = ctx.rest
        return None if dx is None else _Rotary.apply(dx, *rest, not back)


def has_tangent(t: torch.Tensor) -> bool:
    """Whether a forward-mode derivative is asked for along t."""
    return _fwd_ad._current_level >= 0 and _fwd_ad.unpack_dual(t).tangent is not None


def _writes(positions) -> int:
    """How often a tensor has been written to in place (nothing counts that for tensors of inference mode)."""
    return 0 if positions is None or positions.is_inference() else positions._version


def rotary(x: torch.Tensor, positions: Optional[torch.Tensor], w: Sequence[float], turns: torch.Tensor, interleaved: bool = False,
           amplitude: float = 1.0) -> torch.Tensor:
    """x (batch, tokens, heads, width), any strides; positions: int32 or int64, (tokens,) or (batch, tokens), or None for 0, 1, ...;
    differentiable in x."""
    if x.dim() != 4:
        raise ValueError(f"rotary: expected (batch, tokens, heads, width), got shape {tuple(x.shape)}")
    batch, tokens, _, width = x.shape
    if 2 * len(w) > width:
        raise ValueError(f"rotary: {2 * len(w)} columns are turned, but a head has {width}")
    device = x.get_device()
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"rotary: positions are int32 or int64, not {positions.dtype}")
        if positions.shape != (tokens,) and positions.shape != (batch, tokens):
            raise ValueError(f"rotary: positions must have shape ({tokens},) or ({batch}, {tokens}), got {tuple(positions.shape)}")
        if positions.get_device() != device:
            raise ValueError(f"rotary: positions are on {positions.device}, x on {x.device}")
    if device < 0:
        if not x.is_floating_point():
            raise TypeError(f"rotary: a floating point tensor is needed, got {x.dtype}")
        at = torch.arange(tokens, device=x.device) if positions is None else positions
        return rotate_ref(x, at, w, interleaved, amplitude)
    if x.dtype not in _TYPES:
        raise TypeError(f"rotary: no CUDA kernel for dtype {x.dtype}")
    if turns.get_device() != device:
        raise ValueError(f"rotary: the frequencies are on {turns.device}, x on {x.device}; move the module there")
    if torch.is_grad_enabled() and x.requires_grad or has_tangent(x):
        return _Rotary.apply(x, positions, turns, interleaved, amplitude, False)
    return _launch(x, positions, turns, interleaved, amplitude, False)
