"""A paged cache of keys and values: new ones written to their pages, attention that reads them.

CUDA: ``csrc/rotary.cu`` (append) and ``csrc/cache_attn.cu``.  CPU: the same formulas with tensor operations.  These serve evaluation:
nothing here has a gradient."""
from __future__ import annotations

import math
from functools import lru_cache
from typing import Optional

import torch

from .. import lib as _l
from .rotary import _TYPES, has_tangent, rotate_ref, words

MAX_HEAD = 128                    # largest head that attention on CUDA takes
MAX_ROOM = 2 ** 31 - 257          # positions of a table: a tile of keys that starts within them ends within 32 bits


class Layout:
    """What the operators have to know of a cache's tensors, checked once: (pages, heads, page size, head size), rows of whole 16 bytes on CUDA."""
    __slots__ = ("keys", "values", "dtype", "code", "device", "index", "pages", "heads", "page", "width", "strides", "scale")

    def __init__(self, keys: torch.Tensor, values: torch.Tensor):
        if keys.dim() != 4 or keys.shape != values.shape or keys.dtype != values.dtype or keys.device != values.device:
            raise ValueError("KVCache: keys and values are (pages, heads, page size, head size), of one shape, type and device")
        if 0 in keys.shape:
            raise ValueError(f"KVCache: an empty cache of shape {tuple(keys.shape)}")
        if not keys.is_floating_point():
            raise TypeError(f"KVCache: a floating point type is needed, got {keys.dtype}")
        if keys.is_cuda:
            if keys.dtype not in _TYPES:
                raise TypeError(f"KVCache: no CUDA kernel for dtype {keys.dtype}")
            for t in (keys, values):
                s0, s1, s2, s3 = t.stride()
                if s3 != 1 or (t.data_ptr() | (t.shape[3] | s0 | s1 | s2) * t.element_size()) % 16:
                    raise ValueError("KVCache: rows must be contiguous, and they and the cache's strides a multiple of 16 bytes")
        self.keys, self.values, self.dtype, self.code = keys, values, keys.dtype, _TYPES.get(keys.dtype)
        self.device, self.index = keys.device, keys.get_device()
        self.pages, self.heads, self.page, self.width = keys.shape
        self.strides = (*keys.stride()[:3], *values.stride()[:3])
        self.scale = 1.0 / math.sqrt(self.width)


_I32 = torch.int32


def _check_batch(what, c, batch, table, lengths, counts):
    if (table.dtype is _I32 and lengths.dtype is _I32 and table.dim() == 2 and table.shape[0] == batch and table.shape[1] > 0
            and lengths.shape == (batch,) and table.get_device() == c.index == lengths.get_device() and table.shape[1] * c.page <= MAX_ROOM
            and (counts is None or counts.dtype is _I32 and counts.shape == (batch,) and counts.get_device() == c.index)):
        return
    for name, t, dims in (("table", table, 2), ("lengths", lengths, 1), ("counts", counts, 1)):
        if t is None:
            continue
        if t.dtype != _I32:
            raise TypeError(f"{what}: {name} must be int32, not {t.dtype}")
        if t.dim() != dims or t.shape[0] != batch:
            raise ValueError(f"{what}: {name} must have {batch} {'rows' if dims == 2 else 'entries'}, got shape {tuple(t.shape)}")
        if t.device != c.device:
            raise ValueError(f"{what}: {name} is on {t.device}, the cache on {c.device}")
    if table.shape[1] < 1:
        raise ValueError(f"{what}: the table has no columns")
    raise ValueError(f"{what}: a sequence holds up to {MAX_ROOM} positions, the table {table.shape[1]} pages of {c.page}")


def _like_cache(what, name, t, c):
    if t.dtype is not c.dtype or t.get_device() != c.index:
        raise TypeError(f"{what}: {name} is {t.dtype} on {t.device}, the cache {c.dtype} on {c.device}")
    if torch.is_grad_enabled() and (t.requires_grad or c.keys.requires_grad or c.values.requires_grad) or has_tangent(t):
        raise RuntimeError(f"{what}: no gradient goes through a cache; call under torch.no_grad()")


def _rows(t):
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _line(t):
    return t if t.stride(0) == 1 or t.shape[0] < 2 else t.contiguous()


def append(c: Layout, k, v, table, lengths, counts=None, rope=None, q=None):
    """See ``nn.KVCache.Append``.  ``rope``: (frequencies, turns, interleaved, amplitude) or None."""
    what = "KVCache.Append"
    if k.dim() != 4 or k.shape != v.shape or k.shape[2] != c.heads or k.shape[3] != c.width:
        raise ValueError(f"{what}: keys and values must be (batch, tokens, {c.heads}, {c.width}), got {tuple(k.shape)} and {tuple(v.shape)}")
    batch, tokens, heads, width = k.shape
    _like_cache(what, "k", k, c)
    _like_cache(what, "v", v, c)
    if q is not None:
        if q.dim() != 4 or q.shape[0] != batch or q.shape[1] != tokens or q.shape[3] != width:
            raise ValueError(f"{what}: queries must be ({batch}, {tokens}, heads, {width}), got {tuple(q.shape)}")
        _like_cache(what, "q", q, c)
    _check_batch(what, c, batch, table, lengths, counts)
    w, turns, interleaved, amplitude = rope if rope is not None else ((), None, False, 1.0)
    dim = 2 * len(w)
    if dim > width:
        raise ValueError(f"{what}: {dim} columns are turned, but a head has {width}")
    if c.index < 0:
        return _append_ref(c, k, v, table, lengths, counts, w, interleaved, amplitude, q)
    if turns is not None and turns.get_device() != c.index:
        raise ValueError(f"{what}: the frequencies are on {turns.device}, the cache on {c.device}; move the module there")
    k, v, lengths = _rows(k), _rows(v), _line(lengths)
    if table.stride(1) != 1:
        table = table.contiguous()
    ksb, kst, ksh, _ = k.stride()
    vsb, vst, vsh, _ = v.stride()
    out = q_at = out_at = None
    qsb = qst = qsh = q_heads = 0
    if q is not None:
        q = _rows(q)
        q_heads = q.shape[2]
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(q.shape)
        q_at, out_at = q.data_ptr(), out.data_ptr()
        qsb, qst, qsh, _ = q.stride()
    if counts is not None:
        counts = _line(counts)
    _l.call_on(c.index, "gb_cache_append", c.code, q_at, out_at, k.data_ptr(), v.data_ptr(), c.keys.data_ptr(), c.values.data_ptr(),
               words(qsb, qst, qsh, ksb, kst, ksh, vsb, vst, vsh, *c.strides, batch, tokens, q_heads, heads, width, dim, interleaved, table.stride(0),
                     table.shape[1], c.pages, c.page),
               None if turns is None else turns.data_ptr(), amplitude, table.data_ptr(), lengths.data_ptr(), None if counts is None else counts.data_ptr())
    return out


def _places(c, table, lengths, counts, tokens):
    """(positions, whether a token counts, its page, its row), each (batch, tokens)."""
    page = c.page
    at = lengths.long()[:, None] + torch.arange(tokens, device=lengths.device)
    live = torch.ones_like(at, dtype=torch.bool)
    if counts is not None:
        live = torch.arange(tokens, device=lengths.device) < counts.long()[:, None]
    inside = (at >= 0) & (at < table.shape[1] * page)
    if bool((live & ~inside).any()):
        raise ValueError("KVCache: a position lies outside of its sequence's table")
    pages = table.long().gather(1, torch.where(inside, at, 0) // page)
    if bool((live & ((pages < 0) | (pages >= c.pages))).any()):
        raise ValueError("KVCache: a page of the table is none of the cache's")
    return at, live, pages, at % page


def _append_ref(c, k, v, table, lengths, counts, w, interleaved, amplitude, q):
    at, live, pages, rows = _places(c, table, lengths, counts, k.shape[1])
    turned = rotate_ref(k.detach(), at, w, interleaved, amplitude)
    c.keys[pages[live], :, rows[live]] = turned[live]
    c.values[pages[live], :, rows[live]] = v.detach()[live]
    if q is None:
        return None
    return torch.where(live[..., None, None], rotate_ref(q.detach(), at, w, interleaved, amplitude), torch.zeros((), dtype=q.dtype))


@lru_cache(maxsize=4096)
def _plan(code, *sizes):
    """(sizes for the native call, bytes of its workspace, kernels beyond the first one)."""
    batch, tokens, heads, kv, width, _, columns, _, page, prefix = sizes[9:]
    of = code, batch, tokens, heads, kv, width, prefix, columns * page
    n = _l.lib().gb_cache_attn_bytes(*of)
    _l.check(min(n, 0), "gb_cache_attn_bytes")
    return words(*sizes), n, _l.lib().gb_cache_attn_kernels(*of) - 1


def attend(c: Layout, q, table, lengths, counts=None, scale: Optional[float] = None, shared_pages: int = 0):
    """See ``nn.KVCache.Attend``."""
    what = "KVCache.Attend"
    kv, width = c.heads, c.width
    if q.dim() != 4 or q.shape[3] != width or q.shape[2] % kv or q.shape[2] == 0:
        raise ValueError(f"{what}: queries must be (batch, tokens, heads, {width}) with a multiple of {kv} heads, got {tuple(q.shape)}")
    _like_cache(what, "q", q, c)
    batch, tokens, heads, _ = q.shape
    _check_batch(what, c, batch, table, lengths, counts)
    columns = table.shape[1]
    if not 0 <= shared_pages <= columns:
        raise ValueError(f"{what}: {shared_pages} shared pages of a table with {columns} columns")
    if scale is None:
        scale = c.scale
    elif not 0.0 < scale < math.inf:
        raise ValueError(f"{what}: the scale must be a positive number, got {scale}")
    if c.index < 0:
        return _attend_ref(c, q, table, lengths, counts, scale, shared_pages)
    if width > MAX_HEAD:
        raise ValueError(f"{what}: heads of up to {MAX_HEAD} columns on CUDA, got {width}")
    if not 1e-37 <= scale <= 1e38:
        raise ValueError(f"{what}: a scale between 1e-37 and 1e38 on CUDA, which fp32 holds, got {scale}")
    out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(q.shape)
    if batch == 0 or tokens == 0:
        return out
    sb, st, sh, sd = q.stride()
    if sd != 1 or (q.data_ptr() | (sb | st | sh) * q.element_size()) % 16:
        q = q.clone(memory_format=torch.contiguous_format)           # (an expanded or unaligned one, too)
        sb, st, sh, sd = q.stride()
    lengths = _line(lengths)
    if counts is not None:
        counts = _line(counts)
    if table.stride(1) != 1:
        table = table.contiguous()
    sizes, need, more = _plan(c.code, sb, st, sh, *c.strides, batch, tokens, heads, kv, width, table.stride(0), columns, c.pages, c.page,
                              shared_pages * c.page)
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    _l.call_on(c.index, "gb_cache_attn", c.code, q.data_ptr(), c.keys.data_ptr(), c.values.data_ptr(), out.data_ptr(), sizes, table.data_ptr(),
               lengths.data_ptr(), None if counts is None else counts.data_ptr(), scale, None if ws is None else ws.data_ptr(), need)
    _l.kernel_count += more
    return out


def _attend_ref(c, q, table, lengths, counts, scale, shared_pages):
    batch, tokens, heads, width = q.shape
    kv, page = c.heads, c.page
    ct = torch.float64 if q.dtype == torch.float64 else torch.float32
    out = torch.zeros(q.shape, dtype=q.dtype)
    for b in range(batch):
        n = int(lengths[b])
        new = tokens if counts is None else max(0, min(tokens, int(counts[b])))
        end = n + new
        if new == 0 or end <= 0:
            continue
        if end > table.shape[1] * page:
            raise ValueError("KVCache: a position lies outside of its sequence's table")
        row = table[b].long().clone()
        row[:shared_pages] = table[0, :shared_pages].long()
        row = row[:-(-end // page)]
        if bool(((row < 0) | (row >= c.pages)).any()):
            raise ValueError("KVCache: a page of the table is none of the cache's")
        k, v = (t[row].to(ct).transpose(0, 1).reshape(kv, -1, width)[:, :end] for t in (c.keys, c.values))
        rows = q[b, :new].detach().to(ct).reshape(new, kv, heads // kv, width).permute(1, 2, 0, 3)
        s = torch.matmul(rows, k[:, None].transpose(-1, -2)) * scale
        unseen = torch.arange(end) > n + torch.arange(new)[:, None]
        p = torch.softmax(s.masked_fill(unseen, -math.inf), -1)
        p = torch.where(unseen.all(-1)[:, None], torch.zeros((), dtype=ct), p)
        out[b, :new] = torch.matmul(p, v[:, None]).permute(2, 0, 1, 3).reshape(new, heads, width).to(q.dtype)
    return out
