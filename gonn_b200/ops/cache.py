"""A paged cache of keys and values: new ones written to their pages, attention that reads them.

CUDA: ``csrc/rotary.cu`` (append) and ``csrc/cache_attn.cu``.  CPU: the same formulas with tensor operations.  These serve evaluation:
nothing here has a gradient."""
from __future__ import annotations

import math
from ctypes import c_longlong
from functools import lru_cache
from typing import Optional

import torch

from .. import lib as _l
from .rotary import _TYPES, rotate_ref

MAX_HEAD = 128                    # largest head that attention on CUDA takes


def check_cache(k: torch.Tensor, v: torch.Tensor) -> None:
    """Keys and values as the operators take them: (pages, heads, page size, head size), rows of whole 16 bytes on CUDA."""
    if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
        raise ValueError("KVCache: keys and values are (pages, heads, page size, head size), of one shape, type and device")
    if 0 in k.shape:
        raise ValueError(f"KVCache: an empty cache of shape {tuple(k.shape)}")
    if not k.is_floating_point():
        raise TypeError(f"KVCache: a floating point type is needed, got {k.dtype}")
    if k.is_cuda:
        if k.dtype not in _TYPES:
            raise TypeError(f"KVCache: no CUDA kernel for dtype {k.dtype}")
        for t in (k, v):
            if t.stride(3) != 1 or (t.data_ptr() | (t.shape[3] | t.stride(0) | t.stride(1) | t.stride(2)) * t.element_size()) % 16:
                raise ValueError("KVCache: rows must be contiguous, and they and the cache's strides a multiple of 16 bytes")


def _check_batch(what, cache, batch, table, lengths, counts):
    device = cache.device
    for name, t, dims in (("table", table, 2), ("lengths", lengths, 1), ("counts", counts, 1)):
        if t is None:
            continue
        if t.dtype != torch.int32:
            raise TypeError(f"{what}: {name} must be int32, not {t.dtype}")
        if t.dim() != dims or t.shape[0] != batch:
            raise ValueError(f"{what}: {name} must have {batch} {'rows' if dims == 2 else 'entries'}, got shape {tuple(t.shape)}")
        if t.device != device:
            raise ValueError(f"{what}: {name} is on {t.device}, the cache on {device}")
    if table.shape[1] < 1:
        raise ValueError(f"{what}: the table has no columns")
    if table.shape[1] * cache.shape[2] >= 2 ** 31 - 1:
        raise ValueError(f"{what}: a sequence holds fewer than 2^31 - 1 positions, the table {table.shape[1]} pages of {cache.shape[2]}")


def _like_cache(what, name, t, cache):
    if t.dtype != cache.dtype or t.device != cache.device:
        raise TypeError(f"{what}: {name} is {t.dtype} on {t.device}, the cache {cache.dtype} on {cache.device}")
    if torch.is_grad_enabled() and t.requires_grad:
        raise RuntimeError(f"{what}: no gradient goes through a cache; call under torch.no_grad()")


def _rows(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _line(t):
    return t if t is None or t.shape[0] < 2 or t.stride(0) == 1 else t.contiguous()


def append(k_cache, v_cache, k, v, table, lengths, counts=None, rope=None, q=None):
    """See ``nn.KVCache.Append``.  ``rope``: (frequencies, turns, interleaved, amplitude) or None."""
    what = "KVCache.Append"
    if k.dim() != 4 or k.shape != v.shape or k.shape[2] != k_cache.shape[1] or k.shape[3] != k_cache.shape[3]:
        raise ValueError(f"{what}: keys and values must be (batch, tokens, {k_cache.shape[1]}, {k_cache.shape[3]}), got {tuple(k.shape)} and {tuple(v.shape)}")
    batch, tokens, heads, width = k.shape
    _like_cache(what, "k", k, k_cache)
    _like_cache(what, "v", v, k_cache)
    if q is not None:
        if q.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != width:
            raise ValueError(f"{what}: queries must be ({batch}, {tokens}, heads, {width}), got {tuple(q.shape)}")
        _like_cache(what, "q", q, k_cache)
    _check_batch(what, k_cache, batch, table, lengths, counts)
    w, turns, interleaved, amplitude = rope if rope is not None else ((), None, False, 1.0)
    if 2 * len(w) > width:
        raise ValueError(f"{what}: {2 * len(w)} columns are turned, but a head has {width}")
    if not k.is_cuda:
        return _append_ref(k_cache, v_cache, k, v, table, lengths, counts, w, interleaved, amplitude, q)
    if turns is not None and turns.device != k.device:
        raise ValueError(f"{what}: the frequencies are on {turns.device}, the cache on {k.device}; move the module there")
    k, v = _rows(k), _rows(v)
    lengths, counts = _line(lengths), _line(counts)
    if table.stride(1) != 1:
        table = table.contiguous()
    out = None
    qs = (0, 0, 0)
    if q is not None:
        q = _rows(q)
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        qs = q.stride()[:3]
    strides = (c_longlong * 15)(*qs, *k.stride()[:3], *v.stride()[:3], *k_cache.stride()[:3], *v_cache.stride()[:3])
    _l.call_on(k.get_device(), "gb_cache_append", _TYPES[k.dtype], None if q is None else q.data_ptr(), None if q is None else out.data_ptr(),
               k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), strides, batch, tokens, 0 if q is None else q.shape[2], heads,
               width, 2 * len(w), interleaved, None if turns is None else turns.data_ptr(), amplitude, table.data_ptr(), table.stride(0),
               table.shape[1], k_cache.shape[0], k_cache.shape[2], lengths.data_ptr(), None if counts is None else counts.data_ptr())
    return out


def _places(k_cache, table, lengths, counts, tokens):
    """(positions, whether a token counts, its page, its row), each (batch, tokens)."""
    page = k_cache.shape[2]
    at = lengths.long()[:, None] + torch.arange(tokens, device=lengths.device)
    live = torch.ones_like(at, dtype=torch.bool)
    if counts is not None:
        live = torch.arange(tokens, device=lengths.device) < counts.long()[:, None]
    inside = (at >= 0) & (at < table.shape[1] * page)
    if bool((live & ~inside).any()):
        raise ValueError("KVCache: a position lies outside of its sequence's table")
    pages = table.long().gather(1, torch.where(inside, at, 0) // page)
    if bool((live & ((pages < 0) | (pages >= k_cache.shape[0]))).any()):
        raise ValueError("KVCache: a page of the table is none of the cache's")
    return at, live, pages, at % page


def _append_ref(k_cache, v_cache, k, v, table, lengths, counts, w, interleaved, amplitude, q):
    at, live, pages, rows = _places(k_cache, table, lengths, counts, k.shape[1])
    turned = rotate_ref(k.detach(), at, w, interleaved, amplitude)
    k_cache[pages[live], :, rows[live]] = turned[live]
    v_cache[pages[live], :, rows[live]] = v.detach()[live]
    if q is None:
        return None
    return torch.where(live[..., None, None], rotate_ref(q.detach(), at, w, interleaved, amplitude), torch.zeros((), dtype=q.dtype))


@lru_cache(maxsize=1024)
def _workspace(code, batch, tokens, heads, kv, width, prefix):
    n = _l.lib().gb_cache_attn_bytes(code, batch, tokens, heads, kv, width, prefix)
    _l.check(min(n, 0), "gb_cache_attn_bytes")
    return n


def attend(k_cache, v_cache, q, table, lengths, counts=None, scale: Optional[float] = None, shared_pages: int = 0):
    """See ``nn.KVCache.Attend``."""
    what = "KVCache.Attend"
    pages, kv, page, width = k_cache.shape
    if q.dim() != 4 or q.shape[3] != width or q.shape[2] % kv or q.shape[2] == 0:
        raise ValueError(f"{what}: queries must be (batch, tokens, heads, {width}) with a multiple of {kv} heads, got {tuple(q.shape)}")
    _like_cache(what, "q", q, k_cache)
    batch, tokens, heads, _ = q.shape
    _check_batch(what, k_cache, batch, table, lengths, counts)
    if not 0 <= shared_pages <= table.shape[1]:
        raise ValueError(f"{what}: {shared_pages} shared pages of a table with {table.shape[1]} columns")
    scale = 1.0 / math.sqrt(width) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"{what}: the scale must be a positive number, got {scale}")
    if not q.is_cuda:
        return _attend_ref(k_cache, v_cache, q, table, lengths, counts, scale, shared_pages)
    if width > MAX_HEAD:
        raise ValueError(f"{what}: heads of up to {MAX_HEAD} columns on CUDA, got {width}")
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if batch == 0 or tokens == 0:
        return out
    sb, st, sh, sd = q.stride()
    if sd != 1 or q.data_ptr() % 16 or (sb | st | sh) * q.element_size() % 16:
        q = q.contiguous()
        sb, st, sh, sd = q.stride()
    lengths, counts = _line(lengths), _line(counts)
    if table.stride(1) != 1:
        table = table.contiguous()
    code = _TYPES[q.dtype]
    ks, vs = k_cache.stride()[:3], v_cache.stride()[:3]
    need = _workspace(code, batch, tokens, heads, kv, width, shared_pages * page)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    strides = (c_longlong * 9)(sb, st, sh, *ks, *vs)
    _l.call_on(q.get_device(), "gb_cache_attn", code, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), strides, batch, tokens,
               heads, kv, width, table.data_ptr(), table.stride(0), table.shape[1], pages, page, lengths.data_ptr(),
               None if counts is None else counts.data_ptr(), shared_pages * page, scale, ws.data_ptr(), need)
    return out


def _attend_ref(k_cache, v_cache, q, table, lengths, counts, scale, shared_pages):
    batch, tokens, heads, width = q.shape
    kv, page = k_cache.shape[1], k_cache.shape[2]
    ct = torch.float64 if q.dtype == torch.float64 else torch.float32
    out = torch.zeros(q.shape, dtype=q.dtype)
    for b in range(batch):
        n = int(lengths[b])
        c = tokens if counts is None else max(0, min(tokens, int(counts[b])))
        end = n + c
        if c == 0 or end <= 0:
            continue
        if end > table.shape[1] * page:
            raise ValueError("KVCache: a position lies outside of its sequence's table")
        row = table[b].long().clone()
        row[:shared_pages] = table[0, :shared_pages].long()
        row = row[:-(-end // page)]
        if bool(((row < 0) | (row >= k_cache.shape[0])).any()):
            raise ValueError("KVCache: a page of the table is none of the cache's")
        k, v = (t[row].to(ct).transpose(0, 1).reshape(kv, -1, width)[:, :end] for t in (k_cache, v_cache))
        rows = q[b, :c].detach().to(ct).reshape(c, kv, heads // kv, width).permute(1, 2, 0, 3)
        s = torch.matmul(rows, k[:, None].transpose(-1, -2)) * scale
        unseen = torch.arange(end) > n + torch.arange(c)[:, None]
        p = torch.softmax(s.masked_fill(unseen, -math.inf), -1)
        p = torch.where(unseen.all(-1)[:, None], torch.zeros((), dtype=ct), p)
        out[b, :c] = torch.matmul(p, v[:, None]).permute(2, 0, 1, 3).reshape(c, heads, width).to(q.dtype)
    return out
