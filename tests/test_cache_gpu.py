"""Rotary positions and the paged cache on the GPU, against the formulas in fp64.

Tolerances.  Rotation: (a cos - b sin) with cos and sin off by 2e-7 of the amplitude (an angle in 32 bits of a turn, pi 2^-25 = 9.4e-8, and the
function's own 2 units) in fp32 and by 6e-7 in 16 bits (the same angle, and 2^-21 of the hardware's functions within half a turn, as documented: 4.8e-7),
plus three fp32 roundings, then one rounding to the type: eps / 2 of the value.  Attention: a score's sum of D products is off by
at most D 2^-24 of the sum of its magnitudes, its scaling and exponential by 2^-21 of it and 2^-22: together at most d of a weight.  Weights in 16
bits are rounded by eps / 2 each.  With A = sum p |v| / sum p the result is off by at most 2 d A + n 2^-24 A (sums of n terms) + eps / 2 A (16
bits) + eps / 2 of the result (its own rounding)."""
import math

import pytest
import torch

from gonn_b200 import lib, nn

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("status_ok")]
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def half(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------------------------------------------ rotation
def turned(x, at, rope, back=False):
    """(the rotation in fp64, its tolerance)."""
    n = rope.dim // 2
    w = torch.tensor(rope._w, dtype=torch.float64, device=x.device)
    angle = at.double()[..., None, None] * w * (-1 if back else 1)
    z = x.double()
    part, rest = z[..., :rope.dim], z[..., rope.dim:]
    a, b = (part[..., 0::2], part[..., 1::2]) if rope.interleaved else (part[..., :n], part[..., n:])
    c, s = rope.amplitude * torch.cos(angle), rope.amplitude * torch.sin(angle)
    u, v = a * c - b * s, a * s + b * c
    size = rope.amplitude * (a.abs() + b.abs())
    part, err = (torch.stack((p, q), -1).flatten(-2) if rope.interleaved else torch.cat((p, q), -1) for p, q in ((u, v), (size, size)))
    y = torch.cat((part, rest), -1)
    # the angle itself, p w in fp64: 2^-53 of it
    slack = (2e-7 if x.dtype == F32 else 6e-7) + 3 * 2.0 ** -24 + float(at.abs().max()) * 2.0 ** -52 if at.numel() else 0.0
    return y, torch.cat((err * slack, torch.zeros_like(rest)), -1) + y.abs() * half(x.dtype) * 1.001 + 1e-7 * (x.dtype == F16) + 1e-37


def close(got, want):
    y, tol = want
    bad = ~((got.double() - y).abs() <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - y).abs() / tol).max()):.3f} of the tolerance"


SCALINGS = [{}, dict(scaling="linear", factor=4.0), dict(scaling="base", factor=8.0, amplitude=1.3),
            dict(scaling="bands", factor=8.0, original=2048, amplitude=1.25)]


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("shape,dim", [((1, 1, 1, 2), 2), ((1, 1, 32, 128), 128), ((2, 5, 3, 80), 52), ((3, 77, 4, 64), 64), ((2, 33, 5, 7), 6),
                                       ((1, 300, 2, 72), 40), ((2, 3, 2, 2050), 2048), ((5, 129, 1, 24), 24)])
def test_rotary(dtype, inter, shape, dim):
    for kw in SCALINGS[:1] if dim == 2 else SCALINGS:
        rope = nn.RotaryEmbedding(dim, 500000.0, interleaved=inter, device="cuda", **kw)
        x = torch.randn(shape, device="cuda").to(dtype)
        for at in (None, torch.arange(shape[1], device="cuda") + 131000, torch.randint(-3, 2 ** 31 - 1, shape[:2], device="cuda", dtype=torch.int32)):
            p = torch.arange(shape[1], device="cuda") if at is None else at
            close(rope(x, at), turned(x, p, rope))


def test_rotary_gradient():
    rope = nn.RotaryEmbedding(24, interleaved=True, amplitude=1.5, device="cuda")
    x = torch.randn(2, 9, 3, 40, device="cuda", requires_grad=True)
    at = torch.randint(0, 5000, (2, 9), device="cuda")
    dy = torch.randn_like(x)
    dx, = torch.autograd.grad(rope(x, at), x, dy)
    close(dx, turned(dy, at, rope, back=True))
    # differences along a direction: the map is linear
    d = torch.randn_like(x)
    with torch.no_grad():
        slope = ((rope(x + d, at).double() - rope(x - d, at).double()) * dy.double()).sum() / 2
    assert abs(float(slope - (dx.double() * d.double()).sum())) <= 1e-5 * float((dx.double() * d.double()).abs().sum())
    # broadcast gradients, and one of the gradient
    dx, = torch.autograd.grad(rope(x, at).sum(), x, create_graph=False)
    close(dx, turned(torch.ones_like(x), at, rope, back=True))
    g = torch.ones_like(x).requires_grad_()
    first, = torch.autograd.grad(rope(x, at), x, g, create_graph=True)
    again, = torch.autograd.grad(first, g, dy)
    close(again, turned(dy, at, rope))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rotary_strides(dtype):
    rope = nn.RotaryEmbedding(64, device="cuda")
    qkv = torch.randn(2, 33, 3, 4, 64, device="cuda").to(dtype)
    at = torch.arange(33, device="cuda")
    close(rope(qkv[:, :, :2].flatten(2, 3), at), turned(qkv[:, :, :2].flatten(2, 3), at, rope))
    for x in (qkv[:, :, 1], qkv[:, :, 2].transpose(1, 2).contiguous().transpose(1, 2), torch.randn(2, 4, 64, 33, device="cuda").to(dtype).permute(0, 3, 1, 2),
              torch.randn(2 * 33 * 4 * 65 + 1, device="cuda").to(dtype)[1:].view(2, 33, 4, 65)[..., :64]):
        close(rope(x, at), turned(x, at, rope))
    wide = torch.arange(2 * 66, device="cuda").view(2, 66)
    close(rope(qkv[:, :, 0], wide[:, ::2]), turned(qkv[:, :, 0], wide[:, ::2], rope))


def test_rotary_beyond_32_bits():
    n = 2 ** 31 // (64 * 16) + 3
    x = torch.zeros(1, n, 16, 64, device="cuda", dtype=BF)
    x[:, -5:] = torch.randn(1, 5, 16, 64, device="cuda").to(BF)
    rope = nn.RotaryEmbedding(64, device="cuda")
    y = rope(x)
    close(y[:, -5:], turned(x[:, -5:], torch.arange(n - 5, n, device="cuda"), rope))


# ------------------------------------------------------------------------------------------------------------------ the cache
def batch(B, T, H, kv, D, page, lengths, dtype, prefix=0, counts=None, spare=3, seed=0, nan=True):
    """A cache whose sequences' pages lie in any order, with NaN wherever no position is; q, k, v of the new tokens."""
    g = torch.Generator("cuda").manual_seed(seed)
    needs = [max(1, -(-(n + T) // page)) for n in lengths]
    total = prefix + sum(n - prefix for n in needs)
    order = torch.randperm(total + spare, generator=g, device="cuda").int()
    table = torch.full((B, max(needs) + 1), -7, dtype=torch.int32, device="cuda")
    used = prefix
    for b, n in enumerate(needs):
        table[b, :prefix] = order[:prefix]
        table[b, prefix:n] = order[used:used + n - prefix]
        used += n - prefix
    kc, vc = (torch.randn(total + spare, kv, page, D, generator=g, device="cuda").to(dtype) for _ in range(2))
    there = torch.zeros(total + spare, page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lengths):
        p = torch.arange(n, device="cuda")
        there[table[b].long()[p // page], p % page] = True
    if nan:
        for t in (kc, vc):
            t.transpose(1, 2)[~there] = math.nan
    new = [torch.randn(B, T, h, D, generator=g, device="cuda").to(dtype) for h in (H, kv, kv)]
    new[0] *= 2
    c = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    return nn.KVCache.Over(kc, vc), table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), c, new


def attended(cache, q, table, lengths, counts, scale=None):
    """(attention in fp64, its tolerance)."""
    B, T, H, D = q.shape
    kv, page = cache.Keys.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    y, tol = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b in range(B):
        n, c = int(lengths[b]), T if counts is None else max(0, min(T, int(counts[b])))
        if c == 0 or n + c <= 0:
            continue
        at = torch.arange(n + c, device="cuda")
        rows = table[b].long()[at // page]
        k, v = (t[rows, :, at % page].double().transpose(0, 1).repeat_interleave(H // kv, 0) for t in (cache.Keys, cache.Values))
        x = q[b, :c].double().transpose(0, 1)
        s = x @ k.transpose(1, 2) * scale
        hidden = at > n + torch.arange(c, device="cuda")[:, None]
        s = s.masked_fill(hidden, -math.inf)
        p = torch.softmax(s, -1).masked_fill(hidden, 0)
        d = (D * 2.0 ** -24 * (x.abs() @ k.abs().transpose(1, 2)) * scale).amax(-1, keepdim=True) + 2.0 ** -21 * s.masked_fill(hidden, 0).abs().amax(-1, keepdim=True) + 2.0 ** -22
        o, A = p @ v, p @ v.abs()
        e = half(q.dtype)
        t = (2 * d + (n + c) * 2.0 ** -24 + (e if q.dtype != F32 else 0)) * A + e * o.abs() * 1.01 + (2.0 ** -24 if q.dtype == F16 else 0)
        y[b, :c], tol[b, :c] = o.transpose(0, 1), t.transpose(0, 1)
    return y, tol


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("B,T,H,kv,D,dim,page,lengths,counts", [
    (1, 1, 16, 16, 128, 128, 64, [1000], None), (2, 77, 4, 2, 64, 64, 16, [0, 5], None), (5, 13, 6, 3, 72, 40, 24, [1, 0, 100, 23, 24], [13, 0, 1, 7, -2]),
    (3, 4, 1, 1, 8, 2, 1, [0, 3, 9], [5, 4, 2]), (1, 500, 3, 1, 40, 40, 7, [131000], None), (300, 1, 2, 2, 16, 8, 3, [7] * 300, None)])
def test_append(dtype, inter, B, T, H, kv, D, dim, page, lengths, counts):
    cache, table, at, c, (q, k, v) = batch(B, T, H, kv, D, page, lengths, dtype, counts=counts)
    rope = nn.RotaryEmbedding(dim, interleaved=inter, scaling="linear", factor=2.0, amplitude=1.1, device="cuda")
    before = cache.Keys.clone(), cache.Values.clone()
    out = cache.Append(k, v, table, at, counts=c, rotary=rope, q=q)
    where = at.long()[:, None] + torch.arange(T, device="cuda")
    live = torch.ones(B, T, dtype=torch.bool, device="cuda") if c is None else torch.arange(T, device="cuda") < c[:, None]
    want, tol = turned(q, where, rope)
    close(out, (want * live[..., None, None], tol * live[..., None, None]))
    pages = table.long().gather(1, where // page)[live]
    want, tol = turned(k, where, rope)
    close(cache.Keys[pages, :, where[live] % page], (want[live], tol[live]))
    assert torch.equal(cache.Values[pages, :, where[live] % page], v[live])
    # all other rows are as they were, bit for bit
    for t, old in zip((cache.Keys, cache.Values), before):
        old[pages, :, where[live] % page] = t[pages, :, where[live] % page]
        bits = torch.int32 if dtype == F32 else torch.int16
        assert torch.equal(t.view(bits), old.view(bits))
    # without a rotation or queries
    assert cache.Append(k, v, table, at, counts=c) is None
    assert torch.equal(cache.Keys[pages, :, where[live] % page], k[live])


ATTEND = [
    (1, 1, 1, 1, 64, 16, [0], None), (1, 1, 16, 16, 128, 64, [2047], None), (3, 1, 8, 2, 128, 16, [5, 0, 700], None), (2, 5, 6, 2, 64, 24, [100, 3], None),
    (5, 3, 4, 4, 72, 1, [0, 1, 63, 64, 65], [3, 0, 2, 1, -1]), (1, 40, 12, 3, 128, 33, [500], None), (2, 300, 2, 1, 64, 64, [0, 77], [300, 13]),
    (7, 1, 40, 1, 128, 128, [0, 10, 200, 300, 4000, 31, 32], None), (150, 1, 2, 1, 16, 8, list(range(150)), None), (1, 2, 2, 2, 8, 5, [20000], None),
    (2, 17, 8, 1, 104, 200, [1, 1500], [17, 16]),
    # 6, 10, 24 and 48 rows to a key head: in clusters, and dealt out
    (3, 2, 12, 4, 128, 16, [10, 300, 77], None), (3, 2, 12, 4, 128, 16, [10, 300, 15000], None), (2, 2, 6, 2, 64, 64, [9000, 8190], [2, 1]),
    (2, 2, 10, 2, 128, 7, [9001, 3], None), (3, 5, 4, 2, 64, 64, [9000, 77, 9999], [5, 0, 3]), (2, 6, 8, 2, 128, 64, [9000, 4444], None),
    (1, 12, 4, 1, 72, 24, [12345], None), (400, 2, 1, 1, 24, 16, [0] * 399 + [900], [0] * 399 + [2])]


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("B,T,H,kv,D,page,lengths,counts", ATTEND)
def test_attend(dtype, B, T, H, kv, D, page, lengths, counts):
    cache, table, at, c, (q, k, v) = batch(B, T, H, kv, D, page, lengths, dtype, counts=counts)
    cache.Append(k, v, table, at, counts=c)
    close(cache.Attend(q, table, at, counts=c), attended(cache, q, table, at, c))
    close(cache.Attend(q, table, at, counts=c, scale=0.3), attended(cache, q, table, at, c, 0.3))


SHARED = [
    (2, 1, 1, 1, 64, 16, 1, [16, 17], None), (16, 1, 16, 16, 128, 64, 30, [1920 + 9 * i for i in range(16)], None),
    (70, 1, 8, 2, 128, 32, 3, [96 + i for i in range(70)], None), (5, 3, 4, 2, 72, 24, 2, [48, 49, 100, 77, 48], [3, 0, 1, 2, 3]),
    (33, 2, 3, 1, 40, 7, 11, [77 + i for i in range(33)], None), (3, 1, 64, 1, 128, 100, 4, [400, 401, 555], None),
    (300, 1, 4, 1, 64, 16, 40, [640 + i % 50 for i in range(300)], None), (9, 4, 2, 2, 128, 64, 1, [64] * 9, [0] * 9)]


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("B,T,H,kv,D,page,prefix,lengths,counts", SHARED)
def test_shared(dtype, B, T, H, kv, D, page, prefix, lengths, counts):
    cache, table, at, c, (q, k, v) = batch(B, T, H, kv, D, page, lengths, dtype, prefix=prefix, counts=counts)
    cache.Append(k, v, table, at, counts=c)
    want = attended(cache, q, table, at, c)
    close(cache.Attend(q, table, at, counts=c, shared_pages=prefix), want)
    close(cache.Attend(q, table, at, counts=c), want)


def test_attend_twice_is_the_same_bit_for_bit():
    cache, table, at, c, (q, k, v) = batch(40, 1, 8, 2, 128, 16, [17 * i for i in range(40)], BF)
    cache.Append(k, v, table, at)
    first = cache.Attend(q, table, at)
    for _ in range(5):
        assert torch.equal(cache.Attend(q, table, at), first)


def test_large_scores_and_infinities():
    """Scores of several thousand, values that are infinite, scores of minus infinity and NaN."""
    for dtype in (BF, F32):
        cache, table, at, c, (q, k, v) = batch(2, 1, 2, 1, 64, 16, [300, 40], dtype)
        cache.Append(k, v, table, at)
        big = q * 100
        close(cache.Attend(big, table, at), attended(cache, big, table, at, c))
        page, row = int(table[0, 2]), 5
        cache.Values[page, 0, row, 3] = math.inf
        out = cache.Attend(q, table, at)
        assert bool((out[0, :, :, 3] == math.inf).all()) and bool(torch.isfinite(out[1]).all()) and bool(torch.isfinite(out[0, :, :, :3]).all())
        cache.Values[page, 0, row, 3] = 0
        cache.Keys[page, 0, row] = math.nan
        out = cache.Attend(q, table, at)
        assert bool(out[0].isnan().all()) and bool(torch.isfinite(out[1]).all())
        # a key of minus infinity along a positive query has no weight
        cache.Keys[page, 0, row] = 0
        cache.Keys[page, 0, row, 0] = -math.inf
        q[0, 0, :, 0] = 1
        close(cache.Attend(q, table, at)[1:], tuple(t[1:] for t in attended(cache, q, table, at, c)))
        assert bool(torch.isfinite(cache.Attend(q, table, at)).all())


def test_orders_of_the_cache():
    """Rows by heads in the page, keys and values in one tensor, a slice of another cache, strided queries and tables."""
    cache, table, at, c, (q, k, v) = batch(3, 2, 4, 2, 64, 16, [5, 50, 33], BF, nan=False)
    cache.Append(k, v, table, at)
    want = attended(cache, q, table, at, c)
    by_row = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (cache.Keys, cache.Values)]
    both = torch.stack((cache.Keys, cache.Values), 1)
    layers = torch.stack((cache.Keys, cache.Values, cache.Keys), 3)
    wide = torch.zeros(3, 2, 3, 4, 64, device="cuda", dtype=BF)
    wide[:, :, 0] = q
    tables = torch.zeros(3, 2 * table.shape[1], device="cuda", dtype=torch.int32)
    tables[:, ::2] = table
    for keys, values in (by_row, (both[:, 0], both[:, 1]), (layers[..., 0, :], layers[..., 1, :])):
        other = nn.KVCache.Over(keys, values)
        other.Append(k, v, table, at)
        close(other.Attend(wide[:, :, 0], tables[:, ::2], at), want)
    close(cache.Attend(q.transpose(2, 3).contiguous().transpose(2, 3), table, at), want)


def test_beyond_32_bits():
    """Pages behind 2^31 values, a sequence behind 2^17 positions."""
    pages = 2 ** 31 // (2 * 64 * 128) + 9
    keys, values = (torch.zeros(pages, 2, 64, 128, device="cuda", dtype=BF) for _ in range(2))
    keys[-9:], values[-9:] = torch.randn(2, 9, 2, 64, 128, device="cuda").to(BF)
    cache = nn.KVCache.Over(keys, values)
    table = torch.arange(pages - 8, pages, device="cuda", dtype=torch.int32).flip(0).view(2, 4)
    at = torch.tensor([200, 255], device="cuda", dtype=torch.int32)
    q, k, v = (torch.randn(2, 1, h, 128, device="cuda").to(BF) for h in (4, 2, 2))
    cache.Append(k, v, table, at)
    assert torch.equal(cache.Values[int(table[1, 3]), :, 63], v[1, 0])
    close(cache.Attend(q, table, at), attended(cache, q, table, at, None))


def test_tables_too_long_to_number_their_tiles():
    cache = nn.KVCache(1, 1024, 64, 8, dtype=BF, device="cuda")
    q, at = torch.zeros(1, 1, 64, 8, device="cuda", dtype=BF), torch.zeros(1, device="cuda", dtype=torch.int32)
    with pytest.raises(lib.NativeError):
        cache.Attend(q, torch.zeros(1, 2 ** 20, device="cuda", dtype=torch.int32), at)


def test_calls_of_a_new_thread():
    """A thread whose first CUDA call is this one."""
    import threading
    cache, table, at, c, (q, k, v) = batch(2, 1, 4, 2, 64, 64, [100, 3], BF)
    cache.Append(k, v, table, at)
    outs = []
    thread = threading.Thread(target=lambda: outs.append(cache.Attend(q, table, at)))
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    close(outs[0], attended(cache, q, table, at, c))


def test_empty_calls():
    cache = nn.KVCache(4, 16, 2, 64, dtype=BF, device="cuda")
    table, at = torch.zeros(0, 1, device="cuda", dtype=torch.int32), torch.zeros(0, device="cuda", dtype=torch.int32)
    q, k = torch.zeros(0, 1, 4, 64, device="cuda", dtype=BF), torch.zeros(0, 1, 2, 64, device="cuda", dtype=BF)
    assert cache.Append(k, k, table, at, q=q).shape == q.shape and cache.Attend(q, table, at).shape == q.shape
    table, at = torch.zeros(2, 1, device="cuda", dtype=torch.int32), torch.zeros(2, device="cuda", dtype=torch.int32)
    q, k = torch.zeros(2, 0, 4, 64, device="cuda", dtype=BF), torch.zeros(2, 0, 2, 64, device="cuda", dtype=BF)
    assert cache.Append(k, k, table, at, q=q).shape == q.shape and cache.Attend(q, table, at).shape == q.shape
    assert nn.RotaryEmbedding(64, device="cuda")(q).shape == q.shape
    # no position at all is seen: zeros
    q = torch.randn(2, 1, 4, 64, device="cuda").to(BF)
    assert not bool(cache.Attend(q, table, torch.tensor([-1, -9], device="cuda", dtype=torch.int32)).any())


def test_bad_tables_are_reported():
    """Nothing is written, the status tells, and the context stays usable."""
    lib.assert_status_ok()
    cache = nn.KVCache(4, 16, 2, 64, dtype=BF, device="cuda")
    before = cache.Keys.clone()
    k = torch.randn(2, 1, 2, 64, device="cuda").to(BF)
    q = torch.randn(2, 1, 4, 64, device="cuda").to(BF)
    zero = torch.zeros(2, device="cuda", dtype=torch.int32)
    for table, at in ((torch.full((2, 1), 4, device="cuda", dtype=torch.int32), zero), (torch.full((2, 1), -1, device="cuda", dtype=torch.int32), zero),
                      (torch.zeros(2, 1, device="cuda", dtype=torch.int32), zero + 16), (torch.zeros(2, 1, device="cuda", dtype=torch.int32), zero - 1)):
        cache.Append(k, k, table, at)
        assert lib.read_status()[0] == 5
        assert torch.equal(cache.Keys, before)
        for tokens in (1, 70):                                          # few rows, many
            cache.Attend(q.expand(2, tokens, 4, 64), table, at)
            assert lib.read_status()[0] == (0 if int(at[0]) < 0 and tokens == 1 else 5)
    lib.assert_status_ok()


def test_other_streams_and_graphs():
    """Two captured calls replayed on different streams, with lengths that change between replays; none shares a workspace."""
    cache, table, at, c, new = batch(6, 2, 8, 2, 128, 16, [100, 0, 64, 63, 500, 31], BF)          # pages for the second token too
    q, k, v = (t[:, :1] for t in new)
    rope = nn.RotaryEmbedding(128, device="cuda")
    other, table2, at2, c2, (q2, k2, v2) = batch(4, 2, 4, 4, 64, 24, [700, 3, 64, 90], F16, prefix=0)
    rope2 = nn.RotaryEmbedding(32, interleaved=True, device="cuda")

    def step(cache, rope, k, v, table, at, q):
        return cache.Attend(cache.Append(k, v, table, at, rotary=rope, q=q), table, at, shared_pages=25 if table.shape[0] == 70 else 0)

    # a batch over its shared prefix, which two kernels take side by side, and a third joins
    wide, table3, at3, c3, new = batch(70, 2, 4, 1, 64, 16, [400 + i for i in range(70)], BF, prefix=25)
    q3, k3, v3 = (t[:, :1] for t in new)
    args = (cache, rope, k, v, table, at, q), (other, rope2, k2, v2, table2, at2, q2), (wide, rope2, k3, v3, table3, at3, q3)
    side = [torch.cuda.Stream() for _ in args]
    graphs, outs = [], []
    for s, a in zip(side, args):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(*a)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(step(*a))
        graphs.append(g)
    for shift, times in ((0, 20), (1, 1), (-1, 1), (1, 20)):            # (once, too: nothing of the replay before may be left)
        at += shift
        at3 += shift
        torch.cuda.synchronize()
        for _ in range(times):
            for s, g in zip(side, graphs):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for a, out in zip(args, outs):
            turned_q = a[0].Append(a[2], a[3], a[4], a[5], rotary=a[1], q=a[6])
            close(out, attended(a[0], turned_q, a[4], a[5], None))


def test_refusals():
    cache = nn.KVCache(4, 16, 2, 64, dtype=BF, device="cuda")
    k, q = torch.zeros(2, 1, 2, 64, device="cuda", dtype=BF), torch.zeros(2, 1, 4, 64, device="cuda", dtype=BF)
    table, at = torch.zeros(2, 1, device="cuda", dtype=torch.int32), torch.zeros(2, device="cuda", dtype=torch.int32)
    rope = nn.RotaryEmbedding(64)                                       # its frequencies are on the CPU
    with pytest.raises(ValueError):
        rope(q)
    with pytest.raises(ValueError):
        cache.Append(k, k, table, at, rotary=rope)
    with pytest.raises(ValueError):
        cache.Append(k, k, table, at.cpu())
    with pytest.raises(TypeError):
        cache.Attend(q.cpu(), table, at)
    with pytest.raises(TypeError):
        nn.KVCache(4, 16, 2, 64, dtype=torch.float64, device="cuda")
    with pytest.raises(TypeError):
        nn.RotaryEmbedding(64, device="cuda")(q.double())
    with pytest.raises(ValueError):
        nn.KVCache(4, 16, 2, 12, dtype=BF, device="cuda")               # rows of 24 bytes
    wide = nn.KVCache(4, 16, 1, 136, dtype=BF, device="cuda")
    with pytest.raises(ValueError):
        wide.Attend(torch.zeros(2, 1, 1, 136, device="cuda", dtype=BF), table, at)


# ------------------------------------------------------------------------------------------------------------------ layers and models
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("inter", [False, True])
def test_attention_layer_with_rotary(dtype, inter):
    """Forward, gradients, masks and pieces from a cache, against the layer in fp64 on the CPU.  Every result is a chain of a few roundings of values
    of about the result's size: eight of them, at the size of its largest value, are allowed.  In fp32 the sums' own errors are no smaller than that: a
    sum of n products is off by up to n 2^-24 of its terms' magnitudes, which add up to at least the result; n is 256 here (columns; 140 rows in the
    gradients of weights), where in 16 bits it hides behind the rounding of the result."""
    import copy
    torch.manual_seed(3)
    mha = nn.MultiHeadAttention(256, 4, rotary=nn.RotaryEmbedding(48, interleaved=inter), dtype=dtype, device="cuda")
    mha = mha.to("cuda")                                                # the frequencies follow
    exact = copy.deepcopy(mha).cpu().double()
    x = torch.randn(2, 70, 256, device="cuda").to(dtype).requires_grad_()
    x64 = x.detach().cpu().double().requires_grad_()
    dy = torch.randn(2, 70, 256, device="cuda").to(dtype)

    def near(got, want):
        err = float((got.detach().cpu().double() - want).abs().max())
        assert err <= (8 + (256 if dtype == F32 else 0)) * half(dtype) * float(want.detach().abs().max()), (err, float(want.detach().abs().max()))

    y, want = mha(x, causal=True), exact(x64, causal=True)
    near(y, want)
    params, params64 = list(mha.parameters()), list(exact.parameters())
    for g, w in zip(torch.autograd.grad(y, [x, *params], dy), torch.autograd.grad(want, [x64, *params64], dy.cpu().double())):
        if float(w.abs().max()) > 1e-9:                                 # (the key projection's bias has none)
            near(g, w)
    with torch.no_grad():
        near(mha.ForwardMasked(x, causal=True), want)
        cache = nn.KVCache(6, 32, 4, 64, dtype=dtype, device="cuda")
        table, at, outs = torch.tensor([[3, 0, 4], [1, 2, 5]], device="cuda", dtype=torch.int32), torch.zeros(2, device="cuda", dtype=torch.int32), []
        for piece in x.split([40, 1, 1, 28], 1):
            outs.append(mha.ForwardCached(piece, cache, table, at))
            at += piece.shape[1]
        near(torch.cat(outs, 1), want)


def test_model_steps_in_a_graph():
    """A step of a model captured once and replayed token by token, against the whole sequence at once in fp64 on the CPU."""
    import copy
    from gonn_b200.models import GPT
    torch.manual_seed(4)
    model = GPT(vocab=61, d_model=128, n_layers=2, n_heads=2, d_ff=256, max_seq=64, rotary=dict(scaling="linear", factor=2.0), device="cuda")
    ids = torch.randint(0, 61, (3, 20), device="cuda")
    with torch.no_grad():
        want = copy.deepcopy(model).cpu().double()(ids.cpu())
        whole = float((model(ids).cpu().double() - want).abs().max())
        caches = model.Caches(6, 16)
        table, at = torch.arange(6, device="cuda", dtype=torch.int32).view(3, 2), torch.zeros(3, device="cuda", dtype=torch.int32)
        first = model.Step(ids[:, :12], caches, table, at)
        at += 12
        token = ids[:, 12:13].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            model.Step(token, caches, table, at)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = model.Step(token, caches, table, at)
            at += 1
        outs = [first]
        for t in range(12, 20):
            token.copy_(ids[:, t:t + 1])
            graph.replay()
            outs.append(logits.clone())
        steps = float((torch.cat(outs, 1).cpu().double() - want).abs().max())
    # two ways through the same fp32 products: neither is off by much more than the other
    assert steps <= 4 * whole + 2.0 ** -20 * float(want.abs().max()), (steps, whole)


def test_blocks_with_rotary_are_not_evaluated_without_it():
    """The native evaluation of a block knows no rotation and leaves such blocks alone."""
    from gonn_b200.models import GPT
    from gonn_b200.nn import block
    for rotary in (None, True):
        model = GPT(vocab=31, d_model=128, n_layers=1, n_heads=2, d_ff=256, max_seq=32, rotary=rotary, dtype=BF, device="cuda")
        x = torch.randn(1, 20, 128, device="cuda").to(BF)
        with torch.no_grad():
            assert (block.evaluate(x, *model.layers[0]._parts()) is None) == (rotary is not None)
            ids = torch.randint(0, 31, (1, 20), device="cuda")
            taped = None
            with torch.enable_grad():
                taped = model(ids).detach()
            # two ways through the same layers in bf16: sixteen roundings, at the size of the largest logit
            assert float((model(ids).double() - taped.double()).abs().max()) <= 16 * half(BF) * float(taped.double().abs().max())


def test_samples_share_the_prompt():
    """Continuations of one prompt, in bf16: the first token of every sample is the prompt's, and equal draws stay equal."""
    from gonn_b200.models import GPT
    torch.manual_seed(5)
    model = GPT(vocab=61, d_model=128, n_layers=2, n_heads=2, d_ff=256, max_seq=512, rotary=True, dtype=BF, device="cuda")
    ids = torch.randint(0, 61, (1, 150), device="cuda")
    out = model.Generate(ids, 6, samples=80, page_size=16)
    assert out.shape == (80, 156) and torch.equal(out, out[:1].expand(80, -1)) and torch.equal(out[:, :150], ids.expand(80, -1))


def test_steps_behind_the_last_learned_position():
    """Reported as ``forward`` reports them; tokens that do not count may lie there."""
    from gonn_b200.models import GPT
    torch.manual_seed(6)
    model = GPT(vocab=31, d_model=128, n_layers=1, n_heads=2, d_ff=64, max_seq=8, device="cuda")
    ids = torch.randint(0, 31, (2, 12), device="cuda")
    table, at = torch.arange(6, device="cuda", dtype=torch.int32).view(2, 3), torch.zeros(2, device="cuda", dtype=torch.int32)
    with torch.no_grad():
        model(ids)
        assert lib.read_status()[0] == 5
        model.Step(ids, model.Caches(6, 4), table, at)
        assert lib.read_status()[0] == 5
        model.Step(ids[:, :1], model.Caches(6, 4), table, at + 8)
        assert lib.read_status()[0] == 5
        model.Step(ids, model.Caches(6, 4), table, at, counts=torch.tensor([8, 3], device="cuda", dtype=torch.int32))
        lib.assert_status_ok()


def test_positions_changed_behind_the_tape():
    rope = nn.RotaryEmbedding(64, device="cuda")
    x, at = torch.randn(1, 3, 2, 64, device="cuda", requires_grad=True), torch.arange(3, device="cuda")
    y = rope(x, at)
    at += 3
    with pytest.raises(RuntimeError):
        y.sum().backward()
    rope(x).sum().backward()                                            # without positions: 0, 1, ...
    close(x.grad, turned(torch.ones_like(x), torch.arange(3, device="cuda"), rope, back=True))


def test_steps_of_a_layer_under_a_tape_are_refused():
    mha = nn.MultiHeadAttention(128, 2, dtype=BF, device="cuda")
    cache, x = nn.KVCache(1, 16, 2, 64, dtype=BF, device="cuda"), torch.randn(1, 1, 128, device="cuda").to(BF)
    table, at = torch.zeros(1, 1, device="cuda", dtype=torch.int32), torch.zeros(1, device="cuda", dtype=torch.int32)
    for need in (mha.qproj.weight, mha.kproj.weight, mha.vproj.bias):
        for p in mha.parameters():
            p.requires_grad_(p is need)
        with pytest.raises(RuntimeError):
            mha.ForwardCached(x, cache, table, at)
        with torch.no_grad():
            mha.ForwardCached(x, cache, table, at)
    for p in mha.parameters():
        p.requires_grad_(p is mha.outproj.weight)                       # behind the cache: a gradient like any other
    mha.ForwardCached(x, cache, table, at).sum().backward()
    assert mha.outproj.weight.grad is not None


def test_caches_in_tensors_that_need_a_gradient():
    q, k = torch.randn(1, 1, 2, 8, device="cuda"), torch.randn(1, 1, 2, 8, device="cuda")
    table, at = torch.zeros(1, 1, device="cuda", dtype=torch.int32), torch.zeros(1, device="cuda", dtype=torch.int32)
    for which in range(2):
        tensors = [torch.zeros(1, 2, 4, 8, device="cuda") for _ in range(2)]
        cache = nn.KVCache.Over(*tensors)
        tensors[which].requires_grad_()
        for call in (lambda: cache.Append(k, k, table, at), lambda: cache.Attend(q, table, at)):
            with pytest.raises(RuntimeError, match="under torch.no_grad"):
                call()
            with torch.no_grad():
                call()


def ended(B, T, H, kv, D, page, prefix, ends, dtype, counts, seed=0):
    """A batch whose sequences share their first `prefix` pages and end (their last tokens that count included) at `ends`, inside them too; NaN in every
    row behind the last sequence's end."""
    g = torch.Generator("cuda").manual_seed(seed)
    columns = max(prefix, -(-max(ends) // page)) + 1
    order = torch.randperm(prefix + B * (columns - prefix), generator=g, device="cuda").int()
    table = torch.empty(B, columns, dtype=torch.int32, device="cuda")
    table[:, :prefix] = order[:prefix]
    table[:, prefix:] = order[prefix:].view(B, -1)
    kc, vc = (torch.full((order.numel(), kv, page, D), math.nan, device="cuda", dtype=dtype) for _ in range(2))
    for b, n in enumerate(ends):
        p = torch.arange(n, device="cuda")
        pages = table[b].long()[p // page]
        for t in (kc, vc):
            t[pages, :, p % page] = torch.randn(n, kv, D, generator=g, device="cuda").to(dtype)
    c = torch.tensor([T] * B if counts is None else counts, dtype=torch.int32, device="cuda")
    q = torch.randn(B, T, H, D, generator=g, device="cuda").to(dtype)
    return nn.KVCache.Over(kc, vc), q, table, torch.tensor(ends, dtype=torch.int32, device="cuda") - c, None if counts is None else c


ENDED = [(3, 1, 4, 2, 64, 16, 4, [10, 40, 50], None), (70, 1, 8, 1, 128, 32, 3, [33 + i % 40 for i in range(70)], None),
         (5, 3, 4, 2, 72, 24, 2, [3, 30, 47, 20, 48], [3, 0, 1, 2, 3]), (20, 2, 3, 1, 40, 7, 11, [50 + i for i in range(20)], None),
         (2, 1, 2, 1, 128, 64, 1, [5, 63], None), (80, 1, 1, 1, 64, 64, 2, [0] * 40 + [100] * 40, [0] * 40 + [1] * 40),
         (33, 1, 8, 2, 64, 64, 40, [2500 + i for i in range(33)], None), (4, 17, 4, 1, 128, 16, 30, [470, 471, 300, 479], None)]


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("B,T,H,kv,D,page,prefix,ends,counts", ENDED)
def test_sequences_that_end_inside_the_shared_pages(dtype, B, T, H, kv, D, page, prefix, ends, counts):
    cache, q, table, at, c = ended(B, T, H, kv, D, page, prefix, ends, dtype, counts)
    close(cache.Attend(q, table, at, counts=c, shared_pages=prefix), attended(cache, q, table, at, c))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B", [3, 70])
def test_infinite_values_that_a_shorter_sequence_does_not_have(dtype, B):
    """A value of the shared pages behind the end of the first sequence is infinite: the others' alone."""
    cache, q, table, at, c = ended(B, 1, 4, 1, 64, 16, 6, [40] + [90 + i for i in range(B - 1)], dtype, None)
    cache.Values[int(table[0, 3]), :, 2] = math.inf
    out = cache.Attend(q, table, at, shared_pages=6)
    want, tol = attended(cache, q[:1], table, at[:1], None)
    close(out[:1], (want, tol))
    assert bool((out[1:] == math.inf).all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_scales_that_fp32_does_not_hold(dtype):
    cache, table, at, c, (q, k, v) = batch(2, 2, 2, 1, 64, 16, [300, 40], dtype)
    cache.Append(k, v, table, at)
    for scale in (1e-50, 9e-38, 1.1e38, 1e300):
        with pytest.raises(ValueError):
            cache.Attend(q, table, at, scale=scale)
    close(cache.Attend(q, table, at, scale=1e-37), attended(cache, q, table, at, c, 1e-37))       # the mean of what a token sees


def test_tangents():
    fw = torch.autograd.forward_ad
    rope = nn.RotaryEmbedding(24, interleaved=True, amplitude=1.5, device="cuda")
    x, dx = torch.randn(2, 2, 9, 3, 40, device="cuda").unbind(0)
    at = torch.randint(0, 5000, (2, 9), device="cuda")
    for grad in (False, True):
        with fw.dual_level():
            y, dy = fw.unpack_dual(rope(fw.make_dual(x.clone().requires_grad_(grad), dx), at))
        close(y.detach(), turned(x, at, rope))
        close(dy.detach(), turned(dx, at, rope))


def test_angles_in_fp32():
    """Cosine and sine themselves (pairs of 1 and 0): off by the angle's pi 2^-27 and what it is cut off, 2.4e-8 together, and a unit in the last
    place of the function, at most 2^-23 of the value."""
    rope = nn.RotaryEmbedding(64, device="cuda")
    x = torch.zeros(1, 20000, 1, 64, device="cuda")
    x[..., :32] = 1
    for start in (0, 100003):
        at = torch.arange(20000, device="cuda") + start
        y = rope(x, at)[0, :, 0].double()
        angle = at.double()[:, None] * torch.tensor(rope._w, dtype=torch.float64, device="cuda")
        want = torch.cat((torch.cos(angle), torch.sin(angle)), -1)
        # (and p w in fp64, 2^-52 of it on either side)
        worst = ((y - want).abs() - 2.0 ** -23 * want.abs() - float(at[-1]) * 2.0 ** -51).max()
        assert float(worst) <= 2.4e-8


# More row tiles of all heads and sequences than the SMs (148) or two rounds of them (296) hold: their results leave without the joining kernel, in one group of
# runs or in several whose last one is smaller; the last one's table is so long that a group is one run.
MANY = [(4, 300, 16, 8, 128, 64, [0, 77, 500, 64], [300, 13, 0, 299], 0), (5, 300, 14, 14, 64, 24, [3, 0, 100, 23, 24], None, 0),
        (4, 290, 24, 12, 72, 7, [40, 0, 5, 6], [290, -3, 500, 129], 0), (3, 700, 23, 23, 128, 64, [0, 130, 63], None, 0),
        (7, 257, 34, 34, 64, 64, [0, 1, 2, 300, 64, 65, 127], [257, 256, 0, 1, 128, 129, 257], 0), (5, 129, 48, 48, 128, 24, [9, 0, 48, 400, 24], [129, 1, 128, 0, 77], 0),
        (2, 200, 80, 80, 64, 16, [30, 500], None, 2 ** 18)]


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("B,T,H,kv,D,page,lengths,counts,room", MANY)
def test_attend_more_rows_than_a_round(dtype, B, T, H, kv, D, page, lengths, counts, room):
    tiles = -(-T * (H // kv) // 128) * kv * B
    assert tiles > 148
    cache, table, at, c, (q, k, v) = batch(B, T, H, kv, D, page, lengths, dtype, counts=counts)
    if room:
        table = torch.cat((table, torch.full((B, room // page - table.shape[1]), -7, dtype=torch.int32, device="cuda")), 1)
    cache.Append(k, v, table, at, counts=c)
    before = lib.kernel_count
    out = cache.Attend(q, table, at, counts=c)
    assert lib.kernel_count == before + 1                               # no joining kernel
    close(out, attended(cache, q, table, at, c))


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("B,T,H,kv,D,page,prefix,counts", [(310, 2, 32, 8, 64, 64, 4, None), (310, 4, 64, 8, 128, 24, 3, [i % 6 - 1 for i in range(310)])])
def test_shared_more_rows_than_a_round(dtype, B, T, H, kv, D, page, prefix, counts):
    """The prefix's row tiles alone are more than a round."""
    assert -(-B * T * (H // kv) // 128) * kv > 148
    cache, table, at, c, (q, k, v) = batch(B, T, H, kv, D, page, [prefix * page + i % 31 for i in range(B)], dtype, prefix=prefix, counts=counts)
    cache.Append(k, v, table, at, counts=c)
    close(cache.Attend(q, table, at, counts=c, shared_pages=prefix), attended(cache, q, table, at, c))


def test_rotary_given_to_a_layer_later():
    """The native evaluation of a block leaves a layer alone whose rotary positions were assigned."""
    from gonn_b200.models import GPT
    from gonn_b200.nn import block
    model = GPT(vocab=31, d_model=128, n_layers=1, n_heads=2, d_ff=256, max_seq=32, dtype=BF, device="cuda")
    x = torch.randn(1, 20, 128, device="cuda").to(BF)
    with torch.no_grad():
        assert block.evaluate(x, *model.layers[0]._parts()) is not None
        model.layers[0].attn.rotary = nn.RotaryEmbedding(64, device="cuda")
        assert block.evaluate(x, *model.layers[0]._parts()) is None


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("B,T,H,kv,D,page,prefix,ends,counts", [
    (3, 6, 3, 1, 72, 1, 1, [0, 2, 9], None), (8, 3, 8, 2, 8, 7, 1, [2, 1, 4, 5, 0, 2, 1, 0], [0, 3, 1, 2, 2, 3, 2, 1]), (2, 3, 6, 3, 48, 16, 2, [1, 42], None),
    (5, 6, 16, 2, 64, 8, 3, [24, 3, 40, 24, 25], None), (14, 30, 4, 2, 48, 24, 1, [27, 26, 23] * 4 + [48, 5], None), (40, 4, 8, 1, 128, 64, 2, [3, 130] * 20, None)])
def test_tokens_in_front_of_the_first_position(dtype, B, T, H, kv, D, page, prefix, ends, counts):
    """Lengths below zero: tokens in front of position 0 see nothing, behind shared pages too."""
    cache, q, table, at, c = ended(B, T, H, kv, D, page, prefix, ends, dtype, counts)
    want = attended(cache, q, table, at, c)
    assert bool((at < 0).any())
    close(cache.Attend(q, table, at, counts=c, shared_pages=prefix), want)
    close(cache.Attend(q, table, at, counts=c), want)
