"""Microscaled kernels against the CPU oracle and against 64 bits.

Quantised codes have to be equal: rounding is part of the format.  Products are first taken of values whose sums the fp32
accumulator holds exactly (whole numbers times powers of two, every partial sum below 2^24 units), so that results have to be
equal as well; random operands follow with tolerances that count roundings."""
import ctypes
import math

import pytest
import torch

from gonn_b200 import lib as _l
from gonn_b200 import quant as Q
from gonn_b200.nn import Linear, RMSNorm

pytestmark = pytest.mark.gpu

FORMATS = ["mxfp8", "mxfp4"]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
DEV = "cuda"


def wild(*shape, dtype):
    """Values over many magnitudes, zeros and ties among them."""
    t = torch.randn(*shape) * torch.exp2(torch.randint(-12, 12, shape[:-1] + (1,)).float())
    t = torch.where(torch.rand(shape) < 0.1, torch.zeros(()), t)
    t = torch.where(torch.rand(shape) < 0.3, torch.round(t * 8) / 8, t)
    return t.to(dtype)


def equal(q, want):
    assert torch.equal(q.Data.cpu(), want.Data)
    assert torch.equal(q.ScaleCodes().cpu(), want.ScaleCodes())


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 31), (2, 32), (3, 33), (5, 127), (129, 130), (7, 256), (130, 257), (33, 1000), (300, 2048), (1, 8192), (2, 3, 77)])
def test_quantize_is_the_oracle(format, dtype, shape, status_ok):
    t = wild(*shape, dtype=dtype)
    q = Q.QuantizeMX(t.to(DEV), format)
    want = Q.QuantizeMX(t, format)
    equal(q, want)
    # scales behind the last block are zeros
    blocks, rows = -(-shape[-1] // 32), want.Data.shape[0]
    s = q.Scales.cpu().view(-(-rows // 128), -1, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-(-rows // 128) * 128, -1)
    assert not s[:rows, blocks:].any()
    for out in DTYPES:
        assert torch.equal(Q.DequantizeMX(q, out).cpu(), Q.DequantizeMX(want, torch.float64).to(out))


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_extremes(format, dtype, status_ok):
    top = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).smallest_normal
    sub = tiny * torch.finfo(dtype).eps
    rows = [[0.0], [top, -top, 1.0], [tiny, -tiny / 2, sub], [sub, -sub, 3 * sub, 0.0], [math.inf, 1.0, 2.0], [-math.inf], [math.nan, 1.0], [1.0] * 32 + [math.nan] + [2.0] * 40,
            [-0.0, 0.0, -1e-7], [tiny * 2 ** i for i in range(12)]]
    t = torch.zeros(len(rows), 80, dtype=dtype)
    for i, r in enumerate(rows):
        t[i, :len(r)] = torch.tensor(r, dtype=torch.float64).to(dtype)
    q, want = Q.QuantizeMX(t.to(DEV), format), Q.QuantizeMX(t, format)
    assert torch.equal(q.ScaleCodes().cpu(), want.ScaleCodes())
    for out in DTYPES:
        a, b = Q.DequantizeMX(q, out).cpu(), Q.DequantizeMX(want, torch.float64).to(out)
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(0, 1, 1), b.nan_to_num(0, 1, 1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("K,pitch", [(100, 100), (100, 101), (97, 131), (1003, 1003)])
def test_quantize_views(dtype, offset, K, pitch, status_ok):
    """Rows at any address and distance; what lies before, between and behind them is not taken."""
    R = 9
    flat = torch.full((offset + R * pitch + 16,), float("nan"), dtype=dtype)
    view = flat[offset:offset + R * pitch].as_strided((R, K), (pitch, 1), offset)
    view.copy_(wild(R, K, dtype=dtype))
    d = flat.to(DEV)
    dv = d.as_strided((R, K), (pitch, 1), offset)
    for format in FORMATS:
        equal(Q.QuantizeMX(dv, format), Q.QuantizeMX(view, format))
    q, qt = Q.QuantizeMXPair(dv)
    equal(q, Q.QuantizeMX(view))
    equal(qt, Q.QuantizeMX(view.t()))
    equal(Q.QuantizeMX(dv.t()), Q.QuantizeMX(view.t()))
    w = torch.rand(K) + 0.5
    a, _ = Q.AddRMSNormMX(dv, dv, w.to(DEV))
    b, _ = Q.AddRMSNormMX(dv.contiguous(), dv.contiguous(), w.to(DEV))
    assert torch.equal(a.Data, b.Data) and torch.equal(a.ScaleCodes(), b.ScaleCodes())


def test_quantize_broadcast_rows(status_ok):
    row = torch.randn(64, device=DEV)
    equal(Q.QuantizeMX(row.expand(5, 64)), Q.QuantizeMX(row.cpu().expand(5, 64)))
    column = torch.randn(5, 1, device=DEV)
    equal(Q.QuantizeMX(column.expand(5, 64)), Q.QuantizeMX(column.cpu().expand(5, 64)))
    equal(Q.QuantizeMX(column), Q.QuantizeMX(column.cpu()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (31, 33), (32, 128), (128, 128), (129, 127), (300, 1000), (1001, 200), (4, 2048)])
def test_quantize_pair(dtype, shape, status_ok):
    t = wild(*shape, dtype=dtype)
    q, qt = Q.QuantizeMXPair(t.to(DEV))
    equal(q, Q.QuantizeMX(t))
    equal(qt, Q.QuantizeMX(t.t()))


def nearly(q, y, ulps):
    """Whether codes are those of a y that was off by `ulps` roundings of fp32 at most: each value is the nearest number, up to that error
    and half a step of its block."""
    K = y.shape[-1]
    fp8 = q.Format == "mxfp8"
    s = torch.exp2(q.ScaleCodes().double() - 127).repeat_interleave(32, 1)[:, :K]
    v = Q.DequantizeMX(q, torch.float32).double().cpu().reshape(y.shape)
    m = (y / s).abs()
    # the largest magnitude lies where the scale puts it, up to the error of y
    big = torch.nn.functional.pad(m, (0, -K % 32)).view(m.shape[0], -1, 32).amax(2)
    lo, hi = (256, 512) if fp8 else (4, 8)
    rel = ulps * 2.0 ** -24
    assert bool(((big >= lo * (1 - rel)) & (big <= hi * (1 + rel)) | (big == 0)).all())
    # half a step: 2^-4 or 2^-2 of the power of two below the value; what is above the largest number saturates
    mant, least, top = (3, -6, 448.0) if fp8 else (1, 0, 6.0)
    e = (torch.frexp(m).exponent - 1).clamp(min=least)
    half = torch.exp2((e - mant - 1).double())
    allowed = torch.where(m > top, (m - top).abs() + m * rel, half + m * rel)
    assert bool(((v / s - y / s).abs() <= allowed * (1 + 1e-9)).all())


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 40), (1, 255), (9, 256), (301, 257), (700, 768), (5, 1000), (301, 1024), (2, 2048), (400, 2050), (3, 4100), (2, 8192), (2, 10000), (3, 40000)])
@pytest.mark.parametrize("residual", [True, False])
def test_norm(format, dtype, shape, residual, status_ok):
    x, r = torch.randn(shape).to(dtype), torch.randn(shape).to(dtype)
    w = (torch.rand(shape[-1]) + 0.5).to(dtype)
    q, h = Q.AddRMSNormMX(x.to(DEV), r.to(DEV) if residual else None, w.to(DEV), 1e-6, format)
    total = x.double() + (r.double() if residual else 0)
    if residual:
        assert torch.equal(h.cpu(), (x.float() + r.float()).to(dtype))
    y = total / torch.sqrt(total.square().mean(-1, keepdim=True) + 1e-6) * w.double()
    # roundings of y: the sum, its product with 1 / rms and with w (half a unit each), 1 / rms (half), and the sum of squares, whose error
    # enters by half: at most 2 ceil(K / 32) + 12 roundings of a thread's chain and the tree, K no larger than 32 values a thread
    # but for the widest rows
    chain = 32 if shape[-1] <= 32768 else shape[-1] / 1024 + 8
    nearly(cpu(q), y, 4 + chain / 2 + 12)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [520, 768, 2048, 2304, 4096, 8192])
def test_norm_of_many_rows(format, dtype, K, status_ok):
    """More than L2 keeps; a hundred of the rows are compared."""
    rows = (9 << 20) // K + 7
    x, r, w = torch.randn(rows, K, device=DEV).to(dtype), torch.randn(rows, K, device=DEV).to(dtype), (torch.rand(K, device=DEV) + 0.5).to(dtype)
    q, h = Q.AddRMSNormMX(x, r, w, 1e-6, format)
    assert torch.equal(h, (x.float() + r.float()).to(dtype))
    some = torch.cat((torch.arange(0, rows, rows // 98)[:98], torch.tensor([rows - 2, rows - 1])))
    total = x.cpu()[some].double() + r.cpu()[some].double()
    y = total / torch.sqrt(total.square().mean(-1, keepdim=True) + 1e-6) * w.cpu().double()
    part = Q.QTensorMX(q.Data.cpu()[some], Q.microscale._pack_scales(q.ScaleCodes().cpu()[some], int(format == "mxfp4")), format, (100, K))
    nearly(part, y, 4 + 16 + 12)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K", [(40000, 160), (8000, 776), (3000, 2304), (4100, 1003), (100, 20000), (600, 8200)])
def test_norm_codes_are_those_of_64_bits(format, dtype, rows, K, status_ok):
    """Millions of values, some of which lie within a rounding of fp32 of the border between two codes; and rows whose squares fp32 does not
    hold.  (fp64 on the device: its own error, some 1e-15, is a millionth of the distance at which a border was ever met.)"""
    x, r, w = torch.randn(rows, K, device=DEV).to(dtype), torch.randn(rows, K, device=DEV).to(dtype), (torch.rand(K, device=DEV) + 0.5).to(dtype)
    if dtype == torch.float32:
        x[1], r[1] = x[1] * 2.0 ** 70, r[1] * 2.0 ** 70
        x[2], r[2] = x[2] * 2.0 ** -70, r[2] * 2.0 ** -70
    eps = 0.0
    q, _ = Q.AddRMSNormMX(x, r, w, eps, format)
    total = x.double() + r.double()
    y = total / torch.sqrt(total.square().mean(-1, keepdim=True) + eps) * w.double()
    want = Q.microscale._quantize_ref(y.cpu(), int(format == "mxfp4"), (rows, K))
    equal(q, want)


def cpu(q):
    return Q.QTensorMX(q.Data.cpu(), q.Scales.cpu(), q.Format, q.Shape)


def test_norm_special_rows(status_ok):
    x = torch.randn(6, 96, device=DEV)
    x[1] = 0
    x[2, 5] = math.nan
    x[3, 40] = math.inf
    w = torch.ones(96, device=DEV)
    q, _ = Q.AddRMSNormMX(x, None, w)
    v = Q.DequantizeMX(q)
    assert not v[1].any() and torch.isnan(v[2]).all()
    # an infinite sum of squares: the finite values become 0, the infinite one NaN, and with it its block
    assert torch.isnan(v[3, 32:64]).all() and not v[3, :32].any() and not v[3, 64:].any()
    alone, _ = Q.AddRMSNormMX(x[4:5], None, w)
    assert torch.equal(Q.DequantizeMX(alone)[0], v[4])
    mixed, _ = Q.AddRMSNormMX(x.bfloat16(), None, w)             # fp32 weights of 16-bit rows
    same, _ = Q.AddRMSNormMX(x.bfloat16(), None, w.bfloat16())
    assert torch.equal(mixed.Data, same.Data)


def whole(rows, K, format):
    """Quantised whole numbers up to 4 (6) times 1, 2, 4 or 8 for each block: exact in the format."""
    t = torch.randint(-4, 5, (rows, K)).float()
    if format == "mxfp4":
        t = torch.where((t == 4) & (torch.rand(rows, K) < 0.5), torch.tensor(6.0), t)
    s = torch.exp2(torch.randint(0, 4, (rows, -(-K // 32))).float()).repeat_interleave(32, 1)[:, :K]
    return t * s


SHAPES = [(1, 1, 1), (1, 8, 32), (3, 5, 7), (2, 128, 128), (16, 130, 257), (17, 129, 300), (33, 64, 1000), (64, 384, 256), (65, 300, 1000), (128, 256, 512), (129, 257, 640),
          (300, 520, 1000), (1, 2048, 4096), (4, 300, 4096), (40, 100, 4096), (100, 1000, 4000)]
#: 37 tiles of 256 x 256 and more run as pairs of CTAs; 74 pairs at a time
PAIR_SHAPES = [(1700, 1700, 96), (1601, 1543, 333), (2560, 2560, 520), (2600, 2330, 1024), (9473, 256, 64), (256, 9999, 300)]


def product(M, N, K, format, dtype, bias, act):
    a, b = whole(M, K, format), whole(N, K, format)
    qa, qb = Q.QuantizeMX(a.to(DEV), format), Q.QuantizeMX(b.to(DEV), format)
    v = torch.randint(-100, 100, (N,)).to(dtype) if bias else None
    y = Q.MatMulMX(qa, qb, None if v is None else v.to(DEV), dtype, act)
    _l.assert_status_ok()
    want = a.to(DEV, torch.float64) @ b.to(DEV, torch.float64).T
    if bias:
        want = want + v.to(DEV, torch.float64)
    if act == "relu":
        want = want.relu()
    return y, want.to(dtype)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_matmul_exact(format, M, N, K, status_ok):
    for dtype, bias, act in ((torch.float32, False, None), (torch.bfloat16, True, None), (torch.float16, True, "relu")):
        y, want = product(M, N, K, format, dtype, bias, act)
        assert torch.equal(y, want), (dtype, (y.double() - want.double()).abs().max())


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("M,N,K", PAIR_SHAPES)
def test_matmul_exact_pairs(format, M, N, K, status_ok):
    for dtype, bias, act in ((torch.float32, True, None), (torch.bfloat16, True, "relu"), (torch.float16, False, None)):
        y, want = product(M, N, K, format, dtype, bias, act)
        assert torch.equal(y, want), (dtype, (y.double() - want.double()).abs().max())


def off(y, want):
    return ((y.double() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("act", [None, "gelu", "geluexact"])
@pytest.mark.parametrize("M,N,K", [(5, 700, 1000), (1000, 2500, 700), (3000, 1111, 4096)])
def test_matmul_random(format, act, M, N, K, status_ok):
    """fp32 results: the tensor core truncates a sum at the accumulator's last bit once an instruction (32 or 64 of K), at most
    K / 32 times 2^-23 of the largest partial sum, for random signs of its root; 16-bit results are roundings of those."""
    a, b = torch.randn(M, K, device=DEV), torch.randn(N, K, device=DEV) / math.sqrt(K)
    qa, qb, bias = Q.QuantizeMX(a, format), Q.QuantizeMX(b, format), torch.randn(N, device=DEV)
    want = Q.DequantizeMX(qa).double() @ Q.DequantizeMX(qb).double().T + bias.double()
    if act:
        want = torch.nn.functional.gelu(want, approximate="tanh" if act == "gelu" else "none")
    # the hardware's tanh has an error of 2^-11, and erff of a unit
    most = (K / 32 + 2) * 2.0 ** -23 + (2.0 ** -10.5 if act == "gelu" else 0)
    assert off(Q.MatMulMX(qa, qb, bias, torch.float32, act), want) <= most
    assert off(Q.MatMulMX(qa, qb, bias, torch.float16, act), want) <= most + 2.0 ** -11
    assert off(Q.MatMulMX(qa, qb, bias, torch.bfloat16, act), want) <= most + 2.0 ** -8


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("M,N", [(3, 200), (2000, 2100)])
def test_matmul_nan_stays_in_its_rows(format, M, N, status_ok):
    K = 333
    a, b = torch.randn(M, K), torch.randn(N, K)
    a[1, 70] = math.nan
    b[130, 5] = math.inf
    y = Q.MatMulMX(Q.QuantizeMX(a.to(DEV), format), Q.QuantizeMX(b.to(DEV), format))
    nan = torch.zeros(M, N, dtype=torch.bool)
    nan[1] = nan[:, 130] = True
    assert torch.equal(torch.isnan(y).cpu(), nan)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("M,N", [(5, 140), (2000, 2100)])
def test_scales_of_rows_that_are_not_there(format, M, N, status_ok):
    """Scales behind the last row hold anything, NaN's code too."""
    K = 200
    a, b = Q.QuantizeMX(whole(M, K, format).to(DEV), format), Q.QuantizeMX(whole(N, K, format).to(DEV), format)
    y = Q.MatMulMX(a, b)
    for q in (a, b):
        rows = q.Data.shape[0]
        s = q.Scales.view(-(-rows // 128), -1, 32, 4, 4).permute(0, 3, 2, 1, 4)
        at = torch.arange(s.shape[0] * 128, device=DEV).view(s.shape[0], 4, 32)[:, :, :, None, None].expand(s.shape)
        s[at >= rows] = 255
    assert torch.equal(Q.MatMulMX(a, b), y)


def test_products_of_extreme_scales(status_ok):
    """Scales at both ends: 2^-127 and above, sums that overflow."""
    a = torch.full((3, 32), 2.0 ** -120)
    b = torch.full((4, 32), 2.0 ** 100)
    y = Q.MatMulMX(Q.QuantizeMX(a.to(DEV)), Q.QuantizeMX(b.to(DEV)), dtype=torch.float32)
    assert torch.equal(y.cpu(), torch.full((3, 4), 32 * 2.0 ** -20))
    y = Q.MatMulMX(Q.QuantizeMX(b.to(DEV)), Q.QuantizeMX(b.to(DEV)), dtype=torch.float32)
    assert torch.isinf(y).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape,N", [((1, 33), 17), ((7, 64), 128), ((2, 50, 300), 200), ((1001, 1000), 520), ((2100, 768), 2304)])
def test_train_linear(dtype, shape, N, status_ok):
    K = shape[-1]
    x = torch.randn(shape, device=DEV).to(dtype).requires_grad_()
    w = (torch.randn(N, K, device=DEV) / math.sqrt(K)).to(dtype).requires_grad_()
    b = torch.randn(N, device=DEV).to(dtype).requires_grad_()
    dy = torch.randn(*shape[:-1], N, device=DEV).to(dtype)
    y = Q.TrainLinearMX(x, w, b)
    got = (y, *torch.autograd.grad(y, (x, w, b), dy))

    def rounded(t):
        return Q.DequantizeMX(Q.QuantizeMX(t)).double()

    x2, g = x.detach().reshape(-1, K), dy.reshape(-1, N)
    want = (rounded(x2) @ rounded(w).T + b.detach().double(), rounded(g) @ rounded(w.detach().T).T, rounded(g.T) @ rounded(x2.T).T, g.double().sum(0))
    for a, e, length in zip(got, want, (K, N, x2.shape[0], x2.shape[0])):
        assert a.dtype == dtype
        assert off(a.detach().reshape(e.shape), e) <= (length / 32 + 4) * 2.0 ** -23 + torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 5, 3), (1, 300, 1000), (2, 128, 32), (7, 2100, 700), (16, 130, 4097), (16, 64, 8192), (5, 40000, 96)])
def test_few_rows_are_quantised_within_the_product(format, dtype, M, N, K, status_ok):
    """The same bits as quantisation and product one after the other: rows of any address and pitch."""
    w, bias = Q.QuantizeMX(torch.randn(N, K, device=DEV), format), torch.randn(N, device=DEV)
    for offset, pitch in ((0, K), (1, K), (3, K + 5), (8, K + 8)):
        flat = torch.full((offset + M * pitch + 16,), float("nan"), dtype=dtype, device=DEV)
        x = flat.as_strided((M, K), (pitch, 1), offset)
        x.copy_(wild(M, K, dtype=dtype))
        for act in (None, "relu"):
            assert torch.equal(Q.LinearMX(x, w, bias, act), Q.MatMulMX(Q.QuantizeMX(x, format), w, bias, dtype, act))
    x = wild(M, K, dtype=dtype)
    x[0, K // 2] = math.inf
    y = Q.LinearMX(x.to(DEV), w)
    assert torch.isnan(y[0]).all() and not torch.isnan(y[1:]).any()


@pytest.mark.parametrize("format", FORMATS)
def test_loads_that_land_in_any_order(format, status_ok):
    """More weights than L2 holds, rows of C in tiles that start within a scale piece: loads wait for memory and overtake one another."""
    M, N, K = 100, 50304, 3000
    a, b = (torch.randint(-3, 4, (rows, K), device=DEV).float() * torch.exp2(torch.randint(0, 4, (rows, K // 8 // 3), device=DEV).float()).repeat_interleave(24, 1) for rows in (M, N))
    qa, qb = Q.QuantizeMX(a, format), Q.QuantizeMX(b, format)
    want = (Q.DequantizeMX(qa).double() @ Q.DequantizeMX(qb).double().T).float()
    for kind in (0, 32, 64):
        for splits in (1, 2):
            _l.lib().gb_mx_tune(kind, splits if kind else 0)
            try:
                for _ in range(3):
                    y = Q.MatMulMX(qa, qb, None, torch.float32)
                    _l.assert_status_ok()
                    assert torch.equal(y, want)
            finally:
                _l.lib().gb_mx_tune(0, 0)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("kind", [1, 2, 32, 64, 128])
@pytest.mark.parametrize("splits", [1, 2, 3, 5, 8])
def test_every_way_of_a_product(format, kind, splits, status_ok):
    """Either kernel with any number of slices of K, and tiles of any number of rows, give the exact sums; slices that K does not have are none."""
    for M, N, K in ((70, 264, 1500), (300, 512, 4100), (3, 40, 64), (520, 1032, 700)):
        _l.lib().gb_mx_tune(kind, splits)
        try:
            for dtype, act in ((torch.float32, None), (torch.bfloat16, "relu")):
                y, want = product(M, N, K, format, dtype, True, act)
                assert torch.equal(y, want)
        finally:
            _l.lib().gb_mx_tune(0, 0)


def test_train_linear_broadcast_gradient(status_ok):
    """A gradient that is one value everywhere (y.sum()), a gradient of strided rows, and an input that appears twice."""
    x = torch.randint(-4, 5, (70, 64), device=DEV).float().requires_grad_()
    w = torch.randint(-4, 5, (40, 64), device=DEV).float().requires_grad_()
    dx, dw = torch.autograd.grad(Q.TrainLinearMX(x, w).sum(), (x, w))
    assert torch.equal(dx, w.detach().sum(0).expand(70, 64)) and torch.equal(dw, x.detach().sum(0).expand(40, 64))
    dy = torch.randint(-4, 5, (70, 80), device=DEV).float()
    dx, dw = torch.autograd.grad(Q.TrainLinearMX(x, w), (x, w), dy[:, ::2])
    assert torch.equal(dx, dy[:, ::2] @ w) and torch.equal(dw, dy[:, ::2].T @ x)
    (both,) = torch.autograd.grad((Q.TrainLinearMX(x, w) + Q.TrainLinearMX(x, w)).sum(), x)
    assert torch.equal(both, 2 * w.detach().sum(0).expand(70, 64))


@pytest.mark.parametrize("format", FORMATS)
def test_block_of_layers(format, status_ok):
    """Norm, projection with activation, second projection, norm with the residual: as an evaluation runs them."""
    E, Fd, T = 256, 512, 37
    norm, up, down = RMSNorm(E), Linear(E, Fd, activation="gelu"), Linear(Fd, E)
    parts = [Q.MXRMSNorm(norm, format), Q.MXLinear(up, format), Q.MXLinear(down, format)]
    x, r = torch.randn(2, T, E), torch.randn(2, T, E)

    def go(device):
        n, u, d = (p.to(device) for p in parts)
        q, h = n(x.to(device), r.to(device))
        q2, h2 = n(d(u(q, torch.float32)), h)
        return u(q2, torch.float32), h, h2

    want = [t.clone() for t in go("cpu")]
    got = go(DEV)
    assert torch.equal(got[1].cpu(), want[1])
    # a value that moves to the next code is off by a step of it at most; few do
    assert off(got[2].cpu(), want[2].double()) < 1e-2 and off(got[0].cpu(), want[0].double()) < 3e-2


def test_streams_and_graphs(status_ok):
    w = Q.QuantizeMX(torch.randn(700, 512, device=DEV))
    big = Q.QuantizeMX(torch.randn(2048, 512, device=DEV))
    x = torch.randn(2000, 512, device=DEV, dtype=torch.bfloat16)
    few = torch.randn(3, 512, device=DEV, dtype=torch.bfloat16)
    weight = torch.ones(512, device=DEV, dtype=torch.bfloat16)

    def run(x, few):
        q, h = Q.AddRMSNormMX(x, x, weight)
        return Q.LinearMX(q, big), h, Q.LinearMX(few, w, act="relu"), Q.DequantizeMX(Q.QuantizeMX(few, "mxfp4"))

    want = run(x, few)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(run(x, few))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
    graph = torch.cuda.CUDAGraph()
    sx, sf = x.clone(), few.clone()
    with torch.cuda.graph(graph):
        out = run(sx, sf)
    for seed in (1, 2):
        torch.manual_seed(seed)
        sx.copy_(torch.randn_like(sx))
        sf.copy_(torch.randn_like(sf))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, run(sx, sf)))


def test_training_step_in_a_graph(status_ok):
    torch.manual_seed(0)
    x, dy = torch.randn(300, 256, device=DEV, dtype=torch.bfloat16), torch.randn(300, 128, device=DEV, dtype=torch.bfloat16)
    w = torch.randn(128, 256, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    b = torch.randn(128, device=DEV, dtype=torch.bfloat16, requires_grad=True)

    def step():
        y = Q.TrainLinearMX(x, w, b)
        return (y.detach(), *torch.autograd.grad(y, (w, b), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    x.copy_(torch.randn_like(x))
    graph.replay()
    assert all(torch.equal(a, c) for a, c in zip(out, step()))


def test_the_same_twice(status_ok):
    x = torch.randn(1500, 700, device=DEV, dtype=torch.bfloat16)
    w = Q.QuantizeMX(torch.randn(2100, 700, device=DEV), "mxfp4")
    assert torch.equal(Q.LinearMX(x, w), Q.LinearMX(x, w))
    assert torch.equal(Q.LinearMX(x[:9], w), Q.LinearMX(x[:9], w))
    # a row's result does not depend on the rows beside it, within one kernel
    assert torch.equal(Q.LinearMX(x[:9], w)[4], Q.LinearMX(x[4:9], w)[0])


def test_refusals_on_the_device(status_ok):
    x = torch.randn(4, 64, device=DEV)
    q = Q.QuantizeMX(x)
    with pytest.raises(TypeError, match="no CUDA kernel"):
        Q.QuantizeMX(x.double())
    with pytest.raises(TypeError, match="no CUDA kernel"):
        Q.DequantizeMX(q, torch.float64)
    with pytest.raises(TypeError, match="no CUDA kernel"):
        Q.MatMulMX(q, q, dtype=torch.float64)
    with pytest.raises(ValueError, match="operands on"):
        Q.MatMulMX(q, Q.QuantizeMX(x.cpu()))
    with pytest.raises(ValueError, match="bias"):
        Q.MatMulMX(q, q, torch.zeros(4))
    with pytest.raises(ValueError, match="weight"):
        Q.AddRMSNormMX(x, None, torch.ones(64))
    off_by_one = torch.empty(q.Scales.numel() + 1, dtype=torch.uint8, device=DEV)[1:]
    with pytest.raises(ValueError, match="aligned"):
        Q.DequantizeMX(Q.QTensorMX(q.Data, off_by_one, "mxfp8", (4, 64)))


def test_empty_on_the_device(status_ok):
    w = Q.QuantizeMX(torch.randn(5, 40, device=DEV))
    q = Q.QuantizeMX(torch.zeros(0, 40, device=DEV))
    assert Q.DequantizeMX(q).shape == (0, 40) and q.Data.shape == (0, 64) and q.ScaleCodes().shape == (0, 2)
    assert Q.MatMulMX(q, w).shape == (0, 5) and Q.LinearMX(torch.zeros(2, 0, 40, device=DEV), w).shape == (2, 0, 5)
    assert Q.MatMulMX(w, q).shape == (5, 0)
    n, h = Q.AddRMSNormMX(torch.zeros(0, 40, device=DEV), torch.zeros(0, 40, device=DEV), torch.ones(40, device=DEV))
    assert h.shape == (0, 40) and n.Shape == (0, 40)
    x, p, b = torch.zeros(0, 40, device=DEV, requires_grad=True), torch.randn(5, 40, device=DEV, requires_grad=True), torch.randn(5, device=DEV, requires_grad=True)
    grads = torch.autograd.grad(Q.TrainLinearMX(x, p, b).sum(), (x, p, b))
    assert [tuple(g.shape) for g in grads] == [(0, 40), (5, 40), (5,)] and not any(g.any() for g in grads)


@pytest.mark.parametrize("xt,wt,bt", [(torch.float32, torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32, torch.float32),
                                      (torch.float16, torch.bfloat16, torch.float64), (torch.float32, torch.float16, None)])
@pytest.mark.parametrize("M", [7, 700])
def test_train_linear_mixed_types_and_orders(xt, wt, bt, M, status_ok):
    """Parameters in types of their own; x a slice, the weight a transpose, the gradient's rows one row.  Equal to the products by hand."""
    N, K = 200, 300
    x = torch.randn(M, 2 * K, device=DEV).to(xt)[:, 3:3 + K].requires_grad_()
    w = torch.randn(K, N, device=DEV).to(wt).t().requires_grad_()
    b = None if bt is None else torch.randn(N, device=DEV).to(bt).requires_grad_()
    dy = torch.randn(1, N, device=DEV).to(xt).expand(M, N)
    y = Q.TrainLinearMX(x, w, b)
    leaves = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    q = Q.QuantizeMX
    with torch.no_grad():
        assert torch.equal(y, Q.MatMulMX(q(x), q(w), b, xt))
        assert torch.equal(grads[0], Q.MatMulMX(q(dy), q(w.t()), None, xt)) and torch.equal(grads[1], Q.MatMulMX(q(dy.t()), q(x.t()), None, wt))
    assert [(g.dtype, g.shape) for g in grads] == [(t.dtype, t.shape) for t in leaves]
    if b is not None:
        assert off(grads[2], dy.double().sum(0)) <= (M / 128 + 40) * 2.0 ** -24 + torch.finfo(grads[2].dtype).eps / 2


@pytest.mark.parametrize("needs", [(True, False, False), (False, True, False), (False, False, True), (True, False, True), (False, True, True)])
def test_train_linear_asks_for_what_is_needed(needs, status_ok):
    t = [torch.randn(300, 128, device=DEV), torch.randn(64, 128, device=DEV), torch.randn(64, device=DEV)]
    every = [v.clone().requires_grad_() for v in t]
    some = [v.clone().requires_grad_(n) for v, n in zip(t, needs)]
    dy = torch.randn(300, 64, device=DEV)
    want = torch.autograd.grad(Q.TrainLinearMX(*every), every, dy)
    y = Q.TrainLinearMX(*some)
    for _ in range(2):                                 # a graph that is kept gives the same again
        got = torch.autograd.grad(y, [v for v, n in zip(some, needs) if n], dy, retain_graph=True)
        assert all(off(g, w.double()) <= 310 * 2.0 ** -24 for g, w in zip(got, [w for w, n in zip(want, needs) if n]))


def test_two_graphs_replayed_at_once(status_ok):
    """Captured training steps of their own buffers, on two streams at a time, give what each gives alone."""
    torch.manual_seed(2)
    steps = []
    for N, K in ((768, 512), (520, 1000)):
        x, dy = torch.randn(2000, K, device=DEV, dtype=torch.bfloat16), torch.randn(2000, N, device=DEV, dtype=torch.bfloat16)
        w, b = torch.randn(N, K, device=DEV, dtype=torch.bfloat16, requires_grad=True), torch.randn(N, device=DEV, dtype=torch.bfloat16, requires_grad=True)
        wq = Q.QuantizeMX(w.detach(), "mxfp4")

        def step(x=x, w=w, b=b, dy=dy, wq=wq):
            y = Q.TrainLinearMX(x, w, b)
            return (*torch.autograd.grad(y, (w, b), dy), y.detach(), Q.LinearMX(x, wq, b))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        steps.append((graph, out, want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, _, _, stream in steps:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, want, _ in steps:
        assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_training_with_gradient_sinks(status_ok):
    """A model of these layers under the data-parallel wrapper, whose flat buffers take the gradients: the first gradients are autograd's own,
    and a captured step gives the same losses and parameters as one that runs eagerly."""
    from gonn_b200 import nn
    from gonn_b200.distributed.ddp import DistributedDataParallel
    from gonn_b200.utils.graph import GraphedStep
    x = torch.randn(5, 256, 96, device=DEV).bfloat16()

    def model():
        torch.manual_seed(4)
        return nn.Sequential(*(Q.NewMXTrainLinearFrom(nn.Linear(i, o, dtype=torch.bfloat16, device=torch.device(DEV, 0))) for i, o in ((96, 200), (200, 64))))

    def run(graph):
        net = model()
        ddp = DistributedDataParallel(net, optimizer=dict(kind="sgd", lr=1e-3))

        def step(x):
            out = net(x).float().square().mean()
            out.backward()
            ddp.step()
            return out

        if graph:
            step = GraphedStep(step, ddp, (x[0],), warmup=2)
        else:
            step(x[0]), step(x[0])
        losses = [float(step(v)) for v in x]
        return losses, ddp.flat_params.clone()

    (le, pe), (lg, pg) = run(False), run(True)
    assert le == lg and torch.equal(pe, pg)
    net = model()
    net(x[0]).float().square().mean().backward()
    assert all(p.grad is not None and p.grad.shape == p.shape and bool(p.grad.any()) for p in net.parameters())


def test_layers_between_devices_and_files(status_ok, tmp_path):
    m = Q.NewMXLinearFrom(Linear(100, 60), "mxfp4")
    x = torch.randn(9, 100)
    want = m(x)
    m.to(DEV)
    torch.save(m.state_dict(), tmp_path / "layer.pt")
    other = Q.NewMXLinearFrom(Linear(100, 60), "mxfp4").to(DEV)
    other.load_state_dict(torch.load(tmp_path / "layer.pt"))
    assert torch.equal(other(x.to(DEV)), m(x.to(DEV)))
    assert off(m(x.to(DEV)).cpu(), want.double()) <= (100 / 64 + 4) * 2.0 ** -23 + 2.0 ** -24


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("act", ["relu", "gelu", "geluexact"])
@pytest.mark.parametrize("M,N", [(3, 200), (40, 200), (2000, 2100)])
def test_activations_keep_nan(format, act, M, N, status_ok):
    """NaN and infinities of the operands, behind every activation and in every kernel: as on the CPU."""
    K = 333
    a, b = torch.randn(M, K), torch.randn(N, K)
    a[1, 70] = math.nan
    b[130, 5] = math.inf
    nan = torch.zeros(M, N, dtype=torch.bool)
    nan[1] = nan[:, 130] = True
    w = Q.QuantizeMX(b.to(DEV), format)
    for dtype in DTYPES:
        assert torch.equal(torch.isnan(Q.LinearMX(a.to(DEV), w, None, act, dtype)).cpu(), nan)
        assert torch.equal(torch.isnan(Q.MatMulMX(Q.QuantizeMX(a.to(DEV), format), w, torch.ones(N, device=DEV), dtype, act)).cpu(), nan)
    assert torch.equal(torch.isnan(Q.LinearMX(a[:9], cpu(w), None, act)), nan[:9])


def activated(act, dtype, rows):
    """(v, the activation of v as a product's epilogue computes it): products of zeros, v as the bias."""
    v = torch.linspace(-6, 6, 24001, device=DEV)
    zero = Q.QuantizeMX(torch.zeros(rows, 32, device=DEV))
    y = Q.MatMulMX(zero, Q.QuantizeMX(torch.zeros(v.numel(), 32, device=DEV)), v, dtype, act)
    assert all(torch.equal(r, y[0]) for r in y[1:])
    return v.double(), y[0].double()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 300])
def test_gelu_value_by_value(dtype, rows, status_ok):
    """v / (1 + exp(-2u)), relative to each value.  The exponent is rounded five times (two of them constants), each of which moves the result by
    2 |u| 2^-24; the exponential is off by two units, the reciprocal by one, and five operations follow: twelve roundings of 2^-24.  Then
    the rounding to the type, and for fp16 half a step of its subnormal numbers."""
    v, y = activated("gelu", dtype, rows)
    u = math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)
    want = v / (1 + torch.exp(-2 * u))
    rel = (10 * u.abs() + 12) * 2.0 ** -24 + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)
    least = 2.0 ** -25 if dtype == torch.float16 else 0.0
    assert bool(((y - want).abs() <= rel * 1.001 * want.abs() + least).all())


def test_gelu_of_far_values(status_ok):
    """Nothing is left below, everything above, and a NaN stays where it is."""
    v = torch.tensor([-1e30, -3e4, -20.0, math.nan, 9.0, 20.0, math.nan, 3e4, 1e30, -0.0], device=DEV)
    zero, w = Q.QuantizeMX(torch.zeros(1, 32, device=DEV)), Q.QuantizeMX(torch.zeros(10, 32, device=DEV))
    y = Q.MatMulMX(zero, w, v, torch.float32, "gelu")[0]
    assert torch.isnan(y[[3, 6]]).all() and y[:3].abs().max() < 1e-15
    assert torch.equal(y[[4, 5, 7, 8, 9]], v[[4, 5, 7, 8, 9]])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 300])
def test_exact_gelu_value_by_value(dtype, rows, status_ok):
    """v / 2 erfc(-v / sqrt 2), relative to each value, in roundings of 2^-24: the exponent -v^2 / 2 takes three, each of which moves the result by v^2 / 2;
    the exponential four; the polynomial's fit two; its argument, off by five, moves it by up to 2.7 times that; its sums eight; products four."""
    v, y = activated("geluexact", dtype, rows)
    want = v / 2 * torch.special.erfc(-v / math.sqrt(2))
    rel = (1.5 * v ** 2 + 32) * 2.0 ** -24 + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)
    least = 2.0 ** -25 if dtype == torch.float16 else 0.0
    assert bool(((y - want).abs() <= rel * 1.001 * want.abs() + least).all())


def test_exact_gelu_of_far_values(status_ok):
    v = torch.tensor([-1e30, -3e4, -20.0, math.nan, 9.0, 20.0, math.nan, 3e4, 1e30, -0.0], device=DEV)
    zero, w = Q.QuantizeMX(torch.zeros(1, 32, device=DEV)), Q.QuantizeMX(torch.zeros(10, 32, device=DEV))
    y = Q.MatMulMX(zero, w, v, torch.float32, "geluexact")[0]
    assert torch.isnan(y[[3, 6]]).all() and y[:3].abs().max() < 1e-15
    assert torch.equal(y[[4, 5, 7, 8, 9]], v[[4, 5, 7, 8, 9]])


def norm64(x, r, w, eps):
    """The definition.  (K as a tensor: by a number, ``mean`` and ``/`` multiply with a rounded 1 / K on the device; 1003 x 1.0 / 1003 is not 1 then, and
    in rows of one value what are ties would not be any.)"""
    t = x.double() if r is None else x.double() + r.double()
    K = torch.tensor(float(t.shape[-1]), dtype=torch.float64, device=t.device)
    return t / torch.sqrt(t.square().sum(-1, keepdim=True) / K + eps) * w.double()


def norm_codes(x, r, w, eps, format):
    """Codes and scales have to be those of the definition in 64 bits."""
    q, _ = Q.AddRMSNormMX(x, r, w, eps, format)
    equal(q, Q.microscale._quantize_ref(norm64(x, r, w, eps).cpu(), int(format == "mxfp4"), tuple(x.shape)))


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [96, 768, 1003, 2304, 20000])
def test_norm_of_far_rows(format, dtype, K, status_ok):
    """Rows whose 1 / rms, or the sum of x and the residual, fp32 does not hold, and rows of subnormal numbers."""
    w = (torch.rand(K, device=DEV) + 0.5).to(dtype)
    for e in (-130, -140, -100, 60, 120):
        x, r = (torch.randn(40, K, device=DEV) * 2.0 ** (e + 20) * 2.0 ** -20 for _ in range(2))
        for eps in (0.0, 1e-6):
            norm_codes(x.to(dtype), r.to(dtype), w, eps, format)
    x = torch.full((3, K), 3e38, device=DEV).to(dtype)
    norm_codes(x, x, w, 0.0, format)
    norm_codes(torch.randn(40, K, device=DEV).to(dtype), None, w, 1e40, format)


@pytest.mark.parametrize("format", FORMATS)
def test_norm_of_rows_of_one_value(format, status_ok):
    """Without eps a value's quotient is 1, and its product a tie between two codes where the weight is one."""
    c = torch.arange(1, 2001, device=DEV).float()
    for K in (32, 48, 768, 1001):
        w = torch.randint(16, 32, (K,), device=DEV).float() / 16
        norm_codes(c[:, None].expand(2000, K), None, w, 0.0, format)
        norm_codes(c[:, None].expand(2000, K).bfloat16().float(), None, -w, 0.0, format)


@pytest.mark.parametrize("format", FORMATS)
def test_norm_with_far_weights(format, status_ok):
    """Products with the weight that fp32 does not hold are values of blocks with larger scales."""
    x = torch.zeros(4, 96, device=DEV)
    x[0, 3], x[1], x[2, 40:], x[3, 60] = 1, 1, 5, -7
    for w in (3e38, 2e38, 1e37, 1e-38):
        norm_codes(x, None, torch.full((96,), w, device=DEV), 1e-6, format)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("K", [1, 40, 200, 1001, 20001])
def test_norm_pads_rows_of_nan_with_zeros(format, K, status_ok):
    """Codes and scales behind the last value and the last block are zeros whatever the row holds."""
    x = torch.randn(5, K, device=DEV)
    x[1, K // 2] = math.nan
    x[2] = 0
    x[3, K // 3] = math.inf
    q = cpu(Q.AddRMSNormMX(x, None, torch.ones(K, device=DEV), 0.0, format)[0])
    assert (q.ScaleCodes()[1:3] == 255).all()
    used = K if format == "mxfp8" else (K + 1) // 2
    assert not q.Data[:, used:].any() and (format == "mxfp8" or K % 2 == 0 or not (q.Data[:, used - 1] >> 4).any())
    s = q.Scales.view(1, -1, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(128, -1)
    assert not s[:5, -(-K // 32):].any()


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("K", [262144, 300001])
def test_norm_of_very_long_rows(format, K, status_ok):
    """More than 32 vectors of a thread, the last of them not of every thread; what lies behind the result stays as it was."""
    x, r, w = torch.randn(3, K, device=DEV), torch.randn(3, K, device=DEV), torch.rand(K, device=DEV) + 0.5
    x[1] *= 2.0 ** -70
    r[1] *= 2.0 ** -70
    norm_codes(x, r, w, 1e-30, format)
    norm_codes(x.bfloat16(), None, w.bfloat16(), 1e-30, format)
    fmt = int(format == "mxfp4")
    codes, scales = 3 * Q.microscale._row_bytes(K, fmt), Q.microscale._pieces(K, fmt) * 512
    data, s = torch.full((codes + 64,), 77, dtype=torch.uint8, device=DEV), torch.full((scales + 64,), 77, dtype=torch.uint8, device=DEV)
    h = torch.empty_like(x)
    _l.call("gb_mx_add_rms_norm", 2, fmt, x.data_ptr(), K, r.data_ptr(), K, w.data_ptr(), 1, h.data_ptr(), data.data_ptr(), s.data_ptr(), 3, K, 1e-30, _l.current_stream_handle())
    assert (data[codes:] == 77).all() and (s[scales:] == 77).all() and (s[:scales].view(-1, 32, 4, 4)[:, :, 1:] == 77).all()


def power(e):
    """2^e in 64 bits from its bits (a library's power is off by one)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def nearest64(y, format):
    """The values that codes and scales of y stand for, in 64 bits and where y is."""
    mant, least, top, largest = (3, -6, 8, 448.0) if format == "mxfp8" else (1, 0, 2, 6.0)
    rows, K = y.shape
    v = torch.nn.functional.pad(y, (0, -K % 32)).view(rows, -1, 32)
    big = v.abs().amax(-1, keepdim=True)
    e = torch.where(big == 0, -127, torch.frexp(big).exponent - 1 - top).clamp(-127, 127)
    v = v * power(-e)
    step = power((torch.frexp(v).exponent - 1).clamp(min=least) - mant)
    return ((torch.round(v / step) * step).clamp(-largest, largest) * power(e)).view(rows, -1)[:, :K]


def norm_values(x, r, w, eps, format):
    """As norm_codes, on the device."""
    q, _ = Q.AddRMSNormMX(x, r, w, eps, format)
    assert torch.equal(Q.DequantizeMX(q).double(), nearest64(norm64(x, r, w, eps), format))


def test_nearest_is_the_oracle():
    for format in FORMATS:
        y = torch.randn(50, 333, dtype=torch.float64) * torch.exp2(torch.randint(-90, 90, (50, 1)).double())
        assert torch.equal(nearest64(y, format), Q.DequantizeMX(Q.QuantizeMX(y, format), torch.float64))


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("e", [-85, -100, -110, -118])
def test_norm_of_small_blocks(format, e, status_ok):
    """Blocks of values far below the row's others, whose borders count as well: 28 million, of which fp32's roundings move some."""
    x, w = torch.randn(40000, 768, device=DEV), torch.rand(768, device=DEV) + 0.5
    x[:, 64:] *= 2.0 ** e
    norm_values(x, None, w, 1e-6, format)
    x[:, 70::32] = 0
    norm_values(x[:20000], x[20000:], w, 1e-6, format)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("splits", range(1, 9))
def test_every_number_of_slices(format, splits, status_ok):
    """Slices of K over clusters of so many CTAs, some of which have none."""
    for kind in (2, 32, 64, 128):
        for M, N, K in ((5, 200, 1700), (70, 264, 1500), (300, 512, 260)):
            _l.check(_l.lib().gb_mx_tune(kind, splits))
            try:
                y, want = product(M, N, K, format, torch.float32, True, None)
                assert torch.equal(y, want)
                if M <= 16:
                    x, w = whole(M, K, format).to(DEV), Q.QuantizeMX(whole(N, K, format).to(DEV), format)
                    assert torch.equal(Q.LinearMX(x, w), Q.MatMulMX(Q.QuantizeMX(x, format), w, dtype=torch.float32))
            finally:
                _l.lib().gb_mx_tune(0, 0)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("M,N,K", [(4600, 4900, 300), (4600, 4904, 1100), (4599, 4901, 300), (9000, 9000, 40)])
def test_pairs_of_many_tiles(format, M, N, K, status_ok):
    """Four tiles and more a pair of CTAs: accumulators, barriers and the bias' buffers come round more than once.  A bias of its own in every column."""
    a, b = whole(M, K, format).to(DEV), whole(N, K, format).to(DEV)
    qa, qb = Q.QuantizeMX(a, format), Q.QuantizeMX(b, format)
    bias = torch.arange(N, device=DEV).float() - N // 2
    want = a.double() @ b.double().T
    _l.check(_l.lib().gb_mx_tune(1, 1))
    try:
        out = (ctypes.c_longlong * 3)()
        _l.check(_l.lib().gb_mx_plan(M, N, K, FORMATS.index(format), ctypes.addressof(out)))
        assert tuple(out) == (1, 256, 1) and -(-M // 256) * -(-N // 256) >= 4 * 74
        for dtype, v, act in ((torch.float32, bias, None), (torch.bfloat16, None, None), (torch.float16, bias.half(), "relu"), (torch.bfloat16, bias.bfloat16(), None)):
            full = want if v is None else want + v.double()
            full = (full.relu() if act else full).to(dtype)
            for _ in range(3):
                y = Q.MatMulMX(qa, qb, v, dtype, act)
                _l.assert_status_ok()
                assert torch.equal(y, full)
    finally:
        _l.lib().gb_mx_tune(0, 0)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [768, 776, 1536, 2304, 4096, 8192])
def test_norm_codes_of_many_rows(format, dtype, K, status_ok):
    """Every way of dealing out rows that L2 does not keep, every value: with and without a residual, weights of the rows' type and of fp32."""
    rows = (9 << 20) // K + 7
    x, r = torch.randn(rows, K, device=DEV).to(dtype), torch.randn(rows, K, device=DEV).to(dtype)
    w = torch.rand(K, device=DEV) + 0.5
    norm_values(x, r, w.to(dtype), 1e-6, format)
    norm_values(x, None, w, 1e-6, format)
    norm_values(x, r, w, 1e-6, format)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,K", [(60000, 100), (60000, 256), (20000, 300), (8000, 1003), (4000, 2001), (2000, 4100), (2000, 8001), (300, 40001)])
def test_norm_codes_of_either_way(format, dtype, rows, K, status_ok):
    """The same for rows of any length that stay in L2, and at any address."""
    x, r = torch.randn(rows, K, device=DEV).to(dtype), torch.randn(rows, K, device=DEV).to(dtype)
    w = torch.rand(K, device=DEV) + 0.5
    norm_values(x, r, w.to(dtype), 1e-6, format)
    norm_values(x, None, w, 1e-6, format)


def native_calls(run):
    """(name, arguments) of the native calls of run()."""
    calls = []

    def hook(name, fn, args):
        calls.append((name, args))
        return fn(*args)

    _l.set_call_hook(hook)
    try:
        run()
    finally:
        _l.set_call_hook(None)
    return calls


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_a_training_layer_without_a_tape_keeps_nothing(mode, status_ok):
    layer, x = Q.NewMXTrainLinearFrom(Linear(512, 256)).to(DEV), torch.randn(100, 512, device=DEV, requires_grad=True)
    want = layer(x).detach()
    with mode():
        ((name, args),) = native_calls(lambda: layer(x))
        assert name == "gb_mx_train_forward" and args[12:16] == (False, False, None, 0)
        y = layer(x)
    assert torch.equal(y, want) and not y.requires_grad


def test_norm_keeps_the_sum_on_the_tape(status_ok):
    """h is x + residual for gradients as well; without a tape, or leaves that ask for them, it has none."""
    x, r, w = (torch.randn(*s, device=DEV) for s in ((3, 5, 40), (3, 5, 40), (40,)))
    for need in ((True, True), (True, False), (False, True)):
        leaves = [t.clone().requires_grad_(n) for t, n in zip((x, r), need)]
        dy = torch.randn_like(x)
        h = Q.AddRMSNormMX(*leaves, w)[1]
        assert torch.equal(h, x + r)
        asked = [t for t, n in zip(leaves, need) if n]
        assert all(torch.equal(g, 2 * dy) for g in torch.autograd.grad(h * 2, asked, dy))
        with torch.no_grad():
            assert not Q.AddRMSNormMX(*leaves, w)[1].requires_grad
    assert not Q.AddRMSNormMX(x, r, w.requires_grad_())[1].requires_grad
    leaf = x.clone().requires_grad_()
    assert Q.AddRMSNormMX(leaf, None, w)[1] is leaf
    assert not Q.MXRMSNorm(RMSNorm(40).to(DEV))(leaf, r)[1].requires_grad


def test_head_of_a_model(status_ok):
    """A model whose closing projection keeps its weights quantised: the logits are the layer's of the model's own hidden rows."""
    from gonn_b200.models.lm import GPT
    torch.manual_seed(3)
    model = GPT(vocab=100, d_model=64, n_layers=2, n_heads=2, d_ff=128, max_seq=16).to(DEV)
    ids = torch.randint(0, 100, (2, 16)).to(DEV)
    hidden = []
    hook = model.norm.register_forward_hook(lambda m, i, o: hidden.append(o.detach()))
    with torch.no_grad():
        full = model(ids)
        weight = Q.QuantizeMX(model.head.weight)
        model.head = Q.NewMXLinearFrom(model.head)
        y = model(ids)
    assert torch.equal(y, Q.LinearMX(hidden[-1], weight)) and torch.equal(hidden[0], hidden[1])
    assert y.shape == full.shape and y.dtype == full.dtype


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [40, 768, 1003, 2304, 20001])
def test_norm_of_rows_of_zeros(format, dtype, K, status_ok):
    """Padded batches: rows of zeros between others, also with eps 0 (NaN), and beside weights that are not finite.  (In a block with the scale of NaN
    the finite values' codes say nothing: scales and values are compared.)"""
    def compare(x, r, w, eps):
        q, want = cpu(Q.AddRMSNormMX(x, r, w, eps, format)[0]), Q.microscale._quantize_ref(norm64(x, r, w, eps).cpu(), int(format == "mxfp4"), (50, K))
        assert torch.equal(q.ScaleCodes(), want.ScaleCodes())
        a, b = Q.DequantizeMX(q), Q.DequantizeMX(want)
        assert bool(((a == b) | torch.isnan(a) & torch.isnan(b)).all())

    x, r = torch.randn(50, K, device=DEV).to(dtype), torch.randn(50, K, device=DEV).to(dtype)
    x[::3] = r[::3] = 0
    x[1::9, K // 2:] = r[1::9, K // 2:] = 0
    r[2::9] = -x[2::9]
    w = (torch.rand(K, device=DEV) + 0.5).to(dtype)
    for bad in (None, math.inf, -math.inf, math.nan, 0.0):
        if bad is not None:
            w[K // 2] = bad
        for eps in (1e-6, 0.0):
            compare(x, r, w, eps)
            compare(x, None, w, eps)


def test_the_sum_on_the_tape_takes_more_in_place(status_ok):
    """h += what a layer returned, as a residual stream runs on."""
    x, r, y, dy = (torch.randn(6, 40, device=DEV, requires_grad=n) for n in (True, True, True, False))
    h = Q.AddRMSNormMX(x * 2, r, torch.ones(40, device=DEV))[1]
    h += y
    grads = torch.autograd.grad(h, (x, r, y), dy)
    assert torch.equal(grads[0], 2 * dy) and torch.equal(grads[1], dy) and torch.equal(grads[2], dy)


def test_a_training_layers_result_takes_more_in_place(status_ok):
    layer, x = Q.NewMXTrainLinearFrom(Linear(40, 24)).to(DEV), torch.randn(6, 40, device=DEV, requires_grad=True)
    y = layer(x)
    want = torch.autograd.grad(y.sum(), x)[0]
    y = layer(x)
    y += 1
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0], want)


@pytest.mark.parametrize("format", FORMATS)
def test_offsets_beyond_32_bits(format, status_ok):
    """More than 2^31 values (and 2^32 bytes) of rows, codes and results: the last rows are those of the same rows alone."""
    R, K, N, last = 1060000, 2050, 2060, 300
    x = torch.randn(R, K, device=DEV, dtype=torch.bfloat16)
    assert x.numel() > 2 ** 31
    end, w = x[-last:].clone(), torch.rand(K, device=DEV).bfloat16() + 0.5

    def same(q, alone, rows=slice(-last, None)):
        assert torch.equal(q.Data[rows], alone.Data) and torch.equal(Q.DequantizeMX(part(q, rows)), Q.DequantizeMX(alone))

    def part(q, rows):
        return Q.QTensorMX(q.Data[rows].contiguous(), Q.microscale._pack_scales(q.ScaleCodes()[rows].cpu(), FORMATS.index(format)).to(DEV), format, (last, K))

    q = Q.QuantizeMX(x, format)
    same(q, Q.QuantizeMX(end, format))
    assert torch.equal(Q.DequantizeMX(q, torch.bfloat16)[-last:], Q.DequantizeMX(Q.QuantizeMX(end, format), torch.bfloat16))
    n, h = Q.AddRMSNormMX(x, x, w, 1e-6, format)
    m, g = Q.AddRMSNormMX(end, end, w, 1e-6, format)
    same(n, m)
    assert torch.equal(h[-last:], g)
    del h, n
    b, bias = Q.QuantizeMX(torch.randn(N, K, device=DEV), format), torch.randn(N, device=DEV)
    y = Q.MatMulMX(q, b, bias)
    assert y.numel() > 2 ** 31 and torch.equal(y[-last:], Q.MatMulMX(part(q, slice(-last, None)), b, bias))
    del y
    if format == "mxfp8":
        p, t = Q.QuantizeMXPair(x)
        same(p, Q.QuantizeMX(end))
        first = R - R % 128 - 256
        tail = Q.QuantizeMX(x[first:].t())
        assert torch.equal(t.Data[:, first:], tail.Data)
