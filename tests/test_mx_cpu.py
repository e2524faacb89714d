"""Microscaled formats on CPU tensors: the oracle against a plain restatement of the definition, layouts, refusals, layers."""
import copy
import ctypes
import math
import pickle

import pytest
import torch

from gonn_b200 import lib as _l
from gonn_b200 import quant as Q
from gonn_b200.nn import Linear, RMSNorm

FORMATS = ["mxfp8", "mxfp4"]


def numbers(format):
    """The magnitudes of a format, from its bits: exponent and fraction fields, no infinities."""
    if format == "mxfp8":
        return [(f / 8) * 2.0 ** -6 for f in range(8)] + [(1 + f / 8) * 2.0 ** (e - 7) for e in range(1, 16) for f in range(8)][:-1]
    return [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def restated(row, format):
    """(values, scale codes) of a row: block by block, value by value."""
    top, grid = (8, numbers(format)) if format == "mxfp8" else (2, numbers(format))
    values, codes = [], []
    for b in range(0, len(row), 32):
        block = row[b:b + 32]
        if not all(math.isfinite(v) for v in block):
            values += [math.nan] * len(block)
            codes.append(255)
            continue
        big = max(abs(v) for v in block)
        e = -127 if big == 0 else min(127, max(-127, math.frexp(big)[1] - 1 - top))
        codes.append(e + 127)
        for v in block:
            m = abs(v) / 2.0 ** e
            near = min(range(len(grid)), key=lambda i: (abs(grid[i] - m), i % 2))
            values.append(math.copysign(grid[near] * 2.0 ** e, v))
    return values, codes


def same(a, b):
    return bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (2, 32), (5, 33), (130, 97), (2, 3, 300)])
def test_quantize_is_the_definition(format, shape):
    t = torch.randn(*shape, dtype=torch.float64) * torch.exp2(torch.randint(-30, 30, (*shape[:-1], 1)).double())
    t.view(-1)[::7] = 0
    q = Q.QuantizeMX(t, format)
    v = Q.DequantizeMX(q, torch.float64)
    assert v.shape == t.shape and q.Numel() == t.numel()
    rows = t.reshape(-1, shape[-1])
    for r in range(rows.shape[0]):
        values, codes = restated(rows[r].tolist(), format)
        assert v.reshape(rows.shape)[r].tolist() == values
        assert q.ScaleCodes()[r].tolist() == codes


@pytest.mark.parametrize("format", FORMATS)
def test_ties_saturation_extremes(format):
    grid = numbers(format)
    mids = [(a + b) / 2 for a, b in zip(grid, grid[1:])]
    # the largest number of the block fixes the scale at 1
    rows = [grid[-1:] + mids[i:i + 31] for i in range(0, len(mids), 31)]
    rows += [[2.0 ** (9 if format == "mxfp8" else 3) * 0.99, 1.0, -grid[-1], 0.0], [0.0] * 4, [1e-40, -3e-45], [3e38, -1e-30], [math.inf, 1.0], [math.nan, -2.0] + [1.0] * 40]
    for row in rows:
        t = torch.tensor([row], dtype=torch.float64)
        values, codes = restated(row, format)
        q = Q.QuantizeMX(t, format)
        assert same(Q.DequantizeMX(q, torch.float64)[0], torch.tensor(values, dtype=torch.float64)), row
        assert q.ScaleCodes()[0].tolist() == codes


@pytest.mark.parametrize("format", FORMATS)
def test_layout(format):
    """Where the documented bytes lie."""
    R, K = 150, 300
    q = Q.QuantizeMX(torch.randn(R, K), format)
    per = 1 if format == "mxfp8" else 2
    assert q.Data.shape == (R, 320 // per) and q.Scales.numel() == 2 * (3 if format == "mxfp8" else 4) * 512
    codes, P = q.ScaleCodes(), 3 if format == "mxfp8" else 4
    for r in (0, 31, 32, 127, 128, 149):
        for b in range(10):
            assert int(q.Scales[((r // 128) * P + b // 4) * 512 + 16 * (r % 32) + 4 * (r % 128 // 32) + b % 4]) == int(codes[r, b])
    assert int(q.Data[3, 300 // per:].sum()) == 0                # the padding of a row
    if format == "mxfp4":
        one = Q.QuantizeMX(torch.tensor([[1.0, -4.0]]), format)   # scale 1: codes 2 and 8 + 6
        assert int(one.Data[0, 0]) == 2 | 14 << 4


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("act", [None, "relu", "gelu", "geluexact"])
def test_matmul(format, act):
    a, b = torch.randn(2, 3, 70), torch.randn(9, 70)
    qa, qb, bias = Q.QuantizeMX(a, format), Q.QuantizeMX(b, format), torch.randn(9)
    want = Q.DequantizeMX(qa, torch.float64) @ Q.DequantizeMX(qb, torch.float64).T + bias.double()
    if act:
        want = {"relu": torch.relu, "gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh"), "geluexact": torch.nn.functional.gelu}[act](want)
    assert torch.equal(Q.MatMulMX(qa, qb, bias, torch.float64, act), want)
    assert torch.equal(Q.LinearMX(a, qb, bias, act), want.float())
    assert Q.LinearMX(qa, qb, bias, act).dtype == torch.bfloat16


def test_norm_hands_on_the_sum():
    x, r, w = torch.randn(4, 5, 40), torch.randn(4, 5, 40), torch.rand(40) + 0.5
    q, h = Q.AddRMSNormMX(x, r, w, 1e-6, "mxfp8")
    assert torch.equal(h, x + r)
    y = h.float() * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * w
    assert torch.equal(Q.DequantizeMX(q), Q.DequantizeMX(Q.QuantizeMX(y)))
    q, h = Q.AddRMSNormMX(x, None, w)
    assert h is x
    zero, _ = Q.AddRMSNormMX(torch.zeros(2, 40), None, w)
    assert int(Q.DequantizeMX(zero).abs().sum()) == 0


def test_train_linear_gradients():
    x, w, b = (torch.randn(*s, dtype=torch.float64, requires_grad=True) for s in ((2, 11, 37), (13, 37), (13,)))
    dy = torch.randn(2, 11, 13, dtype=torch.float64)
    y = Q.TrainLinearMX(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)

    def rounded(t):
        return Q.DequantizeMX(Q.QuantizeMX(t), torch.float64)

    x2, g = x.detach().reshape(22, 37), dy.reshape(22, 13)
    assert torch.equal(y.detach().reshape(22, 13), rounded(x2) @ rounded(w).T + b.detach())
    assert torch.equal(dx.reshape(22, 37), rounded(g) @ rounded(w.detach().T).T)
    assert torch.equal(dw, rounded(g.T) @ rounded(x2.T).T)
    assert torch.allclose(db, g.sum(0), rtol=1e-12)
    # differences: on values that the format holds exactly, the layer is linear and its gradients are the layer's
    x = torch.randint(-4, 5, (32, 32)).double().requires_grad_()
    w = torch.randint(-4, 5, (32, 32)).double().requires_grad_()
    dy = torch.randint(-4, 5, (32, 32)).double()
    dx, dw = torch.autograd.grad(Q.TrainLinearMX(x, w), (x, w), dy)
    for t, d in ((x, dx), (w, dw)):
        i, j, base = 3, 5, t.detach()[3, 5].item()
        loss = []
        for v in ((base + 1, base - 1) if abs(base) < 4 else (base, base - 2 * math.copysign(1, base))):
            with torch.no_grad():
                t[i, j] = v
                loss.append((v, (Q.TrainLinearMX(x, w) * dy).sum().item()))
        with torch.no_grad():
            t[i, j] = base
        assert (loss[0][1] - loss[1][1]) / (loss[0][0] - loss[1][0]) == pytest.approx(d[i, j].item(), rel=1e-12)


def test_train_linear_asks_for_what_is_needed():
    x, w = torch.randn(3, 8), torch.randn(5, 8, requires_grad=True)
    (dw,) = torch.autograd.grad(Q.TrainLinearMX(x, w).sum(), w)
    assert dw.shape == w.shape
    x.requires_grad_()
    (dx,) = torch.autograd.grad(Q.TrainLinearMX(x, w.detach()).sum(), x)
    assert dx.shape == x.shape
    empty = torch.randn(0, 8, requires_grad=True)
    b = torch.randn(5, requires_grad=True)
    grads = torch.autograd.grad(Q.TrainLinearMX(empty, w, b).sum(), (empty, w, b))
    assert [tuple(g.shape) for g in grads] == [(0, 8), (5, 8), (5,)] and all(not g.any() for g in grads)
    with torch.no_grad():
        assert not Q.TrainLinearMX(x, w).requires_grad


def test_layers():
    lin, norm = Linear(40, 24, activation="gelu"), RMSNorm(40)
    x, r = torch.randn(6, 40), torch.randn(6, 40)
    for format in FORMATS:
        q, h = Q.MXRMSNorm(norm, format)(x, r)
        m = Q.NewMXLinearFrom(lin, format)
        y = m(q, torch.float32)
        n = norm(x + r)
        assert torch.equal(y, m(n)) and torch.equal(h, x + r)
        assert (y - lin(n)).norm() / lin(n).norm() < (0.06 if format == "mxfp8" else 0.3)       # twice a rounding of 2^-4 and 2^-2 of each operand
        again = Q.NewMXLinearFrom(Linear(40, 24, activation="gelu"), format)
        again.load_state_dict(m.state_dict())
        assert torch.equal(again(n), m(n))
    t = Q.NewMXTrainLinearFrom(Linear(40, 24))
    t(x).sum().backward()
    assert t.linear.weight.grad is not None and t.linear.bias.grad is not None
    assert torch.equal(t.Convert()(x), t(x).detach())


def test_empty():
    q = Q.QuantizeMX(torch.zeros(0, 40))
    assert Q.DequantizeMX(q).shape == (0, 40) and q.ScaleCodes().shape == (0, 2)
    w = Q.QuantizeMX(torch.randn(5, 40))
    assert Q.MatMulMX(q, w).shape == (0, 5)
    assert Q.LinearMX(torch.zeros(2, 0, 40), w).shape == (2, 0, 5)


def test_refusals():
    x, w = torch.randn(4, 64), torch.randn(8, 64)
    qx, qw = Q.QuantizeMX(x), Q.QuantizeMX(w)
    with pytest.raises(ValueError, match="formats"):
        Q.QuantizeMX(x, "mxfp6")
    with pytest.raises(ValueError, match="last dimension"):
        Q.QuantizeMX(torch.zeros(4, 0))
    with pytest.raises(ValueError, match="last dimension"):
        Q.QuantizeMX(torch.tensor(1.0))
    with pytest.raises(TypeError, match="floating"):
        Q.QuantizeMX(torch.zeros(4, 4, dtype=torch.int32))
    with pytest.raises(ValueError, match="one row"):
        Q.QuantizeMXPair(torch.zeros(0, 4))
    with pytest.raises(ValueError, match="one format"):
        Q.MatMulMX(qx, Q.QuantizeMX(w, "mxfp4"))
    with pytest.raises(ValueError, match="do not match"):
        Q.MatMulMX(qx, Q.QuantizeMX(torch.randn(8, 65)))
    with pytest.raises(ValueError, match="do not match"):
        Q.MatMulMX(qx, Q.QuantizeMX(torch.randn(2, 8, 64)))
    with pytest.raises(ValueError, match="activation"):
        Q.MatMulMX(qx, qw, act="swish")
    with pytest.raises(ValueError, match="bias"):
        Q.MatMulMX(qx, qw, torch.zeros(7))
    with pytest.raises(ValueError, match="do not belong"):
        Q.DequantizeMX(Q.QTensorMX(qx.Data, qx.Scales, "mxfp8", (4, 128)))
    with pytest.raises(ValueError, match="do not belong"):
        Q.DequantizeMX(Q.QTensorMX(qx.Data, qx.Scales[:-1], "mxfp8", (4, 64)))
    with pytest.raises(ValueError, match="contiguous"):
        Q.DequantizeMX(Q.QTensorMX(qx.Data.t().contiguous().t(), qx.Scales, "mxfp8", (4, 64)))
    with pytest.raises(TypeError, match="uint8"):
        Q.DequantizeMX(Q.QTensorMX(qx.Data.int(), qx.Scales, "mxfp8", (4, 64)))
    with pytest.raises(ValueError, match="residual"):
        Q.AddRMSNormMX(x, torch.zeros(4, 63), torch.ones(64))
    with pytest.raises(ValueError, match="residual"):
        Q.AddRMSNormMX(x, torch.zeros(4, 64, dtype=torch.bfloat16), torch.ones(64))
    with pytest.raises(ValueError, match="weight"):
        Q.AddRMSNormMX(x, None, torch.ones(63))
    with pytest.raises(TypeError, match="weight"):
        Q.AddRMSNormMX(x, None, torch.ones(64, dtype=torch.float16))
    with pytest.raises(ValueError, match="do not match"):
        Q.TrainLinearMX(x, torch.zeros(8, 63))
    with pytest.raises(ValueError, match="activation"):
        Q.MXTrainLinear(Linear(4, 4, activation="relu"))


A, ODD = 4096, 4104                   # addresses that are never read: on a 16-byte boundary, and not


@pytest.mark.parametrize("name,args,what", [
    ("gb_mx_quantize", (0, 0, None, 64, A, A, 4, 64, None), "needed"),
    ("gb_mx_quantize", (0, 0, A, 64, ODD, A, 4, 64, None), "16-byte"),
    ("gb_mx_quantize", (0, 0, A, 64, A, None, 4, 64, None), "needed"),
    ("gb_mx_quantize", (3, 0, A, 64, A, A, 4, 64, None), "dtype"),
    ("gb_mx_quantize", (0, 2, A, 64, A, A, 4, 64, None), "format"),
    ("gb_mx_quantize", (0, 0, A, -1, A, A, 4, 64, None), "pitch"),
    ("gb_mx_quantize", (0, 0, A, 64, A, A, 0, 64, None), "extents"),
    ("gb_mx_quantize", (0, 0, A, 64, A, A, 4, (1 << 30) + 1, None), "extents"),
    ("gb_mx_quantize_both", (0, A, 64, A, A, None, A, None, None, 0, 4, 64, None), "needed"),
    ("gb_mx_quantize_both", (7, A, 64, A, A, A, A, None, None, 0, 4, 64, None), "dtype"),
    ("gb_mx_quantize_both", (0, A, 64, A, A, A, A, A, None, 0, 4, 64, None), "column sums"),
    ("gb_mx_quantize_both", (0, A, 64, A, A, A, A, A, A, 5, 4, 64, None), "column sums"),
    ("gb_mx_dequantize", (0, 0, A, A, None, 4, 64, None), "needed"),
    ("gb_mx_dequantize", (5, 0, A, A, A, 4, 64, None), "dtype"),
    ("gb_mx_add_rms_norm", (0, 0, A, 64, None, 64, None, 0, None, A, A, 4, 64, 1e-6, None), "weight"),
    ("gb_mx_add_rms_norm", (0, 0, A, 64, A, 64, A, 0, None, A, A, 4, 64, 1e-6, None), "room for the sum"),
    ("gb_mx_matmul", (0, A, A, A, None, A, 8, None, 0, 4, 8, 64, 0, 0, None), "boundaries"),
    ("gb_mx_matmul", (0, A, A, A, ODD, A, 8, None, 0, 4, 8, 64, 0, 0, None), "boundaries"),
    ("gb_mx_matmul", (0, A, A, A, A, A, 7, None, 0, 4, 8, 64, 0, 0, None), "pitch"),
    ("gb_mx_matmul", (0, A, A, A, A, A, 8, None, 0, 4, 8, 64, 3, 0, None), "type"),
    ("gb_mx_matmul", (0, A, A, A, A, A, 8, None, 0, 4, 8, 64, 0, 4, None), "activation"),
    ("gb_mx_matmul", (0, A, A, A, A, A, 8, None, 0, 4, 0, 64, 0, 0, None), "extents"),
    ("gb_mx_matmul_rows", (0, 0, A, 64, A, A, A, 8, None, 0, 17, 8, 64, 0, 0, None), "16 at most"),
    ("gb_mx_matmul_rows", (0, 0, None, 64, A, A, A, 8, None, 0, 4, 8, 64, 0, 0, None), "needed"),
    ("gb_mx_linear", (0, 0, A, 64, A, A, A, None, 0, 40, 8, 64, 0, 0, None, 0, None), "scratch"),
    ("gb_mx_linear", (0, 0, A, 64, A, A, A, None, 0, 0, 8, 64, 0, 0, None, 0, None), "extents"),
    ("gb_mx_train_forward", (0, 0, A, 64, A, 64, A, None, 0, 4, 8, 64, 1, 1, A, 0, A, 1 << 30, None), "scratch"),
    ("gb_mx_train_forward", (0, 0, A, 64, A, 64, A, None, 0, 4, 8, 1 << 31, 1, 1, A, 1 << 40, A, 1 << 40, None), "extents"),
    ("gb_mx_train_backward", (0, A, 8, None, A, 0, A, 0, None, 0, 4, 8, 64, A, 1 << 30, None), "kept"),
    ("gb_mx_train_backward", (0, A, 8, A, A, 0, None, 0, A, 0, 4, 8, 64, A, 1 << 30, None), "with dw only"),
    ("gb_mx_tune", (3, 0), "kind"),
])
def test_native_refusals(name, args, what):
    """Every entry of the library looks at its arguments before it touches a device."""
    with pytest.raises(RuntimeError, match=what):
        _l.check(getattr(_l.lib(), name)(*args), name)


def test_copies_keep_their_values():
    t = torch.randn(5, 70)
    for q in (Q.QuantizeMX(t, "mxfp4"), Q.QTensorMX(*(lambda p: (p.Data, p.Scales, p.Format, p.Shape))(Q.QuantizeMX(t)))):
        for other in (copy.copy(q), copy.deepcopy(q), pickle.loads(pickle.dumps(q))):
            assert torch.equal(Q.DequantizeMX(other), Q.DequantizeMX(q)) and other.Shape == (5, 70) and other.Format == q.Format
        assert q.Numel() == 350 and repr(q) == f"QTensorMX({q.Format}, (5, 70))"
    with pytest.raises(AttributeError):
        q.Shape = (70, 5)


def test_a_layer_moves_and_keeps_its_codes():
    m = Q.NewMXLinearFrom(Linear(40, 24), "mxfp4")
    x = torch.randn(3, 40)
    want = m(x)
    again = copy.deepcopy(m).half()                   # codes and scales are bytes, whatever the layer's type
    assert again.codes.dtype == torch.uint8 and again.bias.dtype == torch.float16
    assert torch.equal(again.float().codes, m.codes) and torch.equal(copy.deepcopy(m)(x), want)


@pytest.mark.parametrize("xt,wt,bt", [(torch.float32, torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32, torch.float32), (torch.float32, torch.bfloat16, torch.float32)])
def test_train_linear_mixed_types(xt, wt, bt):
    x, w, b = torch.randn(6, 40).to(xt).requires_grad_(), torch.randn(9, 40).to(wt).requires_grad_(), torch.randn(9).to(bt).requires_grad_()
    y = Q.TrainLinearMX(x, w, b)
    grads = torch.autograd.grad(y.sum(), (x, w, b))
    assert y.dtype == xt and [g.dtype for g in grads] == [xt, wt, bt]
    assert torch.equal(grads[2].float(), torch.full((9,), 6.0))


@pytest.mark.parametrize("format", FORMATS)
def test_norm_of_rows_of_one_value(format):
    """Without eps a value's quotient is 1 and the norm the weight, ties between two codes among them."""
    c = torch.arange(1, 201, dtype=torch.float64)
    for K in (32, 48, 1001):
        w = torch.randint(16, 32, (K,)).double() / 16
        q, _ = Q.AddRMSNormMX(c[:, None].expand(200, K), None, w, 0.0, format)
        want = Q.QuantizeMX(w.expand(200, K), format)
        assert torch.equal(q.Data, want.Data) and torch.equal(q.ScaleCodes(), want.ScaleCodes())


def plan(M, N, K, format):
    out = (ctypes.c_longlong * 3)()
    _l.check(_l.lib().gb_mx_plan(M, N, K, FORMATS.index(format), ctypes.addressof(out)), "gb_mx_plan")
    return tuple(out)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("M,N,K", [(3, 40, 1500), (70, 264, 1500), (520, 1032, 700), (5000, 4000, 4100)])
def test_a_product_runs_as_it_is_told(format, M, N, K):
    """Every kernel, tile and number of slices that gb_mx_tune takes is the one that runs; others are refused, and leave things as they were."""
    tune = _l.lib().gb_mx_tune
    try:
        for kind, most in ((0, 0), (1, 2), (2, 8), (32, 8), (64, 8), (128, 8)):
            for splits in range(1, 10):
                _l.check(tune(0, 0))
                if splits > most:
                    with pytest.raises(RuntimeError, match="splits"):
                        _l.check(tune(kind, splits))
                    continue
                by_size = plan(M, N, K, format)
                _l.check(tune(kind, splits))
                got = plan(M, N, K, format)
                rows = 256 if kind == 1 else 16 if M <= 16 else kind if kind > 2 else got[1]
                assert got == (1 if kind == 1 else 2, rows, splits) and rows in (16, 32, 64, 128, 256)
                _l.check(tune(0, 0))
                assert plan(M, N, K, format) == by_size
    finally:
        tune(0, 0)


def test_products_that_no_launch_holds():
    for kind in (1, 2):
        try:
            _l.check(_l.lib().gb_mx_tune(kind, 1))
            with pytest.raises(RuntimeError, match="too many tiles"):
                _l.check(_l.lib().gb_mx_matmul(0, A, A, A, A, A, 1 << 31, None, 0, (1 << 31) - 1, (1 << 31) - 1, 64, 0, 0, None))
        finally:
            _l.lib().gb_mx_tune(0, 0)


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_a_training_layer_without_a_tape_keeps_nothing(mode, monkeypatch):
    layer, x = Q.NewMXTrainLinearFrom(Linear(40, 24)), torch.randn(6, 40, requires_grad=True)
    want = layer(x).detach()
    monkeypatch.setattr(Q.microscale, "QuantizeMXPair", lambda t: pytest.fail("quantised for gradients that nobody asks for"))
    with mode():
        y = layer(x)
    assert torch.equal(y, want) and not y.requires_grad
    monkeypatch.undo()
    pairs = []
    monkeypatch.setattr(Q.microscale, "QuantizeMXPair", lambda t, f=Q.QuantizeMXPair: (pairs.append(tuple(t.shape)), f(t))[1])
    layer(x.detach()).sum().backward()                 # x, whose transpose dW takes; the gradient of y
    assert pairs == [(6, 40), (6, 24)]


@pytest.mark.parametrize("name,args,kernels", [
    ("gb_mx_linear", (0, 0, A, 64, A, A, A, None, 0, 16, 8, 64, 0, 0, None, 0, None), 1),
    ("gb_mx_linear", (0, 0, A, 64, A, A, A, None, 0, 17, 8, 64, 0, 0, A, 4096, None), 2),
    ("gb_mx_train_backward", (0, A, 8, A, A, 0, A, 0, A, 0, 4, 8, 64, A, 4096, None), 4),
    ("gb_mx_train_backward", (0, A, 8, A, A, 0, A, 0, None, 0, 4, 8, 64, A, 4096, None), 3),
    ("gb_mx_train_backward", (0, A, 8, A, A, 0, None, 0, None, 0, 4, 8, 64, A, 4096, None), 2),
    ("gb_mx_train_forward", (0, 0, A, 64, A, 64, A, None, 0, 4, 8, 64, 1, 1, A, 4096, A, 4096, None), 3),
    ("gb_mx_quantize", (0, 0, A, 64, A, A, 4, 64, None), 1),
])
def test_kernels_that_a_call_launches(name, args, kernels, monkeypatch):
    """The count goes by the arguments (nothing is launched here)."""
    monkeypatch.setitem(_l._fn_cache, name, lambda *a: 0)
    before = _l.kernel_count
    _l.call(name, *args)
    assert _l.kernel_count - before == kernels


def test_norm_keeps_the_sum_on_the_tape():
    """h is x + residual for gradients as well; without a tape, or leaves that ask for them, it has none."""
    x, r, w = (torch.randn(*s) for s in ((3, 5, 40), (3, 5, 40), (40,)))
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
    assert not Q.MXRMSNorm(RMSNorm(40))(leaf, r)[1].requires_grad


def test_head_of_a_model():
    """A model whose closing projection keeps its weights quantised: the logits are the layer's of the model's own hidden rows."""
    from gonn_b200.models.lm import GPT
    torch.manual_seed(3)
    model = GPT(vocab=100, d_model=64, n_layers=2, n_heads=2, d_ff=128, max_seq=16)
    ids = torch.randint(0, 100, (2, 16))
    hidden = []
    hook = model.norm.register_forward_hook(lambda m, i, o: hidden.append(o.detach()))
    with torch.no_grad():
        full = model(ids)
        weight = Q.QuantizeMX(model.head.weight)
        model.head = Q.NewMXLinearFrom(model.head)
        y = model(ids)
    assert torch.equal(y, Q.LinearMX(hidden[-1], weight)) and torch.equal(hidden[0], hidden[1])
    assert y.shape == full.shape and y.dtype == full.dtype


def test_the_sum_on_the_tape_takes_more_in_place():
    """h += what a layer returned, as a residual stream runs on."""
    x, r, y, dy = (torch.randn(6, 40, requires_grad=n) for n in (True, True, True, False))
    h = Q.AddRMSNormMX(x * 2, r, torch.ones(40))[1]
    h += y
    grads = torch.autograd.grad(h, (x, r, y), dy)
    assert torch.equal(grads[0], 2 * dy) and torch.equal(grads[1], dy) and torch.equal(grads[2], dy)


def test_a_training_layers_result_takes_more_in_place():
    layer, x = Q.NewMXTrainLinearFrom(Linear(40, 24)), torch.randn(6, 40, requires_grad=True)
    y = layer(x)
    want = torch.autograd.grad(y.sum(), x)[0]
    y = layer(x)
    y += 1
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0], want)
