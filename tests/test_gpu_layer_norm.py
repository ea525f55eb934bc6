"""Layer norm and its backward on the GPU against the float64 restatement.

Tolerances: an output is rounded once (HALF of its type, relative), after sums
in the type's UNIT.  A thread adds at most 64 values of a row (width / 256 of
a row too wide for shared memory), then at most 5 + 16 steps join the threads, and
the mean, the variance and each product round a few times more: ADDS additions
in a row bound the relative error of every sum.  The mean's error enters xh
divided by the deviation, so AMP = 1 + max|x| rstd multiplies it."""
import pytest
import torch

import operators_ref as R
from gotransformers_b200 import _lib, moe

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def adds(width):
    return 160 + width // 256


def make(rows, width, dtype, wdtype, seed=0, shift=0.3, params=True):
    g = torch.Generator().manual_seed(seed)

    def rand(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64)

    x = (rand(rows, width) * 1.5 + shift).to(dtype)
    w = (1 + 0.2 * rand(width)).to(wdtype) if params else None
    b = (0.3 * rand(width)).to(wdtype) if params else None
    return x, w, b, rand(rows, width).to(dtype), rand(rows, width).to(dtype)


def amp_of(x, eps):
    _, _, rstd = R.layer_norm(x, None, None, eps)
    return 1 + x.double().abs().amax(1) * rstd


def check_forward(x, w, b, eps, got, mean, rstd):
    y, m, r = R.layer_norm(x, w, b, eps)
    u, a = R.UNIT[x.dtype], adds(x.shape[1])
    amp = amp_of(x, eps)[:, None]
    xh = R.layer_norm(x, None, None, eps)[0].abs()
    wm = w.double().abs() if w is not None else 1.0
    bm = b.double().abs() if b is not None else 0.0
    R.within("y", got, y, R.HALF[x.dtype] * y.abs() + u * a * ((amp + xh) * wm + bm) * (1 + R.HALF[x.dtype]))
    R.within("mean", mean, m, u * a * x.double().abs().amax(1))
    R.within("rstd", rstd, r, u * a * r * amp[:, 0])


def check_backward(x, w, dy, dres, eps, got_dx, got_dw, got_db, wdtype, before=None):
    dx, dw, db = R.layer_norm_backward(dy, x, w, eps, dres)
    u, a = R.UNIT[x.dtype], adds(x.shape[1])
    amp = amp_of(x, eps)
    _, _, rstd = R.layer_norm(x, None, None, eps)
    xh = R.layer_norm(x, None, None, eps)[0]
    g = dy.double() if w is None else dy.double() * w.double()
    # dx = rstd (g - m1 - xh m2): m1 and m2 are means of terms up to max|g| and max|g xh|, each with the sums'
    # error and the error of xh, and xh multiplies m2
    gm, xm = g.abs().amax(1), xh.abs().amax(1)
    bound = u * a * amp * rstd * gm * (3 + 3 * xm + xm * xm)
    R.within("dx", got_dx, dx, R.HALF[x.dtype] * dx.abs() + bound[:, None] * (1 + R.HALF[x.dtype])
             + (u * dx.abs() if dres is not None else 0))
    rows = x.shape[0]
    # rows in a row within one team, then teams, runs of partial rows and the runs' sum (fewer than these)
    chain = rows / 296 + 1 + 16 + 296 / 16 + 16 + 4
    tw = u * (chain * (dy.double() * xh).abs().sum(0) + a * (dy.double().abs() * amp[:, None]).sum(0))
    tb = u * chain * dy.double().abs().sum(0)
    if before is not None:
        dw, db = dw + before[0].double(), db + before[1].double()
    h = R.HALF[wdtype]
    R.within("dweight", got_dw, dw, h * dw.abs() + tw * (1 + h) + u * dw.abs())
    R.within("dbias", got_db, db, h * db.abs() + tb * (1 + h) + u * db.abs())


SIZES = [
    (1, 1), (3, 2), (5, 7), (2, 31), (33, 64), (9, 256), (17, 257), (6, 1001), (300, 512), (40, 1024), (7, 2048),
    (5, 4096), (3, 4100), (4, 8192), (2, 16384), (3, 16392), (2, 40001), (1, 70000),
]


@pytest.mark.parametrize("rows,width", SIZES)
@pytest.mark.parametrize("dtype,wdtype", [(BF16, BF16), (BF16, F32), (F32, F32), (F64, F64)])
def test_forward_and_backward(rows, width, dtype, wdtype):
    x, w, b, dy, dres = make(rows, width, dtype, wdtype, seed=rows * 1000 + width)
    eps = 1e-5
    X, W, B, DY, DR = (t.cuda() for t in (x, w, b, dy, dres))
    y, mean, rstd = moe.layer_norm(X, W, B, eps)
    check_forward(x, w, b, eps, y, mean, rstd)
    dx, dw, db = moe.layer_norm_backward(DY, X, mean, rstd, W, residual_gradients=DR)
    assert dw.dtype == wdtype and dx.dtype == dtype
    check_backward(x, w, dy, dres, eps, dx, dw, db, wdtype)


@pytest.mark.parametrize("dtype", [BF16, F32, F64])
@pytest.mark.parametrize("rows,width", [(4, 256), (3, 77), (2, 20000)])
def test_without_parameters_and_residual(dtype, rows, width):
    x, _, _, dy, _ = make(rows, width, dtype, dtype, seed=5, params=False)
    X, DY = x.cuda(), dy.cuda()
    y, mean, rstd = moe.layer_norm(X)
    check_forward(x, None, None, 1e-6, y, mean, rstd)
    dx, dw, db = moe.layer_norm_backward(DY, X, mean, rstd)
    check_backward(x, None, dy, None, 1e-6, dx, dw, db, F64 if dtype == F64 else F32)
    dx2, none, _ = moe.layer_norm_backward(DY, X, mean, rstd, want_parameters=False)
    assert none is None and torch.equal(dx, dx2)


@pytest.mark.parametrize("only", ["weight", "bias"])
def test_one_parameter(only):
    x, w, b, _, _ = make(6, 320, BF16, F32, seed=2)
    w, b = (w, None) if only == "weight" else (None, b)
    y, mean, rstd = moe.layer_norm(x.cuda(), w if w is None else w.cuda(), b if b is None else b.cuda())
    check_forward(x, w, b, 1e-6, y, mean, rstd)


@pytest.mark.parametrize("width,rows", [(2048, 1500), (256, 5000), (1001, 777), (40, 3000), (40001, 400)])
def test_many_rows_and_accumulation(rows, width):
    """More rows than blocks: every block makes several, and the gradients add to what is there."""
    x, w, b, dy, dres = make(rows, width, F32, F32, seed=9)
    X, W, B, DY, DR = (t.cuda() for t in (x, w, b, dy, dres))
    _, mean, rstd = moe.layer_norm(X, W, B)
    before = torch.full((width,), 0.5), torch.full((width,), -2.0)
    dw, db = before[0].cuda(), before[1].cuda()
    dx, dw2, db2 = moe.layer_norm_backward(DY, X, mean, rstd, W, residual_gradients=DR, weight_grad=dw, bias_grad=db)
    assert dw2 is dw and db2 is db
    check_backward(x, w, dy, dres, 1e-6, dx, dw, db, F32, before)
    # the same bits again
    dw3, db3 = before[0].cuda(), before[1].cuda()
    dx3, _, _ = moe.layer_norm_backward(DY, X, mean, rstd, W, residual_gradients=DR, weight_grad=dw3, bias_grad=db3)
    assert torch.equal(dx, dx3) and torch.equal(dw, dw3) and torch.equal(db, db3)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_far_from_zero_and_constant_rows(dtype):
    x, w, b, dy, dres = make(4, 512, dtype, dtype, seed=4, shift=100.0)
    x[2] = 3.0  # no variance: y is the bias
    y, mean, rstd = moe.layer_norm(x.cuda(), w.cuda(), b.cuda(), 1e-3)
    check_forward(x, w, b, 1e-3, y, mean, rstd)
    assert torch.equal(y[2].cpu(), b)
    dx, dw, db = moe.layer_norm_backward(dy.cuda(), x.cuda(), mean, rstd, w.cuda())
    check_backward(x, w, dy, None, 1e-3, dx, dw, db, dtype)


@pytest.mark.parametrize("width", [256, 250, 20001])
def test_addresses_that_start_on_an_element(width):
    rows = 5
    x, w, b, dy, dres = make(rows, width, BF16, BF16, seed=11)

    def shifted(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        v = buf[1:].view(t.shape)
        v.copy_(t)
        return v

    X, W, B, DY, DR = (shifted(t) for t in (x, w, b, dy, dres))
    y, mean, rstd = moe.layer_norm(X, W, B, out=shifted(x))
    check_forward(x, w, b, 1e-6, y, mean, rstd)
    dx, dw, db = moe.layer_norm_backward(DY, X, mean, rstd, W, residual_gradients=DR, input_gradients=shifted(x))
    check_backward(x, w, dy, dres, 1e-6, dx, dw, db, BF16)


@pytest.mark.parametrize("width", [512, 100, 20000])
@pytest.mark.parametrize("alias", ["dy", "x", "dres"])
def test_in_place(width, alias):
    x, w, b, dy, dres = make(700, width, F32, F32, seed=12)
    X, W, B, DY, DR = (t.cuda() for t in (x, w, b, dy, dres))
    y, mean, rstd = moe.layer_norm(X, W, B)
    ref = moe.layer_norm_backward(DY, X, mean, rstd, W, residual_gradients=DR)
    into = {"dy": DY, "x": X, "dres": DR}[alias]
    dx, dw, db = moe.layer_norm_backward(DY, X, mean, rstd, W, residual_gradients=DR, input_gradients=into)
    assert dx is into
    assert torch.equal(dx, ref[0]) and torch.equal(dw, ref[1]) and torch.equal(db, ref[2])
    X2 = x.cuda()
    assert torch.equal(moe.layer_norm(X2, W, B, out=X2)[0], y)


def test_no_rows():
    x, w, b, dy, _ = make(0, 64, F32, F32)
    y, mean, rstd = moe.layer_norm(x.cuda(), w.cuda(), b.cuda())
    assert y.shape == (0, 64)
    dx, dw, db = moe.layer_norm_backward(dy.cuda(), x.cuda(), mean, rstd, w.cuda())
    assert dx.shape == (0, 64) and not dw.any() and not db.any()
    dw.fill_(2)
    db.fill_(3)
    moe.layer_norm_backward(dy.cuda(), x.cuda(), mean, rstd, w.cuda(), weight_grad=dw, bias_grad=db)
    assert (dw == 2).all() and (db == 3).all()


def test_nan_stays_in_its_row():
    x, w, b, _, _ = make(6, 256, BF16, BF16)
    x[1, 3] = float("nan")
    x[4, 0] = float("inf")
    y = moe.layer_norm(x.cuda(), w.cuda(), b.cuda())[0].cpu()
    good = [0, 2, 3, 5]
    assert torch.isfinite(y[good]).all() and torch.isnan(y[1]).all() and torch.isnan(y[4]).all()


def test_differences_in_float64():
    """The GPU's own float64 forward against its backward: central
    differences of step 1e-6 leave about 1e-9 of rounding (2^-53 / 1e-6 of
    values around 1) and 1e-11 of curvature."""
    x, w, b, dy, v = make(5, 96, F64, F64, seed=21)
    X, W, B, DY, V = (t.cuda() for t in (x, w, b, dy, v))
    _, mean, rstd = moe.layer_norm(X, W, B)
    dx, dw, db = moe.layer_norm_backward(DY, X, mean, rstd, W)
    h = 1e-6

    def f(x, w, b):
        return float((moe.layer_norm(x, w, b)[0] * DY).sum())

    u = V[0]
    assert abs((f(X + h * V, W, B) - f(X - h * V, W, B)) / (2 * h) - float((dx * V).sum())) < 1e-6
    assert abs((f(X, W + h * u, B) - f(X, W - h * u, B)) / (2 * h) - float((dw * u).sum())) < 1e-6
    assert abs((f(X, W, B + h * u) - f(X, W, B - h * u)) / (2 * h) - float((db * u).sum())) < 1e-6


def test_streams_and_graphs():
    """Two captured backwards replayed at once on two streams, with what an
    eager call gives on a third."""
    x, w, b, dy, dres = make(2000, 512, BF16, F32, seed=31)
    X, W, B, DY, DR = (t.cuda() for t in (x, w, b, dy, dres))
    y, mean, rstd = moe.layer_norm(X, W, B)
    ref = moe.layer_norm_backward(DY, X, mean, rstd, W, residual_gradients=DR)
    torch.cuda.synchronize()
    runs = []
    for _ in range(2):
        s = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = moe.layer_norm(X, W, B) + moe.layer_norm_backward(DY, X, mean, rstd, W, residual_gradients=DR)
        runs.append((s, graph, out))
    for _ in range(3):
        for s, graph, _ in runs:
            with torch.cuda.stream(s):
                graph.replay()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        eager = moe.layer_norm_backward(DY, X, mean, rstd, W, residual_gradients=DR)
    torch.cuda.synchronize()
    for _, _, out in runs:
        assert torch.equal(out[0], y) and torch.equal(out[1], mean) and torch.equal(out[2], rstd)
        assert all(torch.equal(p, q) for p, q in zip(out[3:], ref))
    assert all(torch.equal(p, q) for p, q in zip(eager, ref))


def test_more_than_2_to_31_values():
    rows, width = (1 << 20) + 3, 2056
    X = torch.zeros(rows, width, dtype=BF16, device="cuda")
    g = torch.Generator().manual_seed(1)
    last = torch.randn(3, width, generator=g).to(BF16)
    X[-3:] = last.cuda()
    y, mean, rstd = moe.layer_norm(X, epsilon=1e-5)
    check_forward(last, None, None, 1e-5, y[-3:], mean[-3:], rstd[-3:])
    assert not y[:-3].any()
    dx, _, _ = moe.layer_norm_backward(X, X, mean, rstd, want_parameters=False, input_gradients=y)
    ref = R.layer_norm_backward(last, last, None, 1e-5)[0]
    # dy = x, so dx is what is left of a difference of equal values: rstd times a few steps of them
    R.within("dx", dx[-3:], ref, R.HALF[BF16] * ref.abs() + 2.0**-24 * adds(width) * 60)


def test_refusals():
    x = torch.zeros(4, 64, dtype=BF16, device="cuda")
    w = torch.zeros(64, dtype=BF16, device="cuda")
    with pytest.raises(ValueError):
        moe.layer_norm(x.T)
    with pytest.raises(ValueError):
        moe.layer_norm(x, w.cpu())
    with pytest.raises(ValueError):
        moe.layer_norm(x, w, w.float())
    with pytest.raises(ValueError):
        moe.layer_norm(x.half())
    with pytest.raises(ValueError):
        moe.layer_norm(x, w[:32])
    with pytest.raises(_lib.GtmoeError):
        moe.layer_norm(x, w.double())
    with pytest.raises(_lib.GtmoeError):
        moe.layer_norm(x, w, epsilon=-1.0)
    # host memory at the C entry
    host = torch.zeros(4, 64, dtype=BF16)
    rc = _lib.lib().gtmoe_layer_norm(host.data_ptr(), 2, 4, 64, None, None, 2, 1e-6, x.data_ptr(), None, None, None)
    assert rc == -1 and b"device memory" in _lib.lib().gtmoe_last_error()
