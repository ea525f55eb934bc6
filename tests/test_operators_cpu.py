"""The handle-less operators' refusals, and their restatements' definitions,
without a GPU.  The addresses passed here are never read: every call is
refused on the host, or stops because there is no device that holds them."""
import ctypes

import numpy as np
import pytest
import torch

import operators_ref as R
from gotransformers_b200 import _lib, moe, synthetic

EINVAL = -1
A = 1 << 20  # addresses no allocation of this process has
STEP = 1 << 28


def addresses(n):
    return [A + i * STEP for i in range(n)]


def norm_forward(**kw):
    x, w, b, y, m, r = addresses(6)
    a = dict(x=x, dtype=2, rows=4, width=8, weight=w, bias=b, wdtype=2, eps=1e-6, y=y, mean=m, rstd=r)
    a.update(kw)
    return _lib.lib().gtmoe_layer_norm(a["x"], a["dtype"], a["rows"], a["width"], a["weight"], a["bias"], a["wdtype"],
                                       a["eps"], a["y"], a["mean"], a["rstd"], None)


def norm_backward(**kw):
    dy, x, w, m, r, res, dx, dw, db, work = addresses(10)
    a = dict(dy=dy, x=x, dtype=1, rows=4, width=8, weight=w, wdtype=1, mean=m, rstd=r, res=res, dx=dx, dw=dw, db=db,
             acc=0, work=work, bytes=1 << 20)
    a.update(kw)
    return _lib.lib().gtmoe_layer_norm_backward(a["dy"], a["x"], a["dtype"], a["rows"], a["width"], a["weight"],
                                                a["wdtype"], a["mean"], a["rstd"], a["res"], a["dx"], a["dw"],
                                                a["db"], a["acc"], a["work"], a["bytes"], None)


def drop(**kw):
    x, res, out = addresses(3)
    a = dict(x=x, res=res, dtype=2, n=64, rate=0.5, seed=1, stream=2, offset=0, out=out)
    a.update(kw)
    return _lib.lib().gtmoe_dropout(a["x"], a["res"], a["dtype"], a["n"], a["rate"], a["seed"], a["stream"],
                                    a["offset"], a["out"], None)


def product(**kw):
    x, w, c, y = addresses(4)
    a = dict(x=x, w=w, dtype=2, rows=16, inputs=8, outputs=8, groups=2, counts=c, y=y)
    a.update(kw)
    return _lib.lib().gtmoe_grouped_product(a["x"], a["w"], a["dtype"], a["rows"], a["inputs"], a["outputs"],
                                            a["groups"], a["counts"], a["y"], None)


def weight_grad(**kw):
    dy, x, c, dw = addresses(4)
    a = dict(dy=dy, x=x, dtype=2, rows=16, inputs=8, outputs=8, groups=2, counts=c, dw=dw, wdtype=2, acc=0, work=None, bytes=0)
    a.update(kw)
    return _lib.lib().gtmoe_grouped_product_weight_grad(a["dy"], a["x"], a["dtype"], a["rows"], a["inputs"],
                                                        a["outputs"], a["groups"], a["counts"], a["dw"], a["wdtype"],
                                                        a["acc"], a["work"], a["bytes"], None)


@pytest.mark.parametrize("call", [norm_forward, norm_backward, drop, product, weight_grad])
def test_good_arguments_reach_the_device_check(call):
    """Well-formed calls get past the argument checks: without a GPU they end
    there, with one the addresses are not device memory."""
    rc = call()
    assert rc in (-2, EINVAL)
    if rc == EINVAL:
        assert b"must be device memory" in _lib.lib().gtmoe_last_error()


@pytest.mark.parametrize("call,bad", [
    (norm_forward, dict(dtype=3)),
    (norm_forward, dict(wdtype=0)),  # float64 weights beside bfloat16 rows
    (norm_forward, dict(dtype=1, wdtype=2)),
    (norm_forward, dict(rows=-1)),
    (norm_forward, dict(width=0)),
    (norm_forward, dict(width=1 << 31)),
    (norm_forward, dict(rows=1 << 60, width=1 << 20)),
    (norm_forward, dict(eps=-1e-6)),
    (norm_forward, dict(eps=float("nan"))),
    (norm_forward, dict(eps=float("inf"))),
    (norm_forward, dict(x=None)),
    (norm_forward, dict(y=None)),
    (norm_forward, dict(x=A + 1)),  # not on a bfloat16
    (norm_forward, dict(y=A + 16)),  # overlaps x shifted
    (norm_forward, dict(mean=A + 8)),  # inside x
    (norm_backward, dict(dy=None)),
    (norm_backward, dict(mean=None)),
    (norm_backward, dict(dx=None)),
    (norm_backward, dict(work=None)),
    (norm_backward, dict(bytes=4 * 2 * 8 * 4 - 1)),  # 4 rows leave 4 partial rows of 2 x 8 float32
    (norm_backward, dict(work=A + 10 * STEP + 4)),
    (norm_backward, dict(dx=A + 4)),  # overlaps dy shifted
    (norm_backward, dict(dw=A)),
    (norm_backward, dict(db=A + 7 * STEP)),  # is dweight
    (norm_backward, dict(work=A)),
    (drop, dict(dtype=-1)),
    (drop, dict(n=-1)),
    (drop, dict(rate=-0.1)),
    (drop, dict(rate=1.0)),
    (drop, dict(rate=float("nan"))),
    (drop, dict(offset=-1)),
    (drop, dict(offset=(1 << 63) - 8)),
    (drop, dict(x=None)),
    (drop, dict(out=None)),
    (drop, dict(out=A + 2)),
    (drop, dict(out=A + STEP + 2)),
    (drop, dict(x=A + 1)),
    (product, dict(dtype=7)),
    (product, dict(rows=-1)),
    (product, dict(rows=1 << 31)),
    (product, dict(inputs=0)),
    (product, dict(outputs=0)),
    (product, dict(groups=0)),
    (product, dict(groups=1025)),
    (product, dict(counts=None)),
    (product, dict(x=None)),
    (product, dict(y=A)),  # in place
    (product, dict(y=A + STEP)),  # over the weights
    (product, dict(counts=A + 2 * STEP + 4)),  # not on an int64
    (weight_grad, dict(wdtype=0)),
    (weight_grad, dict(dtype=1, wdtype=2)),
    (weight_grad, dict(dw=A + STEP)),
    (weight_grad, dict(dw=None)),
    # one group of many rows and few outputs: its sums are split, into workspace
    (weight_grad, dict(groups=1, rows=1 << 16)),
    (weight_grad, dict(groups=1, rows=1 << 16, work=A + 4 * STEP, bytes=64)),
    (weight_grad, dict(groups=1, rows=1 << 16, work=A, bytes=1 << 27)),
    (weight_grad, dict(groups=1, rows=1 << 16, work=A + 4 * STEP + 4, bytes=1 << 27)),
])
def test_refusals(call, bad):
    assert call(**bad) == EINVAL
    assert _lib.lib().gtmoe_last_error() != b""


def test_empty_batches_need_no_pointers():
    assert norm_forward(rows=0, x=None, y=None, mean=None, rstd=None) == 0
    assert norm_backward(rows=0, dy=None, x=None, dx=None, mean=None, rstd=None, dw=None, db=None, work=None) == 0
    assert drop(n=0, x=None, res=None, out=None) == 0
    assert product(rows=0, x=None, y=None) == 0
    assert weight_grad(rows=0, dy=None, x=None, acc=1) == 0


def test_workspace_size():
    n = ctypes.c_int64()
    assert _lib.lib().gtmoe_layer_norm_workspace(2, 1000, 64, ctypes.byref(n)) == 0
    assert 0 < n.value <= 1000 * 64 * 8
    assert _lib.lib().gtmoe_layer_norm_workspace(2, -1, 64, ctypes.byref(n)) == EINVAL
    assert _lib.lib().gtmoe_layer_norm_workspace(2, 1, 64, None) == EINVAL
    f = _lib.lib().gtmoe_grouped_product_workspace
    assert f(2, 1 << 16, 256, 256, 1, ctypes.byref(n)) == 0 and 0 < n.value <= 1 << 27
    assert f(2, 1 << 16, 2048, 2048, 64, ctypes.byref(n)) == 0 and n.value == 0  # tiles for every CTA pair
    assert f(1, 1 << 16, 256, 256, 1, ctypes.byref(n)) == 0 and n.value == 0  # float32
    assert f(2, 1 << 16, 256, 256, 0, ctypes.byref(n)) == EINVAL
    assert f(2, 1 << 16, 256, 256, 1, None) == EINVAL


def test_set_dropout_refuses_without_a_handle():
    assert _lib.lib().gtmoe_set_dropout(None, 0.5, 0, 0) == EINVAL


@pytest.mark.parametrize("call", [
    lambda t: moe.layer_norm(t),
    lambda t: moe.layer_norm(t.numpy()),
    lambda t: moe.layer_norm_backward(t, t, t[:, 0], t[:, 0]),
    lambda t: moe.dropout(t, 0.5, 1),
    lambda t: moe.dropout_backward(t, 0.5, 1),
    lambda t: moe.grouped_product(t, t[None], torch.ones(1, dtype=torch.int64)),
    lambda t: moe.grouped_product_input_gradients(t, t[None], torch.ones(1, dtype=torch.int64)),
    lambda t: moe.grouped_product_weight_gradients(t, t, torch.ones(1, dtype=torch.int64)),
    lambda t: moe.layer_norm(t[0]),
])
def test_host_tensors_are_refused(call):
    with pytest.raises(ValueError):
        call(torch.zeros(4, 4))


def test_generator_is_the_synthetic_inputs():
    """keep()'s words are those of synthetic.py's streams."""
    seed, stream, n = 99, 7, 40
    key = synthetic.stream_key(seed, stream)
    words = synthetic._splitmix64(key + np.arange(n // 2, dtype=np.uint64))
    halves = words.view(np.uint32)
    assert np.array_equal(R.keep(n, 0.25, seed, stream).numpy(), halves >= 0.25 * 2**32)
    # a part of a batch makes the whole batch's decisions, also from an odd element on
    assert torch.equal(R.keep(n, 0.25, seed, stream)[13:], R.keep(n - 13, 0.25, seed, stream, 13))


def test_generator_keeps_the_share_it_should():
    n, rate = 1 << 20, 0.3
    kept = float(R.keep(n, rate, 5).double().mean())
    assert abs(kept - (1 - rate)) < 6 * (rate * (1 - rate) / n) ** 0.5  # six standard deviations


def test_restated_gradients_match_differences():
    """The restatements' gradients against central differences of their
    forwards (step 1e-6, so rounding and curvature each stay below 1e-8 of
    values around 1)."""
    g = torch.Generator().manual_seed(3)

    def rand(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64)

    x, w, b, dy, v, u = rand(3, 7), rand(7), rand(7), rand(3, 7), rand(3, 7), rand(7)
    eps, h = 1e-5, 1e-6
    dx, dw, db = R.layer_norm_backward(dy, x, w, eps)

    def f(x, w, b):
        return float((R.layer_norm(x, w, b, eps)[0] * dy).sum())

    assert abs((f(x + h * v, w, b) - f(x - h * v, w, b)) / (2 * h) - float((dx * v).sum())) < 1e-6
    assert abs((f(x, w + h * u, b) - f(x, w - h * u, b)) / (2 * h) - float((dw * u).sum())) < 1e-6
    assert abs((f(x, w, b + h * u) - f(x, w, b - h * u)) / (2 * h) - float((db * u).sum())) < 1e-6

    counts = [2, 0, 3]
    x, w, dy, vx, vw = rand(5, 4), rand(3, 6, 4), rand(5, 6), rand(5, 4), rand(3, 6, 4)

    def p(x, w):
        return float((R.grouped(x, w, counts) * dy).sum())

    d = (p(x + h * vx, w) - p(x - h * vx, w)) / (2 * h)
    assert abs(d - float((R.grouped_input_gradients(dy, w, counts) * vx).sum())) < 1e-6
    d = (p(x, w + h * vw) - p(x, w - h * vw)) / (2 * h)
    assert abs(d - float((R.grouped_weight_gradients(dy, x, counts) * vw).sum())) < 1e-6
