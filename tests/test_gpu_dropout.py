"""Dropout with the residual on the GPU: the decisions are the restated
generator's, exactly; a kept value is one product and one sum (float32, or
float64) and one rounding to the type."""
import numpy as np
import pytest
import torch

import operators_ref as R
from gotransformers_b200 import _lib, moe

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def make(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return tuple((torch.randn(*shape, generator=g, dtype=torch.float64) + 0.01).to(dtype) for _ in range(2))


def check(x, rate, seed, stream, offset, residual, got):
    ref = R.dropout(x, rate, seed, stream, offset, residual)
    u = R.UNIT[x.dtype]
    # 1 / (1 - rate) and the product round, the sum rounds (3 units of the larger term), then the type does
    big = ref.abs() + (x.double() / (1 - rate)).abs()
    R.within("out", got, ref, R.HALF[x.dtype] * ref.abs() + 3 * u * big)


@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 5), (4, 256), (129, 1001), (64, 2048), (5, 3, 16)])
@pytest.mark.parametrize("dtype", [BF16, F32, F64])
@pytest.mark.parametrize("rate,offset", [(0.1, 0), (0.5, 3), (0.9, 1 << 33), (0.3, (1 << 34) + 1)])
def test_forward_and_backward(shape, dtype, rate, offset):
    x, res = make(shape, dtype, seed=len(shape) + shape[0])
    seed, stream = 12345678901234567, 3
    out = moe.dropout(x.cuda(), rate, seed, stream, offset, residual=res.cuda())
    check(x, rate, seed, stream, offset, res, out)
    plain = moe.dropout(x.cuda(), rate, seed, stream, offset)
    check(x, rate, seed, stream, offset, None, plain)
    kept = R.keep(x.numel(), rate, seed, stream, offset).reshape(x.shape)
    assert torch.equal(plain.cpu() != 0, kept & (x != 0))
    dx = moe.dropout_backward(x.cuda(), rate, seed, stream, offset)
    assert torch.equal(dx, plain)  # the same decisions and arithmetic


@pytest.mark.parametrize("dtype", [BF16, F32, F64])
def test_rate_zero_is_the_sum(dtype):
    x, res = make((33, 40), dtype)
    assert torch.equal(moe.dropout(x.cuda(), 0.0, 1).cpu(), x)
    check(x, 0.0, 1, 0, 0, res, moe.dropout(x.cuda(), 0.0, 1, residual=res.cuda()))


def test_highest_rate_drops_nearly_all():
    x = torch.ones(1 << 16, device="cuda")
    out = moe.dropout(x, 1 - 2.0**-32, 7)
    kept = R.keep(1 << 16, 1 - 2.0**-32, 7)
    assert torch.equal(out.cpu() != 0, kept)


def test_dropped_values_do_not_reach_the_output():
    n, rate = 4096, 0.5
    kept = R.keep(n, rate, 11)
    x = torch.ones(n)
    x[~kept] = torch.tensor([float("nan"), float("inf"), -float("inf")]).repeat(n)[: int((~kept).sum())]
    res = torch.full((n,), 2.0)
    out = moe.dropout(x.cuda(), rate, 11, residual=res.cuda()).cpu()
    assert torch.equal(out, torch.where(kept, 4.0, 2.0))
    assert torch.equal(moe.dropout_backward(x.cuda(), rate, 11).cpu(), torch.where(kept, 2.0, 0.0))
    # a kept NaN does, and stays one value
    x = torch.ones(n)
    i = int(torch.nonzero(kept)[5])
    x[i] = float("nan")
    assert torch.equal(torch.isnan(moe.dropout(x.cuda(), rate, 11)).cpu(), torch.arange(n) == i)


def test_parts_make_the_whole_batchs_decisions():
    x, res = make((100, 37), BF16)
    X, S = x.cuda(), res.cuda()
    whole = moe.dropout(X, 0.4, 9, 2, residual=S)
    for a, b in ((0, 33), (33, 34), (34, 100)):
        part = moe.dropout(X[a:b].contiguous(), 0.4, 9, 2, offset=a * 37, residual=S[a:b].contiguous())
        assert torch.equal(part, whole[a:b])


def test_streams_of_numbers_differ():
    x = torch.ones(1 << 14, device="cuda")
    a, b, c = (moe.dropout(x, 0.5, *s) for s in ((1, 0), (1, 1), (2, 0)))
    for p, q in ((a, b), (a, c), (b, c)):
        same = float((p == q).float().mean())
        assert abs(same - 0.5) < 6 * 0.5 / (1 << 7)  # six standard deviations of 2^14 even decisions


@pytest.mark.parametrize("shift", [1, 3])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_addresses_that_start_on_an_element(shift, dtype):
    x, res = make((50, 24), dtype)
    buf = torch.empty(3, x.numel() + shift, dtype=dtype, device="cuda")
    X, S, O = (buf[i, shift:].view(-1) for i in range(3))
    X.copy_(x.reshape(-1))
    S.copy_(res.reshape(-1))
    moe.dropout(X, 0.2, 3, residual=S, out=O)
    check(x.reshape(-1), 0.2, 3, 0, 0, res.reshape(-1), O)


@pytest.mark.parametrize("into", ["x", "residual"])
def test_in_place(into):
    x, res = make((65, 129), BF16)
    X, S = x.cuda(), res.cuda()
    ref = moe.dropout(X, 0.25, 4, residual=S)
    out = X if into == "x" else S
    assert moe.dropout(X, 0.25, 4, residual=S, out=out) is out
    assert torch.equal(out, ref)
    G = x.cuda()
    ref = moe.dropout_backward(G, 0.25, 4)
    assert torch.equal(moe.dropout_backward(G, 0.25, 4, input_gradients=G), ref)


def test_empty():
    assert moe.dropout(torch.empty(0, 8, device="cuda"), 0.5, 1).numel() == 0


def test_more_than_2_to_31_values():
    n = (1 << 31) + 1001
    x = torch.ones(n, dtype=BF16, device="cuda")
    moe.dropout(x, 0.5, 77, 1, out=x)
    for a in (0, (1 << 31) - 500, n - 1000):
        kept = R.keep(1000, 0.5, 77, 1, a)
        assert torch.equal(x[a:a + 1000].cpu(), torch.where(kept, 2.0, 0.0).to(BF16))


def test_graphs_and_streams():
    x, res = make((1000, 256), BF16)
    X, S = x.cuda(), res.cuda()
    ref = moe.dropout(X, 0.1, 5, residual=S)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = moe.dropout(X, 0.1, 5, residual=S)
    with torch.cuda.stream(s):
        graph.replay()
    eager = moe.dropout(X, 0.1, 5, residual=S)
    torch.cuda.synchronize()
    assert torch.equal(out, ref) and torch.equal(eager, ref)


def test_refusals():
    x = torch.zeros(16, device="cuda")
    for rate in (-0.1, 1.0, 2.0, float("nan")):
        with pytest.raises(_lib.GtmoeError):
            moe.dropout(x, rate, 1)
    with pytest.raises(_lib.GtmoeError):
        moe.dropout(x, 0.5, 1, offset=-1)
    with pytest.raises(ValueError):
        moe.dropout(x, 0.5, 1, residual=x.double())
    with pytest.raises(ValueError):
        moe.dropout(x[::2], 0.5, 1)
    with pytest.raises(_lib.GtmoeError):
        moe.dropout(x[:8], 0.5, 1, out=x[4:12])
