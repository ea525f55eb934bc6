"""Layer norm with random rows on every way that its launch can be laid out:
tiles of four, two and one row, parameters read through L1 or kept in shared
memory, rings that are refilled several times, and, in the backward, teams of
every size.  The restatement runs on the GPU in float64; the tolerances are
those of test_gpu_layer_norm.py."""
import pytest
import torch

import operators_ref as R
from gotransformers_b200 import moe
from test_gpu_layer_norm import adds, check_backward, check_forward

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
EPS = 1e-5


def make(rows, width, dtype, wdtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*s):
        return torch.randn(*s, generator=g, device="cuda")

    x = (rand(rows, width) * 1.5 + 0.3).to(dtype)
    return (x, (1 + 0.2 * rand(width)).to(wdtype), (0.3 * rand(width)).to(wdtype), rand(rows, width).to(dtype),
            rand(rows, width).to(dtype))


def hold(name, got, ref, tol):
    over = (got.double() - ref).abs() - tol
    assert torch.isfinite(got).all() and float(over.max()) <= 0, (name, float(over.max()), int((over > 0).sum()))


def pieces(rows, width):
    step = max(1, (1 << 24) // width)
    return [slice(r, min(rows, r + step)) for r in range(0, rows, step)]


# rows, width, dtype, weight dtype
SIZES = [
    (60001, 512, BF16, BF16),   # four rows to a warp, refilled (28416 rows are in flight)
    (100003, 256, BF16, F32),
    (30005, 512, F32, F32),
    (28001, 256, F64, F64),
    (20001, 2048, BF16, BF16),  # two rows
    (16387, 2048, BF16, F32),
    (9001, 1024, F32, F32),
    (9001, 512, F64, F64),
    (8195, 4096, BF16, BF16),   # one row, the parameters in shared memory
    (8195, 4096, BF16, F32),
    (9007, 2056, BF16, F32),
    (6003, 2048, F32, F32),
    (5003, 1100, F32, F32),
    (5003, 600, F64, F64),
    (3001, 8192, BF16, BF16),
    (2000, 4096, BF16, BF16),   # one row, few rows
    (7105, 40, BF16, F32),      # narrow rows: four to a warp, less than a warp's vectors each
    (50001, 8, BF16, BF16),
]


@pytest.mark.parametrize("rows,width,dtype,wdtype", SIZES)
def test_random_rows(rows, width, dtype, wdtype):
    x, w, b, dy, dres = make(rows, width, dtype, wdtype, rows + width)
    y, mean, rstd = moe.layer_norm(x, w, b, EPS)
    dx, dw, db = moe.layer_norm_backward(dy, x, mean, rstd, w, residual_gradients=dres)
    u, a, h = R.UNIT[dtype], adds(width), R.HALF[dtype]
    wm, bm = w.double().abs(), b.double().abs()
    sums = [torch.zeros(width, dtype=F64, device="cuda") for _ in range(5)]
    for s in pieces(rows, width):
        xs, dys = x[s].double(), dy[s].double()
        ry, m, r = R.layer_norm(xs, w, b, EPS)
        xh = (xs - m[:, None]) * r[:, None]
        amp = 1 + xs.abs().amax(1) * r
        hold("y", y[s], ry, h * ry.abs() + u * a * ((amp[:, None] + xh.abs()) * wm + bm) * (1 + h))
        hold("mean", mean[s], m, u * a * xs.abs().amax(1))
        hold("rstd", rstd[s], r, u * a * r * amp)
        rdx, rdw, rdb = R.layer_norm_backward(dys, xs, w, EPS, dres[s])
        gm, xm = (dys * w.double()).abs().amax(1), xh.abs().amax(1)
        bound = u * a * amp * r * gm * (3 + 3 * xm + xm * xm)
        hold("dx", dx[s], rdx, h * rdx.abs() + bound[:, None] * (1 + h) + u * rdx.abs())
        for at, v in zip(sums, (rdw, rdb, (dys * xh).abs().sum(0), dys.abs().sum(0),
                                (dys.abs() * amp[:, None]).sum(0))):
            at += v
    rdw, rdb, mag, dmag, amag = sums
    chain, wh = rows / 296 + 1 + 16 + 296 / 16 + 16 + 4, R.HALF[wdtype]
    hold("dweight", dw, rdw, (wh + u) * rdw.abs() + u * (chain * mag + a * amag) * (1 + wh))
    hold("dbias", db, rdb, (wh + u) * rdb.abs() + u * chain * dmag * (1 + wh))
    # and the same bits again, as on rows that go elsewhere
    again = moe.layer_norm(x, w, b, EPS, out=x)
    assert again[0] is x and all(torch.equal(p, q) for p, q in zip(again, (y, mean, rstd)))


def test_gradients_past_2_to_31_values():
    """The last three rows are random, with gradients of their own; all before
    them are zeros, which add exactly nothing.  A row read or written 2^31
    values too early would leave gradients of zero."""
    rows, width = (1 << 20) + 3, 2056
    x, dy, dres = (torch.zeros(rows, width, dtype=BF16, device="cuda") for _ in range(3))
    g = torch.Generator().manual_seed(1)
    lx, ldy, ldres = (torch.randn(3, width, generator=g).to(BF16) for _ in range(3))
    x[-3:], dy[-3:], dres[-3:] = lx.cuda(), ldy.cuda(), ldres.cuda()
    w, b = (1 + 0.2 * torch.randn(width, generator=g)).to(BF16), torch.zeros(width, dtype=BF16)
    y, mean, rstd = moe.layer_norm(x, w.cuda(), b.cuda(), EPS)
    check_forward(lx, w, b, EPS, y[-3:], mean[-3:], rstd[-3:])
    dx, dw, db = moe.layer_norm_backward(dy, x, mean, rstd, w.cuda(), residual_gradients=dres, input_gradients=y)
    assert float(dx[-3:].abs().mean()) > 0.1 and not dx[:-3].any()
    check_backward(lx, w, ldy, ldres, EPS, dx[-3:], dw, db, BF16)
