"""Long sums of the grouped products: how many terms there are, and whether
they have one sign or repeat, may not show beyond each result's own precision.

The tensor cores cut additions towards zero (at most 2^-23 of the sum each),
so a sum is made in runs of stages of 64 terms, four additions to a stage: 8
stages for float32 results, 16 for bfloat16 ones.  Runs are added with
rounding, and what sixteen of them round off is carried along, so the bounds
below are those of a run.  The SIMT cores make sums of more than 1024 terms in
runs of 256 rounded additions and carry what every run's addition rounds off."""
import pytest
import torch

import operators_ref as R
from gotransformers_b200 import moe

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def device_counts(counts):
    return torch.tensor(counts, dtype=torch.int64, device="cuda")


def spread(rows, columns, seed, scaled):
    """Positive values with a factor of their own, between 1 and 2, per row or
    per column, so that sums over the other axis fall anywhere between two
    bfloat16 numbers."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    v = 0.75 + 0.5 * torch.rand(rows, columns, generator=g, device="cuda")
    f = 1 + torch.rand((rows, 1) if scaled == "rows" else (1, columns), generator=g, device="cuda")
    return (v * f).to(BF16)


def lean(got, ref):
    """The mean relative error: where it points."""
    return float(((got.double() - ref) / ref).mean())


@pytest.mark.parametrize("call", ["product", "input gradients", "weight gradients"])
def test_bfloat16_results_do_not_lean(call):
    """65536 results, each a sum of many terms of one sign.  Roundings to
    bfloat16 err evenly to both sides, at most 2^-8 each with a deviation of at
    most 2^-8 / sqrt(3): the mean of 256 x 256 of them whose 256 row factors
    and 256 column factors are independent is within 8 deviations / 256.  The
    cut additions of a run are at most 64 * 2^-23, half of that on average for
    an even cut and half again because partial sums grow evenly; one sum over
    all the terms would lean by 1.6e-3 (262144 terms)."""
    n = 1 << 18 if call != "weight gradients" else 60000
    if call == "weight gradients":
        x, dy = spread(n, 256, 1, "columns"), spread(n, 256, 2, "columns")
        ref = dy.double().T @ x.double()
        # 80 groups: no group's rows are split
        got = moe.grouped_product_weight_gradients(dy, x, device_counts([n] + [0] * 79))[0]
    else:
        x, w = spread(256, n, 3, "rows"), spread(256, n, 4, "rows")
        ref = x.double() @ w.double().T
        c = device_counts([256])
        if call == "product":
            got = moe.grouped_product(x, w[None], c)
        else:
            got = moe.grouped_product_input_gradients(x, w.T.contiguous()[None], c)
    assert abs(lean(got, ref)) <= 8 * 2.0**-8 / 3**0.5 / 256 + 64 * 2.0**-23 / 4
    R.within("results", got, ref.cpu(), ref.cpu().abs() * (R.HALF[BF16] + (64 + 33) * 2.0**-23))
    moe.check_operators()


@pytest.mark.parametrize("inputs,outputs,counts", [
    (8200, 72, [70, 0, 300]), (72, 8200, [70, 0, 300]), (16384, 264, [1, 257]), (264, 20000, [33, 128, 95]),
    (140000, 40, [5, 20]), (40, 140000, [5, 20]),
])
def test_products_over_many_terms_are_exact_on_whole_numbers(inputs, outputs, counts):
    """More than one run, and more runs than are kept in registers."""
    g = torch.Generator().manual_seed(inputs)
    rows, groups = sum(counts) + 3, len(counts)
    x = torch.randint(-4, 5, (rows, inputs), generator=g).to(BF16)
    w = torch.randint(-4, 5, (groups, outputs, inputs), generator=g).to(BF16)
    dy = torch.randint(-4, 5, (rows, outputs), generator=g).to(BF16)
    x[-3:], dy[-3:] = float("nan"), float("nan")
    n, C = rows - 3, device_counts(counts)
    y = torch.full((rows, outputs), 7.0, dtype=BF16, device="cuda")
    dx = torch.full((rows, inputs), 7.0, dtype=BF16, device="cuda")
    moe.grouped_product(x.cuda(), w.cuda(), C, out=y)
    moe.grouped_product_input_gradients(dy.cuda(), w.cuda(), C, input_gradients=dx)
    assert torch.equal(y[:n].cpu(), R.grouped(x[:n], w, counts).to(BF16))
    assert torch.equal(dx[:n].cpu(), R.grouped_input_gradients(dy[:n], w, counts).to(BF16))
    assert (y[n:] == 7).all() and (dx[n:] == 7).all()
    moe.check_operators()


@pytest.mark.parametrize("groups", [80, 1])
def test_float32_weight_gradients_of_constant_rows(groups):
    """16.8 million equal rows.  A run's sums are exact here, and where the
    runs' sum rounds, it rounds the same way again and again: 1.6e-4 of it if
    they were added one by one.  Carried along, at most the 2^-24 of 16 runs
    and of the last addition are left; a group that is split has at most 148
    parts, added one by one."""
    n = (1 << 24) + 37
    x = torch.full((n, 8), 171 / 128, dtype=BF16, device="cuda")
    dw = moe.grouped_product_weight_gradients(x, x, device_counts([n] + [0] * (groups - 1)), dtype=F32)[0]
    ref = n * (171 / 128) ** 2
    tol = 17 * 2.0**-24 + (148 * 2.0**-24 if groups == 1 else 0)
    assert float((dw.double() / ref - 1).abs().max()) <= tol
    moe.check_operators()


@pytest.mark.parametrize("groups", [80, 1])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_infinite_sums_stay_infinite(groups, dtype):
    n = 40000
    x, dy = spread(n, 64, 5, "columns"), spread(n, 64, 6, "columns")
    x[100, 3], x[39999, 7], x[20000, 9], x[5, 11] = float("inf"), float("inf"), float("nan"), -float("inf")
    dw = moe.grouped_product_weight_gradients(dy, x, device_counts([n] + [0] * (groups - 1)), dtype=dtype)[0].cpu()
    inf = torch.full((64,), float("inf"), dtype=dtype)
    assert torch.equal(dw[:, 3], inf) and torch.equal(dw[:, 7], inf) and torch.equal(dw[:, 11], -inf)
    assert torch.isnan(dw[:, 9]).all()
    rest = [c for c in range(64) if c not in (3, 7, 9, 11)]
    assert torch.isfinite(dw[:, rest]).all()


@pytest.mark.parametrize("value,n", [(1.0, (1 << 25) + 37), (171 / 128, (1 << 22) + 37)])
@pytest.mark.parametrize("dtype,width,wdtype", [(F32, 8, F32), (BF16, 7, F32), (BF16, 7, BF16)])
def test_equal_rows_on_the_simt_cores(value, n, dtype, width, wdtype):
    """Float32 operands, and bfloat16 ones that the tensor cores cannot
    address.  One float32 sum stops growing at 2^24 ones, and rounds equal
    values alike again and again.  A run's partial sums grow evenly, so its 256
    additions err by at most 129 * 2^-24 of it; what is carried along can make
    each err by 2^-24 of 2^-24 of the total."""
    x = torch.full((n, width), value, dtype=dtype, device="cuda")
    dw = moe.grouped_product_weight_gradients(x, x, device_counts([n]), dtype=wdtype)[0]
    ref = n * value * value
    half = R.HALF[BF16] if wdtype == BF16 else 0
    assert float((dw.double() / ref - 1).abs().max()) <= half + 131 * 2.0**-24 + n * 2.0**-48


@pytest.mark.parametrize("value", [1.0, 171 / 128])
@pytest.mark.parametrize("call", ["product", "input gradients"])
def test_equal_terms_on_the_simt_cores(value, call):
    n = (1 << 24) + 4099
    x = torch.full((3, n), value, device="cuda")
    if call == "product":
        y = moe.grouped_product(x, x[:2].view(1, 2, n), device_counts([3]))
    else:
        y = moe.grouped_product_input_gradients(x, x[:2].reshape(1, n, 2), device_counts([3]))
    ref = n * value * value
    assert float((y.double() / ref - 1).abs().max()) <= 131 * 2.0**-24 + n * 2.0**-48


@pytest.mark.parametrize("n", [255, 257, 512, 513, 768, 1024, 1025, 1280, 1300])
@pytest.mark.parametrize("inputs,outputs", [(20, 24), (200, 130)])
def test_runs_on_the_simt_cores_are_exact_on_whole_numbers(n, inputs, outputs):
    """Terms around a run's end, in each direction and tile, added to what is there too."""
    g = torch.Generator().manual_seed(n)

    def whole(*s):
        return torch.randint(-4, 5, s, generator=g).float()

    for rows, k, m, counts in ((9, n, outputs, [4, 5]), (300, n, outputs, [300]), (9, inputs, n, [4, 5]),
                               (300, inputs, n, [300]), (2 * n, inputs, outputs, [n, n])):
        x, w, dy, C = whole(rows, k), whole(len(counts), m, k), whole(rows, m), device_counts(counts)
        assert torch.equal(moe.grouped_product(x.cuda(), w.cuda(), C).cpu(), R.grouped(x, w, counts).float())
        dx = moe.grouped_product_input_gradients(dy.cuda(), w.cuda(), C).cpu()
        assert torch.equal(dx, R.grouped_input_gradients(dy, w, counts).float())
        dw = w.cuda()
        moe.grouped_product_weight_gradients(dy.cuda(), x.cuda(), C, weight_grad=dw)
        assert torch.equal(dw.cpu(), (R.grouped_weight_gradients(dy, x, counts) + w.double()).float())
    moe.check_operators()


def test_infinite_sums_on_the_simt_cores_stay_infinite():
    n = 5000
    x, dy = spread(n, 63, 5, "columns").float(), spread(n, 65, 6, "columns").float()
    x[100, 3], x[4999, 7], x[2000, 9], x[5, 11] = float("inf"), float("inf"), float("nan"), -float("inf")
    dw = moe.grouped_product_weight_gradients(dy, x, device_counts([n]))[0].cpu()
    inf = torch.full((65,), float("inf"))
    assert torch.equal(dw[:, 3], inf) and torch.equal(dw[:, 7], inf) and torch.equal(dw[:, 11], -inf)
    assert torch.isnan(dw[:, 9]).all()
    rest = [c for c in range(63) if c not in (3, 7, 9, 11)]
    assert torch.isfinite(dw[:, rest]).all()


def test_a_row_tail_after_seconds_of_whole_stages():
    """80 groups are not split: one pair of SMs takes 700 million rows by
    itself, 280 ns per 64 of them and three seconds in all, before it gets to
    the stage that the group's last 37 rows do not fill.  What waits for that
    stage may not give up after two."""
    n = 700_000_037
    x = torch.ones(n, 8, dtype=BF16, device="cuda")
    x[-1] = 4096.0
    moe.check_operators()
    dw = moe.grouped_product_weight_gradients(x, x, device_counts([0] * 79 + [n]), dtype=F32)
    moe.check_operators()
    assert not dw[:-1].any()
    ref = n - 1 + 4096.0**2
    assert float((dw[-1].double() / ref - 1).abs().max()) <= 17 * 2.0**-24
