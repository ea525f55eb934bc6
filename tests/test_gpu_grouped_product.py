"""The products of rows grouped by expert and the gradients of both factors,
on the GPU against the float64 restatement.

Sums of small whole numbers are exact in float32 whatever their order, so on
such inputs a result has to equal the restatement's, rounded once.  On normal
inputs a sum of n products is off by at most n units of the products'
magnitudes (the tensor cores may cut each addition instead of rounding it: a
unit is 2^-23 for bfloat16 operands)."""
import pytest
import torch

import operators_ref as R
from gotransformers_b200 import _lib, moe

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
UNIT = {BF16: 2.0**-23, F32: 2.0**-24, F64: 2.0**-53}


def make(counts, inputs, outputs, dtype, seed=0, whole=False, extra=0):
    g = torch.Generator().manual_seed(seed)
    rows, groups = sum(counts) + extra, len(counts)

    def rand(*s):
        if whole:
            return torch.randint(-4, 5, s, generator=g).to(dtype)
        return torch.randn(*s, generator=g, dtype=torch.float64).to(dtype)

    return rand(rows, inputs), rand(groups, outputs, inputs), rand(rows, outputs)


def device_counts(counts):
    return torch.tensor(counts, dtype=torch.int64, device="cuda")


def check_exact(counts, inputs, outputs, dtype, wdtype=None, seed=0):
    """Whole numbers: the results are the restatement's, rounded once."""
    x, w, dy = make(counts, inputs, outputs, dtype, seed, whole=True)
    X, W, DY, C = x.cuda(), w.cuda(), dy.cuda(), device_counts(counts)
    wdtype = wdtype or dtype
    y = moe.grouped_product(X, W, C).cpu()
    dx = moe.grouped_product_input_gradients(DY, W, C).cpu()
    dw = moe.grouped_product_weight_gradients(DY, X, C, dtype=wdtype).cpu()
    assert torch.equal(y, R.grouped(x, w, counts).to(dtype)), "y"
    assert torch.equal(dx, R.grouped_input_gradients(dy, w, counts).to(dtype)), "dx"
    assert torch.equal(dw, R.grouped_weight_gradients(dy, x, counts).to(wdtype)), "dw"
    moe.check_operators()


def check_normal(counts, inputs, outputs, dtype, wdtype=None, seed=0):
    x, w, dy = make(counts, inputs, outputs, dtype, seed)
    X, W, DY, C = x.cuda(), w.cuda(), dy.cuda(), device_counts(counts)
    wdtype = wdtype or dtype
    u, h = UNIT[dtype], R.HALF[dtype]

    def hold(name, got, ref, mag, n, half):
        R.within(name, got, ref, half * ref.abs() + (n + 2) * u * mag * (1 + half))

    hold("y", moe.grouped_product(X, W, C), R.grouped(x, w, counts), R.grouped(x.abs(), w.abs(), counts), inputs, h)
    hold("dx", moe.grouped_product_input_gradients(DY, W, C), R.grouped_input_gradients(dy, w, counts),
         R.grouped_input_gradients(dy.abs(), w.abs(), counts), outputs, h)
    hold("dw", moe.grouped_product_weight_gradients(DY, X, C, dtype=wdtype), R.grouped_weight_gradients(dy, x, counts),
         R.grouped_weight_gradients(dy.abs(), x.abs(), counts), max(counts), R.HALF[wdtype])
    moe.check_operators()


COUNTS = [
    [1], [0, 1, 0], [5, 0, 3], [0, 0], [7, 8, 9, 15, 16, 17], [63, 64, 65], [127, 128, 129, 1], [255, 0, 257],
    [300, 1, 2, 0, 700], [513], [16] * 20,
]


@pytest.mark.parametrize("counts", COUNTS, ids=str)
@pytest.mark.parametrize("dtype,wdtype", [(BF16, BF16), (BF16, F32), (F32, F32), (F64, F64)])
def test_whole_numbers_over_counts(counts, dtype, wdtype):
    check_exact(counts, 192, 320, dtype, wdtype, seed=len(counts))


@pytest.mark.parametrize("inputs,outputs", [
    (8, 8), (16, 8), (8, 264), (64, 64), (72, 40), (120, 128), (128, 136), (256, 256), (264, 520), (512, 248),
    (1000, 88), (96, 1032), (1, 1), (3, 5), (65, 64), (64, 65), (100, 31), (257, 515),
])
@pytest.mark.parametrize("dtype,wdtype", [(BF16, F32), (F32, F32)])
def test_whole_numbers_over_sizes(inputs, outputs, dtype, wdtype):
    check_exact([70, 0, 259, 33], inputs, outputs, dtype, wdtype, seed=inputs)


@pytest.mark.parametrize("dtype,wdtype", [(BF16, BF16), (BF16, F32), (F32, F32), (F64, F64)])
def test_normal_values(dtype, wdtype):
    check_normal([37, 0, 300, 129], 264, 200, dtype, wdtype)
    check_normal([40, 3], 101, 77, dtype, wdtype)


def test_long_sums():
    """A reduction long enough for every ring of buffers to go around many times, in each direction."""
    check_exact([2000, 3001], 264, 520, BF16, F32)
    check_exact([20, 300], 4104, 264, BF16, F32)
    check_exact([20, 300], 264, 4104, BF16, F32)


@pytest.mark.parametrize("counts", [[5000], [3000, 5001], [0, 9000, 1, 0], [2049, 512, 4096, 7000], [16384]], ids=str)
@pytest.mark.parametrize("inputs,outputs", [(256, 256), (72, 264), (520, 40)])
def test_weight_gradients_whose_sums_are_split(counts, inputs, outputs):
    """Few tiles and many rows: parts of a group in units of their own, added by a second kernel."""
    assert outputs * inputs <= 1 << 17
    check_exact(counts, inputs, outputs, BF16, F32)
    check_exact(counts, inputs, outputs, BF16, BF16)
    x, _, dy = make(counts, inputs, outputs, BF16, 3, whole=True)
    ref = R.grouped_weight_gradients(dy, x, counts)
    for dtype in (F32, BF16):
        before = torch.randint(-9, 10, ref.shape).to(dtype)
        dw = before.cuda()
        moe.grouped_product_weight_gradients(dy.cuda(), x.cuda(), device_counts(counts), weight_grad=dw)
        assert torch.equal(dw.cpu(), (ref + before.double()).to(dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_split_and_whole_groups_added_to(dtype):
    """One CTA pair's units go back and forth between parts of a split group,
    which TMA stores, and groups that are added to from shared memory: the two
    share the epilogue's buffers."""
    counts = [9000, 5, 300, 7001, 64, 1, 8192, 700, 4097, 2]
    x, _, dy = make(counts, 520, 264, BF16, 21, whole=True)
    X, DY, C = x.cuda(), dy.cuda(), device_counts(counts)
    ref = R.grouped_weight_gradients(dy, x, counts)
    before = torch.randint(-9, 10, ref.shape).to(dtype)
    want = (ref + before.double()).to(dtype)
    for _ in range(20):
        dw = before.cuda()
        moe.grouped_product_weight_gradients(DY, X, C, weight_grad=dw)
        assert torch.equal(dw.cpu(), want)


@pytest.mark.parametrize("rows,groups", [(1536, 1), (65536, 1), (20000, 3), (40000, 80)])
def test_float32_weight_gradients_keep_their_digits(rows, groups):
    """Runs of 768 rows are 48 additions that cut at most 2^-23 of the sum
    each; the runs (at most 86) are added with rounding.  Relative to the sums
    themselves, which random terms bring to about the same size as any part's:
    48 * 2^-23 + 86 * 2^-24.  One run over 65536 rows would lose 6.6e-5."""
    counts = [rows // groups] * groups
    x, _, dy = make(counts, 64, 72, BF16, 17)
    dw = moe.grouped_product_weight_gradients(dy.cuda(), x.cuda(), device_counts(counts), dtype=F32)
    R.near("dw", dw, R.grouped_weight_gradients(dy, x, counts), 48 * 2.0**-23 + 86 * 2.0**-24)


def positive(rows, columns, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (0.75 + 0.5 * torch.rand(rows, columns, generator=g, device="cuda")).to(BF16)


def test_bfloat16_weight_gradients_of_long_groups():
    """Values of one sign, whose sums lose the most where additions are cut: a
    million rows in one sum would be 7.0e-3 short.  In runs of 768 rows it is
    48 cut additions of at most 2^-23 and 1366 rounded ones, then the rounding
    to bfloat16.  80 groups: the sums are not split."""
    counts = [(1 << 20) + 37, 5] + [0] * 77 + [70000]
    x, dy = positive(sum(counts), 64, 1), positive(sum(counts), 72, 2)
    for dtype in (BF16, F32):
        dw = moe.grouped_product_weight_gradients(dy, x, device_counts(counts), dtype=dtype)
        at = 0
        for g, n in enumerate(counts):
            ref = dy[at:at + n].double().T @ x[at:at + n].double()
            at += n
            tol = R.HALF[dtype] + 48 * 2.0**-23 + 1367 * 2.0**-24
            R.within(f"dw[{g}]", dw[g].cpu(), ref.cpu(), tol * ref.abs().cpu())
    moe.check_operators()


@pytest.mark.parametrize("direction", ["product", "input gradients"])
def test_sums_over_very_long_rows(direction):
    """A million products of one sign per value.  Rounded additions err
    independently: beyond 8 * sqrt(n) * 2^-24 of the sum with a probability of
    2 exp(-32) per value (one sum on the tensor cores would be 7e-3 short)."""
    n, counts = 1 << 20, [3, 29]
    x, w = positive(32, n, 3), positive(2 * 8, n, 4).view(2, 8, n)
    if direction == "product":
        y = moe.grouped_product(x, w, device_counts(counts))
    else:
        y = moe.grouped_product_input_gradients(x, w.transpose(1, 2).contiguous(), device_counts(counts))
    for g, r in ((0, slice(0, 3)), (1, slice(3, 32))):
        ref = x[r].double() @ w[g].double().T
        R.within("y", y[r].cpu(), ref.cpu(), (R.HALF[BF16] + 8 * 2.0**10 * 2.0**-24) * ref.abs().cpu())
    moe.check_operators()


def test_many_groups():
    g = torch.Generator().manual_seed(8)
    counts = torch.randint(0, 6, (1024,), generator=g).tolist()
    check_exact(counts, 64, 72, BF16, F32)
    check_exact(counts, 20, 9, F32)
    check_exact(torch.randint(0, 300, (100,), generator=g).tolist(), 136, 264, BF16)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_accumulation(dtype):
    counts = [30, 0, 200]
    x, _, dy = make(counts, 136, 264, dtype, 3, whole=True)
    C = device_counts(counts)
    before = torch.randint(-9, 10, (3, 264, 136)).float()
    dw = before.cuda()
    assert moe.grouped_product_weight_gradients(dy.cuda(), x.cuda(), C, weight_grad=dw) is dw
    assert torch.equal(dw.cpu(), (R.grouped_weight_gradients(dy, x, counts) + before).float())
    if dtype == BF16:
        dw = before.to(BF16).cuda()
        moe.grouped_product_weight_gradients(dy.cuda(), x.cuda(), C, weight_grad=dw)
        assert torch.equal(dw.cpu(), (R.grouped_weight_gradients(dy, x, counts) + before).to(BF16))


@pytest.mark.parametrize("inputs,outputs", [(128, 264), (60, 33)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_after_the_last_group(inputs, outputs, dtype):
    """They hold NaN, are not read, and the outputs' rows stay as they were."""
    counts, extra = [50, 0, 121], 90
    x, w, dy = make(counts, inputs, outputs, dtype, 4, whole=True, extra=extra)
    n = sum(counts)
    x[n:], dy[n:] = float("nan"), float("nan")
    X, W, DY, C = x.cuda(), w.cuda(), dy.cuda(), device_counts(counts)
    y = torch.full((n + extra, outputs), 7.0, dtype=dtype, device="cuda")
    dx = torch.full((n + extra, inputs), 7.0, dtype=dtype, device="cuda")
    moe.grouped_product(X, W, C, out=y)
    moe.grouped_product_input_gradients(DY, W, C, input_gradients=dx)
    dw = moe.grouped_product_weight_gradients(DY, X, C)
    assert (y[n:] == 7).all() and (dx[n:] == 7).all()
    assert torch.equal(y[:n].cpu(), R.grouped(x[:n], w, counts).to(dtype))
    assert torch.equal(dx[:n].cpu(), R.grouped_input_gradients(dy[:n], w, counts).to(dtype))
    assert torch.equal(dw.cpu(), R.grouped_weight_gradients(dy[:n], x[:n], counts).to(dtype))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_not_a_number_stays_in_its_group(dtype):
    """A group's NaN and infinities reach no other group: not through tiles
    that its rows or weights share with their neighbours'."""
    counts, inputs, outputs = [40, 33, 50], 200, 136
    x, w, dy = make(counts, inputs, outputs, dtype, 5, whole=True)
    ref = make(counts, inputs, outputs, dtype, 5, whole=True)
    s = slice(40, 73)
    x[s], dy[s], w[1] = float("nan"), float("inf"), float("nan")
    X, W, DY, C = x.cuda(), w.cuda(), dy.cuda(), device_counts(counts)
    y, dx = moe.grouped_product(X, W, C).cpu(), moe.grouped_product_input_gradients(DY, W, C).cpu()
    dw = moe.grouped_product_weight_gradients(DY, X, C).cpu()
    ry, rdx = R.grouped(ref[0], ref[1], counts).to(dtype), R.grouped_input_gradients(ref[2], ref[1], counts).to(dtype)
    rdw = R.grouped_weight_gradients(ref[2], ref[0], counts).to(dtype)
    keep = torch.ones(123, dtype=torch.bool)
    keep[s] = False
    assert torch.equal(y[keep], ry[keep]) and torch.equal(dx[keep], rdx[keep])
    assert torch.equal(dw[[0, 2]], rdw[[0, 2]])
    assert torch.isnan(y[s]).all() and torch.isnan(dx[s]).all() and torch.isnan(dw[1]).all()


def test_impossible_counts_are_reported_and_stay_in_bounds():
    x, w, dy = make([100], 64, 72, BF16, 6, whole=True)
    w = w.repeat(3, 1, 1)
    X, W, DY = x.cuda(), w.cuda(), dy.cuda()
    moe.check_operators()
    for counts in ([50, -3, 20], [60, 70, 80], [1 << 40, 1 << 62, 5], [(1 << 63) - 1, (1 << 63) - 1, 1]):
        C = device_counts(counts)
        for call in (lambda: moe.grouped_product(X, W, C), lambda: moe.grouped_product_input_gradients(DY, W, C),
                     lambda: moe.grouped_product_weight_gradients(DY, X, C)):
            call()
            with pytest.raises(_lib.GtmoeError) as e:
                moe.check_operators()
            assert e.value.code == -1
            moe.check_operators()  # cleared
    # and on the SIMT cores
    moe.grouped_product(X.float(), W.float(), device_counts([-1, 5, 5]))
    with pytest.raises(_lib.GtmoeError):
        moe.check_operators()


@pytest.mark.parametrize("shift", [1, 4])
def test_addresses_that_start_on_an_element(shift):
    counts = [33, 90]
    x, w, dy = make(counts, 128, 72, BF16, 7, whole=True)

    def shifted(t):
        v = torch.empty(t.numel() + shift, dtype=t.dtype, device="cuda")[shift:].view(t.shape)
        v.copy_(t)
        return v

    X, W, DY, C = shifted(x), shifted(w), shifted(dy), device_counts(counts)
    y = moe.grouped_product(X, W, C, out=shifted(dy))
    dx = moe.grouped_product_input_gradients(DY, W, C, input_gradients=shifted(x))
    dw = moe.grouped_product_weight_gradients(DY, X, C)
    assert torch.equal(y.cpu(), R.grouped(x, w, counts).to(BF16))
    assert torch.equal(dx.cpu(), R.grouped_input_gradients(dy, w, counts).to(BF16))
    assert torch.equal(dw.cpu(), R.grouped_weight_gradients(dy, x, counts).to(BF16))


def test_no_rows():
    x, w, dy = make([0, 0], 64, 72, BF16)
    C = device_counts([0, 0])
    assert moe.grouped_product(x.cuda(), w.cuda(), C).shape == (0, 72)
    assert moe.grouped_product_input_gradients(dy.cuda(), w.cuda(), C).shape == (0, 64)
    dw = moe.grouped_product_weight_gradients(dy.cuda(), x.cuda(), C, dtype=F32)
    assert dw.shape == (2, 72, 64) and not dw.any()
    dw = torch.ones(2, 72, 64, device="cuda")
    moe.grouped_product_weight_gradients(dy.cuda(), x.cuda(), C, weight_grad=dw)
    assert (dw == 1).all()
    moe.check_operators()


def test_results_repeat():
    counts = [500, 20, 700]
    x, w, dy = make(counts, 264, 520, BF16, 9)
    X, W, DY, C = x.cuda(), w.cuda(), dy.cuda(), device_counts(counts)

    def all_three():
        return (moe.grouped_product(X, W, C), moe.grouped_product_input_gradients(DY, W, C),
                moe.grouped_product_weight_gradients(DY, X, C, dtype=F32))

    ref = all_three()
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(all_three(), ref))


def test_differences_in_float64():
    """Central differences of step 1e-6 of the GPU's float64 product."""
    counts = [9, 0, 17]
    x, w, dy = make(counts, 24, 40, F64, 10)
    vx, vw, _ = make(counts, 24, 40, F64, 11)
    X, W, DY, VX, VW, C = x.cuda(), w.cuda(), dy.cuda(), vx.cuda(), vw.cuda(), device_counts(counts)
    h = 1e-6

    def f(x, w):
        return float((moe.grouped_product(x, w, C) * DY).sum())

    dx = moe.grouped_product_input_gradients(DY, W, C)
    dw = moe.grouped_product_weight_gradients(DY, X, C)
    # values around 200, so rounding leaves 200 * 2^-53 * (terms in a row) / 1e-6 < 1e-5
    assert abs((f(X + h * VX, W) - f(X - h * VX, W)) / (2 * h) - float((dx * VX).sum())) < 1e-5
    assert abs((f(X, W + h * VW) - f(X, W - h * VW)) / (2 * h) - float((dw * VW).sum())) < 1e-5


def test_graphs_and_streams():
    """Two captured graphs replayed at once, with new counts in the same tensor, beside an eager call."""
    counts, later = [200, 0, 350, 50], [100, 300, 0, 200]
    x, w, dy = make(counts, 264, 136, BF16, 12, whole=True)
    X, W, DY, C = x.cuda(), w.cuda(), dy.cuda(), device_counts(counts)
    moe.grouped_product(X, W, C)
    torch.cuda.synchronize()
    runs = []
    for _ in range(2):
        s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = (moe.grouped_product(X, W, C), moe.grouped_product_input_gradients(DY, W, C),
                   moe.grouped_product_weight_gradients(DY, X, C, dtype=F32))
        runs.append((s, graph, out))
    for now in (counts, later):
        C.copy_(device_counts(now))
        torch.cuda.synchronize()
        for _ in range(3):
            for s, graph, _ in runs:
                with torch.cuda.stream(s):
                    graph.replay()
        eager = moe.grouped_product(X, W, C)
        torch.cuda.synchronize()
        ref = (R.grouped(x, w, now).to(BF16), R.grouped_input_gradients(dy, w, now).to(BF16),
               R.grouped_weight_gradients(dy, x, now).float())
        assert torch.equal(eager.cpu(), ref[0])
        for _, _, out in runs:
            assert all(torch.equal(p.cpu(), q) for p, q in zip(out, ref))
    moe.check_operators()


def test_weights_past_2_to_31_values():
    groups, outputs, inputs = 130, 4096, 4104
    w = torch.zeros(groups, outputs, inputs, dtype=BF16, device="cuda")
    counts = [0] * groups
    counts[0], counts[-1] = 3, 40
    x, wl, dy = make([40], inputs, outputs, BF16, 13, whole=True)
    w[-1] = wl[0].cuda()
    X = torch.cat([x[:3], x]).cuda()
    DY = torch.cat([dy[:3], dy]).cuda()
    C = device_counts(counts)
    assert torch.equal(moe.grouped_product(X, w, C)[3:].cpu(), R.grouped(x, wl, [40]).to(BF16))
    assert torch.equal(moe.grouped_product_input_gradients(DY, w, C)[3:].cpu(),
                       R.grouped_input_gradients(dy, wl, [40]).to(BF16))
    dw = moe.grouped_product_weight_gradients(DY, X, C, weight_grad=w)[-1].cpu()
    assert torch.equal(dw, (R.grouped_weight_gradients(dy, x, [40])[0] + wl[0].double()).to(BF16))
    assert not w[1:-1].any()


def test_refusals():
    x, w, dy = (t.cuda() for t in make([10], 16, 24, BF16))
    C = device_counts([10])
    with pytest.raises(ValueError):
        moe.grouped_product(x, w.float(), C)
    with pytest.raises(ValueError):
        moe.grouped_product(x, w[:, :, :8].contiguous(), C)
    with pytest.raises(ValueError):
        moe.grouped_product(x, w, C.int())
    with pytest.raises(ValueError):
        moe.grouped_product(x, w, C.cpu())
    with pytest.raises(ValueError):
        moe.grouped_product(x, w, device_counts([5, 5]))
    with pytest.raises(ValueError):
        moe.grouped_product(x.T, w, C)
    with pytest.raises(ValueError):
        moe.grouped_product_weight_gradients(dy[:5], x, C)
    with pytest.raises(_lib.GtmoeError):
        moe.grouped_product_weight_gradients(dy, x, C, dtype=F64)
    with pytest.raises(_lib.GtmoeError):
        moe.grouped_product_weight_gradients(dy.float(), x.float(), C, dtype=BF16)
    square = torch.zeros(8, 8, dtype=BF16, device="cuda")
    with pytest.raises(_lib.GtmoeError):
        moe.grouped_product(square, torch.zeros(1, 8, 8, dtype=BF16, device="cuda"), device_counts([8]), out=square)
