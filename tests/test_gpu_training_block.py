"""The operators together, as a training step uses them: a block x +
dropout(experts(layer_norm(x))), forward and backward.

Float64 rows throughout, so the only differences to the restatement are
summation orders: relative 1e-9, as for gtmoe_backward."""
import numpy as np
import pytest
import torch

import operators_ref as R
from gotransformers_b200 import _lib, moe
from gpu_helpers import TOL, gpu_moe, rel_l2
from moe_cases import make_case
from oracle import oracle as O

pytestmark = pytest.mark.gpu
TOL_STEP = 1e-9


def norm_params(d, seed):
    g = torch.Generator().manual_seed(seed)
    return (1 + 0.2 * torch.randn(d, generator=g, dtype=torch.float64),
            0.3 * torch.randn(d, generator=g, dtype=torch.float64))


def test_block_around_frozen_experts():
    """layer_norm -> MixtureOfExperts -> dropout with the residual, and back
    through dropout_backward, MixtureOfExperts.backward and
    layer_norm_backward with the residual's gradients."""
    T, d, rate, seed, step, eps = 96, 256, 0.2, 17, 4, 1e-5
    spec, x, _ = make_case(T=T, d=d, h=128, n_shared=1, n_routed=8, k=2, precision=O.INT8, seed=31)
    w, b = norm_params(d, 5)
    dout = torch.from_numpy(np.random.default_rng(6).standard_normal((T, d)))
    xt = torch.from_numpy(x)

    xn, _, _ = R.layer_norm(xt, w, b, eps)
    ref = O.moe_forward(spec, xn.numpy(), None, threads=4)
    dmoe = R.dropout(dout, rate, seed, step)
    back = O.moe_backward(spec, xn.numpy(), dmoe.numpy())
    dx, dw, db = R.layer_norm_backward(torch.from_numpy(back["dx"]), xt, w, eps, dout)

    m = gpu_moe(spec)
    s = torch.cuda.Stream()
    m.set_stream(s.cuda_stream)
    m.set_training(True)
    with torch.cuda.stream(s):
        X, W, B, D = xt.cuda(), w.cuda(), b.cuda(), dout.cuda()
        gn, mean, rstd = moe.layer_norm(X, W, B, eps)
        y = m.forward(gn)
        out = moe.dropout(y, rate, seed, step, residual=X)
        gdx = m.backward(moe.dropout_backward(D, rate, seed, step))
        gx, gw, gb = moe.layer_norm_backward(gdx, X, mean, rstd, W, residual_gradients=D)
    torch.cuda.synchronize()
    assert np.array_equal(m.last_chosen_experts, ref["chosen"])
    assert rel_l2(gn.cpu().numpy(), xn.numpy()) <= TOL_STEP
    # the experts' forward runs on bfloat16 rows: its own tolerance
    want = R.dropout(torch.from_numpy(ref["out"]), rate, seed, step)
    assert rel_l2((out - X).cpu().numpy(), want.numpy()) <= TOL[O.INT8]
    assert rel_l2(gx.cpu().numpy(), dx.numpy()) <= TOL_STEP
    assert rel_l2(gw.cpu().numpy(), dw.numpy()) <= TOL_STEP
    assert rel_l2(gb.cpu().numpy(), db.numpy()) <= TOL_STEP
    m.close()


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16])
def test_block_with_trained_experts(dtype):
    """The mixture routes; dense SwiGLU experts run as grouped products over
    its permutation and load, with every gradient, against autograd of the
    restated block in float64 from the same rounded inputs."""
    T, d, hd, E, k, rate, seed, step, eps = 150, 64, 96, 6, 2, 0.25, 3, 9, 1e-5
    g = torch.Generator().manual_seed(8)

    def rand(*s, scale=1.0):
        return (scale * torch.randn(*s, generator=g, dtype=torch.float64)).to(dtype)

    x, dout = rand(T, d), rand(T, d)
    wg, wu, wd = rand(E, hd, d, scale=d**-0.5), rand(E, hd, d, scale=d**-0.5), rand(E, d, hd, scale=hd**-0.5)
    w, b = (t.to(dtype) for t in norm_params(d, 9))

    # the mixture's routing of the normalized rows
    spec, _, _ = make_case(T=4, d=d, h=32, n_shared=0, n_routed=E, k=k, precision=O.FLOAT32, seed=12)
    m = gpu_moe(spec)
    s = torch.cuda.Stream()
    m.set_stream(s.cuda_stream)
    with torch.cuda.stream(s):
        X, W, B, D = x.cuda(), w.cuda(), b.cuda(), dout.cuda()
        WG, WU, WD = wg.cuda(), wu.cuda(), wd.cuda()
        xn, mean, rstd = moe.layer_norm(X, W, B, eps)
        m.forward(xn)
        perm = torch.from_numpy(m.last_rows_for_expert).long()
        load = torch.from_numpy(m.last_expert_load())
        chosen, gates = torch.from_numpy(m.last_chosen_experts).long(), torch.from_numpy(m.last_gates)
        expert = torch.repeat_interleave(torch.arange(E), load)
        slot = (chosen[perm] == expert[:, None]).long().argmax(1)
        gate = gates[perm, slot]
        P, L, G = perm.cuda(), load.cuda(), gate.cuda().to(dtype)[:, None]

        xp = xn[P].contiguous()
        a, u = moe.grouped_product(xp, WG, L), moe.grouped_product(xp, WU, L)
        sg = torch.sigmoid(a)
        hid = (a * sg * u).contiguous()
        y = moe.grouped_product(hid, WD, L)
        mix = torch.zeros_like(X).index_add_(0, P, y * G)
        out = moe.dropout(mix, rate, seed, step, residual=X)

        dmix = moe.dropout_backward(D, rate, seed, step)
        dy = (dmix[P] * G).contiguous()
        dhid = moe.grouped_product_input_gradients(dy, WD, L)
        dwd = moe.grouped_product_weight_gradients(dy, hid, L)
        da = (dhid * u * sg * (1 + a * (1 - sg))).contiguous()
        du = (dhid * a * sg).contiguous()
        dxp = moe.grouped_product_input_gradients(da, WG, L) + moe.grouped_product_input_gradients(du, WU, L)
        dwg, dwu = moe.grouped_product_weight_gradients(da, xp, L), moe.grouped_product_weight_gradients(du, xp, L)
        dxn = torch.zeros_like(X).index_add_(0, P, dxp)
        dx, dw, db = moe.layer_norm_backward(dxn, X, mean, rstd, W, residual_gradients=D)
    torch.cuda.synchronize()
    moe.check_operators()
    m.close()

    leaves = [t.double().requires_grad_() for t in (x, w, b, wg, wu, wd)]
    lx, lw, lb, lwg, lwu, lwd = leaves
    rn = R.layer_norm(lx, lw, lb, eps)[0]
    rp = rn[perm]
    parts, r = [], 0
    for e, n in enumerate(load.tolist()):
        rows = rp[r:r + n]
        ra = rows @ lwg[e].T
        parts.append((ra * torch.sigmoid(ra) * (rows @ lwu[e].T)) @ lwd[e].T)
        r += n
    rmix = torch.zeros(T, d, dtype=torch.float64).index_add(0, perm, torch.cat(parts) * gate[:, None])
    rout = lx + torch.where(R.keep(T * d, rate, seed, step).reshape(T, d), rmix / (1 - rate), 0.0)
    rout.backward(dout.double())
    # a value passes at most 16 roundings of the type (HALF each) and sums of up to 150 terms in UNIT between
    # input and output; roundings of one type add up in the 2-norm at most linearly
    tol = 16 * R.HALF[dtype] + 16 * 160 * R.UNIT[dtype]
    R.near("out", out, rout.detach(), tol)
    for name, got, leaf in zip(("dx", "dw", "db", "dwg", "dwu", "dwd"), (dx, dw, db, dwg, dwu, dwd), leaves):
        R.near(name, got, leaf.grad, tol)


@pytest.mark.parametrize("on_device", [True, False])
@pytest.mark.parametrize("prec,T,dtype", [(O.INT8, 40, torch.float32), (O.FP4, 300, torch.bfloat16),
                                          (O.FLOAT32, 17, torch.float64)])
def test_block_step_with_dropout(prec, T, dtype, on_device):
    """gtmoe_forward_block with a rate: the mixture's part of the block step
    goes through dropout()'s decisions; rate 0 gives the old step's bits."""
    if dtype == torch.bfloat16 and not on_device:
        pytest.skip("host rows are float64 or float32")
    spec, x, ids = make_case(T=T, d=256, h=128, n_shared=1, n_routed=8, k=2, precision=prec, seed=73)
    rate, seed, step = 0.3, 21, 6
    m = gpu_moe(spec)
    s = torch.cuda.Stream()
    m.set_stream(s.cuda_stream)
    m.set_norm(1.0 + 0.1 * np.random.default_rng(2).standard_normal(spec.d), 1e-6)
    xt = torch.from_numpy(x).to(dtype)
    with torch.cuda.stream(s):
        rows = xt.cuda() if on_device else xt.numpy()

        def block():
            out = m.forward_block(rows, ids)
            return out.cpu() if on_device else torch.from_numpy(out)

        plain = block()
        chosen = m.last_chosen_experts.copy()
        for step in (6, 7):
            m.set_dropout(rate, seed, step)
            got = block()
            assert np.array_equal(m.last_chosen_experts, chosen)
            kept = R.keep(T * spec.d, rate, seed, step).reshape(T, spec.d)
            assert torch.equal(got[~kept], xt[~kept])  # the residual alone
            # kept: the mixture's output (rounded to the type) over 1 - rate, plus x, against the old step's (out - x),
            # which was rounded with x added: a few roundings of the type each, float32 sums in between
            mix = plain.double() - xt.double()
            want = xt.double() + mix / (1 - rate)
            h = R.HALF[dtype] if dtype != torch.float64 else 2.0**-24  # expert outputs are float32
            tol = 4 * h * (want.abs() + plain.double().abs() + xt.double().abs())
            R.within("out", torch.where(kept, got.double(), want), want, tol)
        m.set_dropout(0.0)
        assert torch.equal(block(), plain)
    with pytest.raises(_lib.GtmoeError):
        m.set_dropout(1.0)
    m.close()


@pytest.mark.parametrize("other", [1.0, [1.0] * 64, np.ones(64, np.float32)], ids=["number", "list", "array"])
def test_parameters_that_are_no_tensors_are_refused(other):
    """ValueError, as for every other misuse, wherever a tensor is expected."""
    x = torch.ones(8, 64, device="cuda")
    counts = torch.tensor([8], device="cuda")
    w = torch.ones(64, device="cuda")
    y, mean, rstd = moe.layer_norm(x, w, w)
    calls = [
        lambda: moe.layer_norm(other),
        lambda: moe.layer_norm(x, other, w),
        lambda: moe.layer_norm(x, w, other),
        lambda: moe.layer_norm(x, None, other),
        lambda: moe.layer_norm(x, w, w, out=other),
        lambda: moe.layer_norm_backward(y, x, mean, rstd, other),
        lambda: moe.layer_norm_backward(y, x, other, rstd, w),
        lambda: moe.layer_norm_backward(y, x, mean, rstd, None, None, None, other, other),
        lambda: moe.layer_norm_backward(y, x, mean, rstd, w, residual_gradients=other),
        lambda: moe.dropout(x, 0.5, 1, residual=other),
        lambda: moe.grouped_product(x, other, counts),
        lambda: moe.grouped_product(x, torch.ones(1, 64, 64, device="cuda"), other),
        lambda: moe.grouped_product_weight_gradients(y, x, other),
        lambda: moe.grouped_product_weight_gradients(y, x, counts, other),
    ]
    for call in calls:
        with pytest.raises(ValueError):
            call()
