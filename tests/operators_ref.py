"""Float64 restatements of the handle-less operators, and the tolerances the
GPU results are held to.

A rounding is off by at most half a step, relative to the value: HALF below.
Sums of n terms made in float32 are off by at most (additions in a row) *
2^-24 * (sum of the terms' magnitudes)."""
import numpy as np
import torch

HALF = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24, torch.float64: 2.0**-53}
# one step of the type the sums are made in
UNIT = {torch.bfloat16: 2.0**-24, torch.float32: 2.0**-24, torch.float64: 2.0**-53}
M64 = (1 << 64) - 1


def layer_norm(x, w, b, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    y = (x - mean) * rstd
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    return y, mean[:, 0], rstd[:, 0]


def layer_norm_backward(dy, x, w, eps, dres=None):
    dy, x = dy.double(), x.double()
    _, mean, rstd = layer_norm(x, None, None, eps)
    xh = (x - mean[:, None]) * rstd[:, None]
    g = dy if w is None else dy * w.double()
    dx = rstd[:, None] * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    if dres is not None:
        dx = dx + dres.double()
    return dx, (dy * xh).sum(0), dy.sum(0)


def split_mix64(z):
    with np.errstate(over="ignore"):
        z = z + np.uint64(0x9E3779B97F4A7C15)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        return z ^ (z >> np.uint64(31))


def keep(n, rate, seed, stream=0, offset=0):
    """keep(i) of elements offset .. offset + n - 1."""
    key = split_mix64(np.array([(seed & M64) ^ ((stream * 0xD1B54A32D192ED03) & M64)], np.uint64))[0]
    e = np.arange(n, dtype=np.uint64) + np.uint64(offset)
    with np.errstate(over="ignore"):
        word = split_mix64(key + (e >> np.uint64(1)))
    half = np.where(e & np.uint64(1), word >> np.uint64(32), word & np.uint64(0xFFFFFFFF))
    return torch.from_numpy(half >= np.uint64(int(rate * 2.0**32)))


def dropout(x, rate, seed, stream=0, offset=0, residual=None):
    k = keep(x.numel(), rate, seed, stream, offset).reshape(x.shape)
    y = torch.where(k, x.double() / (1 - rate), torch.zeros((), dtype=torch.float64))
    return y if residual is None else y + residual.double()


def _parts(counts):
    r = 0
    for g, m in enumerate(counts):
        yield g, slice(r, r + m)
        r += m


def grouped(x, w, counts):
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64)
    for g, s in _parts(counts):
        y[s] = x[s].double() @ w[g].double().T
    return y


def grouped_input_gradients(dy, w, counts):
    dx = torch.zeros(dy.shape[0], w.shape[2], dtype=torch.float64)
    for g, s in _parts(counts):
        dx[s] = dy[s].double() @ w[g].double()
    return dx


def grouped_weight_gradients(dy, x, counts):
    dw = torch.zeros(len(counts), dy.shape[1], x.shape[1], dtype=torch.float64)
    for g, s in _parts(counts):
        dw[g] = dy[s].double().T @ x[s].double()
    return dw


def within(name, got, ref, tol):
    """Every element of got is within tol (a tensor or number) of ref."""
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    assert torch.isfinite(got).all(), f"{name} has values that are not finite"
    over = (got - ref).abs() - tol
    assert (over <= 0).all(), f"{name}: off by {float((got - ref).abs().max()):.3e}, {int((over > 0).sum())} values past the tolerance"


def near(name, got, ref, tol):
    """The 2-norm of the error is within tol of the reference's."""
    got = got.detach().cpu().double()
    err = float((got - ref).norm()) / max(float(ref.norm()), 1e-300)
    assert err <= tol, f"{name}: relative error {err:.3e} above {tol:.3e}"
