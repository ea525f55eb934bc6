"""The training operators of a mixture-of-experts block, as cases to be measured.

Three operators, each in its plain form (elementary torch operations in 32 bits, rounded once at the end) and as this
package's calls:

* ``layer_norm``: y = (x - mean) * rstd * weight + bias over each row, and its backward: the input gradients (with the
  block's residual gradients added) and the weight and bias gradients, summed over the rows;
* ``dropout``: residual + x * keep / (1 - rate), where the keep decision of element i is a function of (seed, stream,
  i) alone, and its backward, which makes the same decisions again;
* ``grouped``: the matrix products of rows sorted by expert with each expert's own dense weights (outputs x inputs),
  and the gradients of both factors.

A case's ``train`` says whether a pass is the forward alone or the forward with the whole backward."""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one decoding step of a few sequences: latency
        {"name": "norm_step", "op": "layer_norm", "train": False, "dtype": "bf16", "wdtype": "bf16", "rows": 8,
         "width": 2048, "residual": False},
        # a small float32 model with an odd width, trained: every reduction over ragged rows
        {"name": "norm_odd_f32", "op": "layer_norm", "train": True, "dtype": "f32", "wdtype": "f32", "rows": 777,
         "width": 1001, "residual": False},
        # a training step of the 2048-wide block: forward, then the backward with the residual's gradients added
        {"name": "norm_train", "op": "layer_norm", "train": True, "dtype": "bf16", "wdtype": "f32", "rows": 16384,
         "width": 2048, "residual": True},
        # the 4096-wide block on a large batch
        {"name": "norm_train_large", "op": "layer_norm", "train": True, "dtype": "bf16", "wdtype": "bf16",
         "rows": 65536, "width": 4096, "residual": True},
        # the 256-wide float32 layer's batch of 512 tokens: latency
        {"name": "dropout_small", "op": "dropout", "train": False, "dtype": "f32", "rows": 512, "width": 256,
         "rate": 0.1, "residual": True},
        # a training step of the 2048-wide block
        {"name": "dropout_train", "op": "dropout", "train": True, "dtype": "bf16", "rows": 16384, "width": 2048,
         "rate": 0.1, "residual": True},
        # the 4096-wide block on a large batch
        {"name": "dropout_train_large", "op": "dropout", "train": True, "dtype": "bf16", "rows": 65536, "width": 4096,
         "rate": 0.3, "residual": True},
        # 64 decoding tokens that choose 6 of 64 experts each: the weights' bytes count
        {"name": "grouped_step", "op": "grouped", "train": False, "dtype": "bf16", "wdtype": "bf16", "rows": 384,
         "groups": 64, "inputs": 2048, "outputs": 1408},
        # a small float32 layer with odd sizes, trained
        {"name": "grouped_odd_f32", "op": "grouped", "train": True, "dtype": "f32", "wdtype": "f32", "rows": 1021,
         "groups": 8, "inputs": 257, "outputs": 515},
        # prefill of 16384 tokens, 6 of 64 experts each, one expert layer
        {"name": "grouped_prefill", "op": "grouped", "train": False, "dtype": "bf16", "wdtype": "bf16", "rows": 98304,
         "groups": 64, "inputs": 2048, "outputs": 1408},
        # a training step of a layer of 16 experts, weight gradients kept in float32
        {"name": "grouped_train", "op": "grouped", "train": True, "dtype": "bf16", "wdtype": "f32", "rows": 8192,
         "groups": 16, "inputs": 1024, "outputs": 2048},
        # a training step of the 64-expert layer on a large batch
        {"name": "grouped_train_large", "op": "grouped", "train": True, "dtype": "bf16", "wdtype": "f32",
         "rows": 98304, "groups": 64, "inputs": 1408, "outputs": 2048},
    ]


def _log_int(rng, low, high, multiple=1):
    """A whole number between low and high, spread over its logarithm, a multiple of `multiple`."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(v / multiple)) * multiple))


def draw(rng):
    op = rng.choice(["layer_norm", "dropout", "grouped", "grouped"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op in ("layer_norm", "dropout"):
        width = _log_int(rng, 64, 8192, rng.choice([1, 8, 64]))
        rows = _log_int(rng, 1, min(65536, 134217728 // width))
        case = {"op": op, "train": rng.random() < 0.7, "dtype": dtype, "rows": rows, "width": width,
                "residual": rng.random() < 0.6}
        if op == "layer_norm":
            case["wdtype"] = rng.choice([dtype, "f32"])
        else:
            case["rate"] = round(rng.uniform(0.02, 0.6), 3)
        return case
    groups = _log_int(rng, 1, 128)
    # tensor-core sizes in bf16, and now and then odd ones; float32 and odd sizes on smaller batches
    odd = rng.random() < 0.2
    small = odd or dtype == "f32"
    high = 1100 if small else 2304
    inputs = _log_int(rng, 64, high, 1 if odd else 8)
    outputs = _log_int(rng, 64, high, 1 if odd else 8)
    rows = _log_int(rng, 1, 16384 if small else 65536)
    return {"op": op, "train": rng.random() < 0.6, "dtype": dtype,
            "wdtype": "f32" if dtype == "f32" else rng.choice(["bf16", "f32"]), "rows": rows, "groups": groups,
            "inputs": inputs, "outputs": outputs}


def _counts(rows, groups, seed):
    """Rows of each group, unevenly popular, in sum `rows`; a group may have none."""
    rng = np.random.default_rng(seed * 7919 + rows * 31 + groups)
    p = np.exp(0.4 * rng.standard_normal(groups))
    return rng.multinomial(rows, p / p.sum()).astype(np.int64)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=dev) * scale + shift).to(dtype)

    s = {"case": case}
    if case["op"] == "layer_norm":
        n, d, wdt = case["rows"], case["width"], DTYPES[case["wdtype"]]
        s["x"] = normal(n, d, scale=1.5, shift=0.2)
        s["weight"] = normal(d, scale=0.1, shift=1.0, dtype=wdt)
        s["bias"] = normal(d, scale=0.1, dtype=wdt)
        s["epsilon"] = 1e-6
        if case["train"]:
            s["dy"] = normal(n, d)
            s["dres"] = normal(n, d) if case["residual"] else None
    elif case["op"] == "dropout":
        n, d = case["rows"], case["width"]
        s["x"] = normal(n, d)
        s["residual"] = normal(n, d) if case["residual"] else None
        s["seed"], s["stream"] = 1234567 + seed, 5
        if case["train"]:
            s["dout"] = normal(n, d)
    else:
        n, e, k, m = case["rows"], case["groups"], case["inputs"], case["outputs"]
        counts = _counts(n, e, seed)
        s["largest"] = int(counts.max())
        s["counts"] = torch.from_numpy(counts).to(dev)
        s["x"] = normal(n, k)
        s["weights"] = normal(e, m, k, scale=k**-0.5)
        if case["train"]:
            s["dy"] = normal(n, m)
    return s


# ---- the plain forms


def _plain_layer_norm(s):
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + s["epsilon"])
    xh = c * rstd
    out = {"y": (xh * w + b).to(s["x"].dtype)}
    if s["case"]["train"]:
        dy = s["dy"].float()
        gy = dy * w
        dx = rstd * (gy - gy.mean(1, keepdim=True) - xh * (gy * xh).mean(1, keepdim=True))
        if s["dres"] is not None:
            dx = dx + s["dres"].float()
        out["dx"] = dx.to(s["x"].dtype)
        out["dweight"] = (dy * xh).sum(0).to(s["weight"].dtype)
        out["dbias"] = dy.sum(0).to(s["bias"].dtype)
    return out


def _shift_right(z, n):
    """The logical right shift of 64-bit words held in int64."""
    return (z >> n) & ((1 << (64 - n)) - 1)


def _signed(v):
    return v - (1 << 64) if v >= 1 << 63 else v


def _mix(z):
    """SplitMix64 of 64-bit words held in int64."""
    z = z + _signed(0x9E3779B97F4A7C15)
    z = (z ^ _shift_right(z, 30)) * _signed(0xBF58476D1CE4E5B9)
    z = (z ^ _shift_right(z, 27)) * _signed(0x94D049BB133111EB)
    return z ^ _shift_right(z, 31)


def _plain_keep(n, rate, seed, stream, device):
    """Whether element i of n is kept: half i % 2 (the low one first) of word i // 2 is at least rate * 2^32."""
    start = (seed ^ (stream * 0xD1B54A32D192ED03)) & ((1 << 64) - 1)
    key = _mix(torch.full((1,), _signed(start), dtype=torch.int64, device=device))
    words = _mix(key + torch.arange((n + 1) // 2, dtype=torch.int64, device=device))
    halves = torch.stack((words & 0xFFFFFFFF, _shift_right(words, 32)), 1).reshape(-1)[:n]
    return halves >= int(rate * 2.0**32)


def _plain_dropout(s):
    x, rate = s["x"], s["case"]["rate"]
    keep = _plain_keep(x.numel(), rate, s["seed"], s["stream"], x.device).reshape(x.shape)
    y = torch.where(keep, x.float() * (1.0 / (1.0 - rate)), 0.0)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(x.dtype)}
    if s["case"]["train"]:
        out["dx"] = torch.where(keep, s["dout"].float() * (1.0 / (1.0 - rate)), 0.0).to(x.dtype)
    return out


def _plain_grouped(s):
    x, w, counts = s["x"], s["weights"].float(), s["counts"]
    ends = counts.cumsum(0)
    row = torch.arange(x.shape[0], device=x.device)
    group = torch.searchsorted(ends, row, right=True)
    place = row - (ends - counts)[group]

    def padded(a):
        p = torch.zeros(w.shape[0], s["largest"], a.shape[1], device=a.device)
        p[group, place] = a.float()
        return p

    xp = padded(x)
    out = {"y": torch.bmm(xp, w.transpose(1, 2))[group, place].to(x.dtype)}
    if s["case"]["train"]:
        dyp = padded(s["dy"])
        out["dx"] = torch.bmm(dyp, w)[group, place].to(x.dtype)
        out["dw"] = torch.bmm(dyp.transpose(1, 2), xp).to(DTYPES[s["case"]["wdtype"]])
    return out


# ---- the package's calls


def _own_layer_norm(s):
    from gotransformers_b200 import moe

    y, mean, rstd = moe.layer_norm(s["x"], s["weight"], s["bias"], s["epsilon"])
    out = {"y": y}
    if s["case"]["train"]:
        out["dx"], out["dweight"], out["dbias"] = moe.layer_norm_backward(
            s["dy"], s["x"], mean, rstd, s["weight"], residual_gradients=s["dres"])
    return out


def _own_dropout(s):
    from gotransformers_b200 import moe

    rate, seed, stream = s["case"]["rate"], s["seed"], s["stream"]
    out = {"y": moe.dropout(s["x"], rate, seed, stream, residual=s["residual"])}
    if s["case"]["train"]:
        out["dx"] = moe.dropout_backward(s["dout"], rate, seed, stream)
    return out


def _own_grouped(s):
    from gotransformers_b200 import moe

    out = {"y": moe.grouped_product(s["x"], s["weights"], s["counts"])}
    if s["case"]["train"]:
        out["dx"] = moe.grouped_product_input_gradients(s["dy"], s["weights"], s["counts"])
        out["dw"] = moe.grouped_product_weight_gradients(s["dy"], s["x"], s["counts"],
                                                         dtype=DTYPES[s["case"]["wdtype"]])
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"layer_norm": _own_layer_norm, "dropout": _own_dropout, "grouped": _own_grouped}[op](state)
    return {"layer_norm": _plain_layer_norm, "dropout": _plain_dropout, "grouped": _plain_grouped}[op](state)


def work(case):
    """Each input read once and each output written once, forward and backward together."""
    size = {"bf16": 2, "f32": 4}
    es, n = size[case["dtype"]], case["rows"]
    if case["op"] == "layer_norm":
        ws, d = size[case["wdtype"]], case["width"]
        values, params, flops = 2 * n * d, 2 * d, 8 * n * d
        if case["train"]:
            values += (2 + int(case["residual"])) * n * d
            params += 2 * d
            flops += 14 * n * d
        return {"bytes": values * es + params * ws, "flops": flops}
    if case["op"] == "dropout":
        d = case["width"]
        values, flops = (2 + int(case["residual"])) * n * d, 2 * n * d
        if case["train"]:
            values += 2 * n * d
            flops += n * d
        return {"bytes": values * es, "flops": flops}
    e, k, m = case["groups"], case["inputs"], case["outputs"]
    product = 2 * n * k * m
    moved = es * (n * k + min(e, n) * m * k + n * m)
    if not case["train"]:
        return {"bytes": moved, "flops": product}
    return {"bytes": moved + es * (n * m + n * k) + size[case["wdtype"]] * e * m * k, "flops": 3 * product}


# ---- from the definitions, in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "layer_norm":
        return _exact_layer_norm(case, s)
    if case["op"] == "dropout":
        return _exact_dropout(case, s)
    return _exact_grouped(case, s)


def _exact_layer_norm(case, s):
    n, d = case["rows"], case["width"]
    w, b = s["weight"].double(), s["bias"].double()
    y = torch.empty(n, d, dtype=torch.float64, device=w.device)
    dx = torch.empty_like(y) if case["train"] else None
    dw, db = torch.zeros_like(w), torch.zeros_like(b)
    step = max(1, (1 << 25) // d)
    for r in range(0, n, step):
        x = s["x"][r:r + step].double()
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        inv = (var + s["epsilon"]).rsqrt()
        xh = (x - mean) * inv
        y[r:r + step] = torch.addcmul(b, xh, w)
        if case["train"]:
            dy = s["dy"][r:r + step].double()
            gy = dy * w
            t = (d * gy - gy.sum(1, keepdim=True) - xh * (gy * xh).sum(1, keepdim=True)) * (inv / d)
            dx[r:r + step] = t if s["dres"] is None else t + s["dres"][r:r + step].double()
            dw += torch.einsum("rd,rd->d", dy, xh)
            db += torch.einsum("rd->d", dy)
    return {"y": y, "dx": dx, "dweight": dw, "dbias": db} if case["train"] else {"y": y}


def _exact_dropout(case, s):
    n = case["rows"] * case["width"]
    with np.errstate(over="ignore"):
        def split_mix(z):
            z = z + np.uint64(0x9E3779B97F4A7C15)
            z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
            z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
            return z ^ (z >> np.uint64(31))

        one = np.array([s["seed"] ^ ((s["stream"] * 0xD1B54A32D192ED03) & 0xFFFFFFFFFFFFFFFF)], dtype=np.uint64)
        key = split_mix(one)[0]
        kept = np.empty(n + n % 2, dtype=bool)
        step = 1 << 22
        for j in range(0, kept.size // 2, step):
            words = split_mix(key + np.arange(j, min(kept.size // 2, j + step), dtype=np.uint64))
            kept[2 * j:2 * j + 2 * words.size] = words.view(np.uint32) >= np.uint32(math.floor(case["rate"] * 2**32))
    keep = torch.from_numpy(kept[:n].reshape(case["rows"], case["width"])).to(s["x"].device).double()
    y = s["x"].double() * keep / (1.0 - case["rate"])
    if s["residual"] is not None:
        y += s["residual"].double()
    if not case["train"]:
        return {"y": y}
    return {"y": y, "dx": s["dout"].double() * keep / (1.0 - case["rate"])}


def _exact_grouped(case, s):
    x, w = s["x"], s["weights"]
    y = torch.zeros(case["rows"], case["outputs"], dtype=torch.float64, device=x.device)
    dx = torch.zeros(case["rows"], case["inputs"], dtype=torch.float64, device=x.device) if case["train"] else None
    dw = torch.zeros(w.shape, dtype=torch.float64, device=x.device) if case["train"] else None
    r = 0
    for e, m in enumerate(s["counts"].tolist()):
        a, we = x[r:r + m].double(), w[e].double()
        y[r:r + m] = a @ we.T
        if case["train"]:
            d = s["dy"][r:r + m].double()
            dx[r:r + m] = d @ we
            dw[e] = d.T @ a
        r += int(m)
    return {"y": y, "dx": dx, "dw": dw} if case["train"] else {"y": y}
