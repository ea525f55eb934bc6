"""The operators beside autograd: a tensor that a call writes into counts as
changed, so that a backward pass that saved it before refuses to run on the
new values."""
import pytest
import torch

from gotransformers_b200 import moe

pytestmark = pytest.mark.gpu
F32 = torch.float32


def calls():
    x = torch.randn(6, 8, device="cuda")
    w3 = torch.randn(2, 8, 8, device="cuda")
    w, counts = torch.ones(8, device="cuda"), torch.tensor([2, 4], device="cuda")
    y, mean, rstd = moe.layer_norm(x, w, w)
    return {
        "layer_norm": (6, 8, lambda t: moe.layer_norm(x, w, w, out=t)),
        "layer_norm in place": (6, 8, lambda t: moe.layer_norm(t, w, w, out=t)),
        "layer_norm_backward": (6, 8, lambda t: moe.layer_norm_backward(y, x, mean, rstd, w, input_gradients=t)),
        "its weight gradients": (8, None, lambda t: moe.layer_norm_backward(y, x, mean, rstd, w, weight_grad=t,
                                                                            bias_grad=w.clone())),
        "its bias gradients": (8, None, lambda t: moe.layer_norm_backward(y, x, mean, rstd, w, weight_grad=w.clone(),
                                                                          bias_grad=t)),
        "dropout": (6, 8, lambda t: moe.dropout(x, 0.5, 1, out=t)),
        "dropout into the residual": (6, 8, lambda t: moe.dropout(x, 0.5, 1, residual=t, out=t)),
        "dropout_backward": (6, 8, lambda t: moe.dropout_backward(x, 0.5, 1, input_gradients=t)),
        "grouped_product": (6, 8, lambda t: moe.grouped_product(x, w3, counts, out=t)),
        "its input gradients": (6, 8, lambda t: moe.grouped_product_input_gradients(x, w3, counts, input_gradients=t)),
        "its weight gradients, added to": (2, 64, lambda t: moe.grouped_product_weight_gradients(
            x, x, counts, weight_grad=t.view(2, 8, 8))),
    }


@pytest.mark.parametrize("name", list(range(11)))
def test_written_tensors_count_as_changed(name):
    rows, columns, call = list(calls().values())[name]
    shape = (rows,) if columns is None else (rows, columns)
    t = torch.rand(shape, device="cuda")
    leaf = torch.ones(shape, device="cuda", requires_grad=True)
    loss = (leaf * t).sum()  # saves t
    before = t._version
    call(t)
    assert t._version == before + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_read_tensors_do_not():
    x = torch.randn(6, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    y, mean, rstd = moe.layer_norm(x, w, w)
    moe.layer_norm_backward(y, x, mean, rstd, w)
    moe.dropout(x, 0.5, 1, residual=y)
    assert x._version == w._version == y._version == mean._version == 0


def test_inference_tensors_are_written():
    with torch.inference_mode():
        x = torch.randn(6, 8, device="cuda")
        out = torch.empty_like(x)
        assert torch.equal(moe.dropout(x, 0.5, 1, out=out), moe.dropout(x, 0.5, 1))
