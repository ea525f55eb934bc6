"""Every pair of arguments that may not share memory, for each handle-less
operator, without a GPU: the addresses are never read."""
import pytest

import test_operators_cpu as T
from gotransformers_b200 import _lib

EINVAL = -1
BYTES = 16  # less than any argument below has

# the arguments that a call only reads, those that it writes, and the pairs
# that may be one and the same
CALLS = {
    "norm_forward": (T.norm_forward, ["x", "weight", "bias"], ["y", "mean", "rstd"], {("x", "y")}),
    "norm_backward": (T.norm_backward, ["dy", "x", "w", "m", "r", "res"], ["dx", "dw", "db", "work"],
                      {("dy", "dx"), ("x", "dx"), ("res", "dx")}),
    "drop": (T.drop, ["x", "res"], ["out"], {("x", "out"), ("res", "out")}),
    "product": (T.product, ["x", "w", "counts"], ["y"], set()),
    "weight_grad": (T.weight_grad, ["dy", "x", "counts"], ["dw"], set()),
}


def address_of(call, name):
    """Where test_operators_cpu's call puts an argument."""
    order = {
        "norm_forward": ["x", "weight", "bias", "y", "mean", "rstd"],
        "norm_backward": ["dy", "x", "w", "m", "r", "res", "dx", "dw", "db", "work"],
        "drop": ["x", "res", "out"],
        "product": ["x", "w", "counts", "y"],
        "weight_grad": ["dy", "x", "counts", "dw"],
    }[call]
    return T.A + order.index(name) * T.STEP


def pairs():
    for call, (_, reads, writes, may) in CALLS.items():
        for w in writes:
            for other in reads + [o for o in writes if o < w]:
                yield pytest.param(call, other, w, (other, w) in may, id=f"{call}-{other}-{w}")


@pytest.mark.parametrize("call,other,written,may_be_it", list(pairs()))
def test_written_arguments_overlap_no_other(call, other, written, may_be_it):
    f, at = CALLS[call][0], address_of(call, other)
    rc = f(**{written: at})
    message = _lib.lib().gtmoe_last_error()
    if may_be_it:
        # the same place is allowed: the call ends at the device check
        assert rc == -2 or b"device memory" in message
        assert f(**{written: at + BYTES}) == EINVAL and b"overlaps" in _lib.lib().gtmoe_last_error()
    else:
        assert rc == EINVAL and b"overlaps" in message
