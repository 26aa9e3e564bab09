"""The norm and rotation of heads without a GPU: the tests' formulas against
differences, and calls that are refused before anything is read."""

import numpy as np
import pytest

from _attention import fake, head_norm, head_norm_backward, mod, table_of


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(8, 8), (7, 4), (6, 0)])
def test_gradient_formula_against_differences(dim, rotary, interleaved):
    rng = np.random.default_rng(1)
    x, dy = rng.standard_normal((3, 2, dim)), rng.standard_normal((3, 2, dim))
    w = rng.standard_normal(dim)
    table, pos, eps = table_of(50, rotary), np.array([0, 7, 49]), 1e-3

    def loss(x, w):
        return float((head_norm(x, w, table, pos, eps, interleaved)[0] * dy).sum())

    r = head_norm(x, w, table, pos, eps, interleaved)[1]
    dx, dw, _, _ = head_norm_backward(dy, x, r, w, table, pos, interleaved)
    h = 1e-6
    for arr, grad, at in [(x, dx, (1, 1, 3)), (x, dx, (0, 0, dim - 1)), (x, dx, (2, 0, 0)), (w, dw, (2,)), (w, dw, (dim - 1,))]:
        keep = arr[at]
        arr[at] = keep + h
        up = loss(x, w)
        arr[at] = keep - h
        down = loss(x, w)
        arr[at] = keep
        # a central difference is off by O(h^2) and by the losses' rounding over 2 h
        assert abs((up - down) / (2 * h) - grad[at]) < 1e-7 * max(1.0, abs(grad[at]))


def call(ops, **change):
    a = {"query": fake((2, 5, 4, 16)), "key": fake((2, 5, 2, 16)), "table": fake((9, 16), "float32"),
         "positions": fake((5,), "int64"), "query_weight": None, "key_weight": None}
    a.update(change)
    return ops.qk_norm_rope(*a.values())


@pytest.mark.parametrize("change", [
    {"query": fake((2, 5, 4, 16), "int32")},
    {"query": fake((2, 5, 4, 16), "float16")},                       # another dtype than the keys
    {"key": fake((2, 5, 2, 16), device=-1)},                         # host memory
    {"key": fake((2, 5, 2, 16), device=1)},                          # another device
    {"query": fake((16,)), "key": fake((16,))},
    {"table": fake((9, 16), "float16")},
    {"positions": fake((5,), "float32")},
    {"query_weight": fake((16,), "float32")},
    {"query": fake((5, 2, 1026)), "key": fake((5, 1, 1026))},
], ids=["integers", "mixed", "host", "device", "no_heads", "table_type", "position_type", "weight_type", "wide"])
def test_declined(ops, change):
    with pytest.raises(mod("tensor").DeclinedError):
        call(ops, **change)


@pytest.mark.parametrize("change,message", [
    ({"key": fake((2, 4, 2, 16))}, "tokens"),
    ({"key": fake((2, 5, 2, 8))}, "head size"),
    ({"table": fake((9, 15), "float32")}, "rotates"),
    ({"table": fake((9, 18), "float32")}, "rotates"),
    ({"positions": fake((4,), "int64")}, "expand"),
    ({"positions": fake((2, 2, 5), "int64")}, "expand"),
    ({"query_weight": fake((8,))}, "weight"),
    ({"key_weight": fake((2, 16))}, "weight"),
])
def test_refused(ops, change, message):
    with pytest.raises(mod("tensor").DeviceError, match=message):
        call(ops, **change)


@pytest.mark.parametrize("change,error", [
    ({0: fake((2, 5, 4, 8))}, "DeviceError"),
    ({1: fake((2, 5, 2, 16), "float32")}, "DeclinedError"),
    ({6: fake((2, 5, 2), "float32")}, "DeviceError"),
    ({7: fake((2, 5, 2), "float16")}, "DeclinedError"),
], ids=["gradient_shape", "gradient_type", "statistics_shape", "statistics_type"])
def test_backward_refused(ops, change, error):
    a = [fake((2, 5, 4, 16)), fake((2, 5, 2, 16)), fake((2, 5, 4, 16)), fake((2, 5, 2, 16)), fake((9, 16), "float32"),
         fake((5,), "int64"), fake((2, 5, 4), "float32"), fake((2, 5, 2), "float32")]
    for i, t in change.items():
        a[i] = t
    with pytest.raises(getattr(mod("tensor"), error)):
        ops.qk_norm_rope_backward(*a, output_mask=(False,) * 4)


def test_null_operand(ops):
    with pytest.raises(mod("tensor").DeviceError, match="null"):
        call(ops, table=None)


def test_more_axes_than_a_tensor_has(ops):
    """Refused before an axis past the last one is looked at."""
    query = fake((2, 5, 4, 16))
    query._ref.ndim = 10 ** 9
    with pytest.raises(mod("tensor").DeviceError, match="dimensions"):
        call(ops, query=query)
