"""What stands between a model's products, without a GPU: the tests' formulas
against differences, and calls that are refused before anything is read."""

import math

import numpy as np
import pytest

from _attention import fake, mod
from _layers import Join, Probs, kept


def difference(loss, arr, at, h=1e-6):
    keep = arr[at]
    arr[at] = keep + h
    up = loss()
    arr[at] = keep - h
    down = loss()
    arr[at] = keep
    return (up - down) / (2 * h)


SHAPE = (2, 3, 6)


def check_join(operands, eps1, eps2, dz, dh, **rest):
    """Every gradient at three places against the loss's differences."""
    def loss():
        j = Join(eps1=eps1, eps2=eps2, **operands, **rest)
        return float((j.z * dz).sum() + ((j.h * dh).sum() if eps2 else 0.0))

    j = Join(eps1=eps1, eps2=eps2, **operands, **rest)
    grads, _ = j.backward(dz, dh if eps2 else None, j.r1, j.r2 if eps2 else None)
    names = {"dx": "x", "dy": "y", "dgate": "gate", "dw1": "w1", "dw2": "w2"}
    assert set(grads) == {d for d, n in names.items() if operands.get(n) is not None}
    for d, grad in grads.items():
        arr = operands[names[d]]
        assert grad.shape == arr.shape
        for flat in (0, arr.size // 2, arr.size - 1):
            at = np.unravel_index(flat, arr.shape)
            # a central difference is off by O(h^2) and by the losses' rounding over 2 h
            assert abs(difference(loss, arr, at) - grad[at]) < 1e-6 * max(1.0, abs(grad[at])), d


@pytest.mark.parametrize("eps1,eps2", [(1e-3, 1e-3), (None, 1e-3), (1e-3, None)])
@pytest.mark.parametrize("gate", [None, (6,), (2, 1, 6), (2, 3, 1), (2, 3, 6), (1,)], ids=str)
def test_join_gradients_against_differences(gate, eps1, eps2):
    rng = np.random.default_rng(1)
    x, y, dz, dh = (rng.standard_normal(SHAPE) for _ in range(4))
    w1, w2 = rng.standard_normal(6), rng.standard_normal(6)
    operands = {"x": x, "y": y, "gate": None if gate is None else rng.standard_normal(gate), "w1": w1 if eps1 else None,
                "w2": w2 if eps2 else None}
    check_join(operands, eps1, eps2, dz, dh, a=0.9, b=0.4, keep=kept(0.3, 5, SHAPE), p=0.3)


def test_norm_gradients_against_differences():
    rng = np.random.default_rng(3)
    x, dz, dh = (rng.standard_normal(SHAPE) for _ in range(3))
    check_join({"x": x, "w2": rng.standard_normal(6)}, None, 1e-3, dz, dh)


@pytest.mark.parametrize("scale", [1.0, 0.6, 2.5])
def test_log_prob_gradient_against_differences(scale):
    rng = np.random.default_rng(2)
    x, t = rng.standard_normal((4, 9)) * 2, np.array([3, 0, -100, 8])
    a, b = rng.standard_normal(4), rng.standard_normal(4)

    def loss():
        p = Probs(x, t, scale)
        return float((p.given()[0] * a).sum() + (p.h * b).sum())

    dx, _ = Probs(x, t, scale).backward(a, b)
    for at in [(0, 3), (0, 0), (1, 8), (2, 2), (3, 8), (3, 1)]:
        assert abs(difference(loss, x, at) - dx[at]) < 1e-7


def test_top_of_equal_and_undefined_logits():
    x = np.array([[1.0, 3.0, 3.0, 0.0, 3.0], [np.nan, 2.0, np.inf, np.nan, 1.0], [-np.inf] * 5])
    assert Probs(x).top(4)[0].tolist() == [[1, 2, 4, 0], [0, 3, 2, 1], [0, 1, 2, 3]]


# ---- refusals --------------------------------------------------------------------

BF = "bfloat16"


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("x,p,seed,error,message", [
    (fake((4, 8), "int32"), 0.5, 1, "DeclinedError", "float"),
    (fake((4, 8), device=-1), 0.5, 1, "DeclinedError", "device"),
    (fake((4, 8)), -0.1, 1, "DeviceError", "between"),
    (fake((4, 8)), 1.5, 1, "DeviceError", "between"),
    (fake((4, 8)), math.nan, 1, "DeviceError", "between"),
    (fake((4, 8)), 0.5, fake((1,), "int32"), "DeclinedError", "seed"),
    (fake((4, 8)), 0.5, fake((1,), "int64", device=1), "DeclinedError", "seed"),
    (fake((4, 8)), 0.5, fake((2,), "int64"), "DeviceError", "one number"),
    (None, 0.5, 1, "DeviceError", "null"),
], ids=["integers", "host", "negative", "above_one", "nan", "seed_type", "seed_device", "two_seeds", "null"])
def test_dropout_refused(ops, backward, x, p, seed, error, message):
    call = ops.seeded_dropout_backward if backward else ops.seeded_dropout
    with pytest.raises(getattr(mod("tensor"), error), match=message):
        call(x, p, seed)


def join_args(**change):
    a = {"residual": fake((2, 5, 16)), "branch": fake((2, 5, 16)), "branch_eps": 1e-6}
    a.update(change)
    return a


@pytest.mark.parametrize("change,error,message", [
    ({"residual": fake((2, 5, 16), "int64")}, "DeclinedError", "float"),
    ({"residual": fake((2, 5, 16), device=-1)}, "DeclinedError", "device"),
    ({"residual": fake((), BF)}, "DeclinedError", "rows"),
    ({"residual": fake((2, 5, 0)), "branch": fake((2, 5, 0))}, "DeviceError", "no elements"),
    ({"residual": fake((5, 16385)), "branch": fake((5, 16385))}, "DeclinedError", "wider"),
    ({"residual": None}, "DeviceError", "null"),
    ({"branch": fake((2, 5, 16), "float32")}, "DeclinedError", "branch"),
    ({"branch": fake((2, 5, 16), device=1)}, "DeclinedError", "branch"),
    ({"branch": fake((2, 4, 16))}, "DeviceError", "shape"),
    ({"branch": fake((5, 16))}, "DeviceError", "shape"),
    ({"weight": fake((8,))}, "DeviceError", "weight"),
    ({"weight": fake((1, 16))}, "DeviceError", "weight"),
    ({"branch_weight": fake((16,), "float16")}, "DeclinedError", "weight"),
    ({"branch_weight": fake((16,)), "branch_eps": None}, "DeviceError", "weight"),
    ({"weight": fake((16,)), "eps": None}, "DeviceError", "weight"),
    ({"gate": fake((16,), "float32")}, "DeclinedError", "gate"),
    ({"gate": fake((8,))}, "DeviceError", "expand"),
    ({"gate": fake((5, 1, 16))}, "DeviceError", "expand"),
    ({"gate": fake((2, 2, 5, 16))}, "DeviceError", "axes"),
    ({"gate": fake((5, 16))}, "DeclinedError", "repeats"),
    ({"gate": fake((1, 5, 1))}, "DeclinedError", "repeats"),
    ({"branch": None, "branch_eps": None, "gate": fake((16,))}, "DeviceError", "without a branch"),
    ({"branch": None}, "DeviceError", "without a branch"),
    ({"branch": None, "branch_eps": None, "residual_scale": 2.0}, "DeviceError", "without a branch"),
    ({"branch": None, "branch_eps": None, "p": 0.5}, "DeviceError", "without a branch"),
    ({"branch": None, "branch_eps": None, "eps": None}, "DeviceError", "neither"),
    ({"residual_scale": math.inf}, "DeviceError", "finite"),
    ({"branch_scale": math.nan}, "DeviceError", "finite"),
    ({"branch_scale": 1e39}, "DeviceError", "finite"),
    ({"eps": math.nan}, "DeviceError", "eps"),
    ({"branch_eps": math.nan}, "DeviceError", "eps"),
    ({"p": 2.0}, "DeviceError", "between"),
    ({"p": 0.5, "seed": fake((1,), "float32")}, "DeclinedError", "seed"),
])
def test_join_refused(ops, change, error, message):
    with pytest.raises(getattr(mod("tensor"), error), match=message):
        ops.residual_norm(**join_args(**change))


def test_join_negative_eps(ops):
    with pytest.raises(ValueError):
        ops.residual_norm(fake((4, 8)), eps=-1e-6)


@pytest.mark.parametrize("change,error,message", [
    ({"grad_sum": None, "grad_normed": None}, "DeviceError", "no gradient"),
    ({"grad_sum": fake((2, 5, 16), "float32")}, "DeclinedError", "gradients"),
    ({"grad_normed": fake((2, 5, 8))}, "DeviceError", "shape"),
    ({"rstd": None}, "DeviceError", "statistics"),
    ({"rstd": fake((2, 5), "float16")}, "DeclinedError", "statistics"),
    ({"rstd": fake((2, 5, 1), "float32")}, "DeviceError", "statistics"),
    ({"branch_rstd": fake((10,), "float32")}, "DeviceError", "statistics"),
    ({"branch_weight": fake((16,)), "branch_rstd": None}, "DeviceError", "weight"),
    ({"branch": None}, "DeviceError", "without a branch"),
    ({"residual": None}, "DeviceError", "null"),
])
def test_join_backward_refused(ops, change, error, message):
    a = {"grad_sum": fake((2, 5, 16)), "grad_normed": fake((2, 5, 16)), "residual": fake((2, 5, 16)), "branch": fake((2, 5, 16)),
         "branch_rstd": fake((2, 5), "float32"), "rstd": fake((2, 5), "float32")}
    a.update(change)
    with pytest.raises(getattr(mod("tensor"), error), match=message):
        ops.residual_norm_backward(**a)


@pytest.mark.parametrize("change,error,message", [
    ({"logits": fake((4, 9), "int32")}, "DeclinedError", "float"),
    ({"logits": fake((4, 9), device=-1)}, "DeclinedError", "device"),
    ({"logits": fake((), BF), "targets": None}, "DeclinedError", "rows"),
    ({"logits": fake((4, 0))}, "DeviceError", "no logits"),
    ({"logits": None}, "DeviceError", "null"),
    ({"targets": fake((4,), "float32")}, "DeclinedError", "targets"),
    ({"targets": fake((4,), "int64", device=1)}, "DeclinedError", "targets"),
    ({"targets": fake((5,), "int64")}, "DeviceError", "targets"),
    ({"targets": fake((4, 1), "int64")}, "DeviceError", "targets"),
    ({"scale": 0.0}, "DeviceError", "scale"),
    ({"scale": -1.0}, "DeviceError", "scale"),
    ({"scale": math.nan}, "DeviceError", "scale"),
    ({"scale": 1e39}, "DeviceError", "scale"),
    ({"top": -1}, "DeviceError", "negative"),
    ({"top": 10}, "DeviceError", "alternatives"),
    ({"logits": fake((4, 99)), "top": 65}, "DeclinedError", "alternatives"),
])
def test_log_probs_refused(ops, change, error, message):
    a = {"logits": fake((4, 9)), "targets": fake((4,), "int64")}
    a.update(change)
    with pytest.raises(getattr(mod("tensor"), error), match=message):
        ops.token_log_probs(**a)


@pytest.mark.parametrize("change,error,message", [
    ({"grad_logprob": None}, "DeviceError", "no gradient"),
    ({"targets": None}, "DeviceError", "without their tokens"),
    ({"grad_entropy": fake((4,), "float32")}, "DeviceError", "without the entropy"),
    ({"grad_logprob": fake((4,))}, "DeclinedError", "float32"),
    ({"grad_logprob": fake((4, 9), "float32")}, "DeviceError", "shape"),
    ({"stats": fake((4,), "float32")}, "DeviceError", "shape"),
    ({"stats": None}, "DeviceError", "null"),
    ({"scale": 0.0}, "DeviceError", "scale"),
])
def test_log_probs_backward_refused(ops, change, error, message):
    a = {"grad_logprob": fake((4,), "float32"), "grad_entropy": None, "logits": fake((4, 9)), "targets": fake((4,), "int64"),
         "stats": fake((4, 2), "float32")}
    a.update(change)
    with pytest.raises(getattr(mod("tensor"), error), match=message):
        ops.token_log_probs_backward(**a)


@pytest.mark.parametrize("shape", [(1 << 30, 4), (1 << 15, 1 << 15, 4)], ids=str)
def test_more_rows_than_are_counted(ops, shape):
    x, row, strides = fake(shape), fake(shape[:-1], "float32"), (0,) * len(shape)
    for call in (lambda: ops.residual_norm(x), lambda: ops.residual_norm(fake(shape, strides=strides), x),
                 lambda: ops.residual_norm_backward(x, x, x, rstd=row), lambda: ops.token_log_probs(x, fake(shape[:-1], "int64")),
                 lambda: ops.token_log_probs_backward(row, None, x, fake(shape[:-1], "int64"), fake(shape[:-1] + (2,), "float32"))):
        with pytest.raises(mod("tensor").DeviceError, match=f"{1 << 30} rows"):
            call()


def test_more_logits_than_are_counted(ops):
    with pytest.raises(mod("tensor").DeviceError, match="logits"):
        ops.token_log_probs(fake((1, 1 << 31)))


@pytest.mark.parametrize("call", ["dropout", "join", "probs"])
def test_more_axes_than_a_tensor_has(ops, call):
    """Refused before an axis past the last one is looked at."""
    x = fake((2, 5, 16))
    x._ref.ndim = 10 ** 9
    with pytest.raises(mod("tensor").DeviceError, match="dimensions"):
        {"dropout": lambda: ops.seeded_dropout(x, 0.5, 1), "join": lambda: ops.residual_norm(x),
         "probs": lambda: ops.token_log_probs(x)}[call]()
