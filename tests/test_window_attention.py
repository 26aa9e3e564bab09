"""Attention with a sliding window and first tokens without a GPU: the tests'
formulas against differences and against a row at a time, and calls that are
refused before anything is read."""

import numpy as np
import pytest

from _attention import F32, Attention, fake, mod, seen


def operands(b, tq, tk, h, hk, d, seed=0):
    rng = np.random.default_rng(seed)
    return [rng.standard_normal(s) for s in ((b, tq, h, d), (b, tk, hk, d), (b, tk, hk, d))]


def test_definition_a_row_at_a_time():
    q, k, v = operands(2, 5, 9, 4, 2, 3)
    lengths, starts, window, sinks = [9, 6], [4, -1], 2, 1
    a = Attention(F32, q, k, v, window, sinks, 0.7, lengths, starts)
    for b in range(2):
        for i in range(5):
            p = starts[b] + i
            js = [j for j in range(lengths[b]) if 0 <= p < lengths[b] and j <= p and (j > p - window or j < sinks)]
            for h in range(4):
                if not js:
                    assert a.lse[b, h, i] == -np.inf and (a.out[b, h, i] == 0).all()
                    continue
                e = np.exp(np.array([0.7 * (q[b, i, h] @ k[b, j, h // 2]) for j in js]))
                assert np.allclose(a.lse[b, h, i], np.log(e.sum()), rtol=1e-13)
                assert np.allclose(a.out[b, h, i], sum(x * v[b, j, h // 2] for x, j in zip(e, js)) / e.sum(), rtol=1e-12)


def test_gradient_formula_against_differences():
    q, k, v = operands(2, 4, 6, 4, 2, 3, 1)
    do = np.random.default_rng(2).standard_normal(q.shape)
    rule = dict(window=3, sinks=1, lengths=[6, 4], starts=[2, 1])

    def loss():
        return float((Attention.tokens(Attention(F32, q, k, v, **rule).out) * do).sum())

    grads, _ = Attention(F32, q, k, v, **rule).backward(do, F32)
    h = 1e-6
    rng = np.random.default_rng(3)
    for arr, grad in zip((q, k, v), grads):
        for _ in range(12):
            at = tuple(rng.integers(0, n) for n in arr.shape)
            keep = arr[at]
            arr[at] = keep + h
            up = loss()
            arr[at] = keep - h
            down = loss()
            arr[at] = keep
            assert abs((up - down) / (2 * h) - grad[at]) < 1e-7 * max(1.0, abs(grad[at]))


def test_what_is_seen():
    s = seen(4, 6, 2, 1)
    assert s.astype(int).tolist() == [[1, 1, 1, 0, 0, 0], [1, 0, 1, 1, 0, 0], [1, 0, 0, 1, 1, 0], [1, 0, 0, 0, 1, 1]]
    assert not seen(3, 6, 0, 0).any() and seen(3, 6, 0, 2).sum() == 6
    assert seen(3, 6, -1, 0, length=0).sum() == 0 and seen(3, 6, -1, 0, length=2, start=0).sum(1).tolist() == [1, 2, 0]


def call(ops, **change):
    a = {"query": fake((2, 5, 4, 16)), "key": fake((2, 7, 2, 16)), "value": fake((2, 7, 2, 16)), "window": 4, "sinks": 1,
         "scale": None, "lengths": None, "starts": None}
    a.update(change)
    return ops.sliding_window_attention(**a)


@pytest.mark.parametrize("change", [
    {"query": fake((2, 5, 4, 16), "int32")},
    {"query": fake((2, 5, 4, 16), "float16")},
    {"value": fake((2, 7, 2, 16), "float32")},
    {"query": fake((2, 5, 4, 16), device=-1)},
    {"key": fake((2, 7, 2, 16), device=1)},
    {"query": fake((5, 4, 16))},
    {"query": fake((2, 5, 4, 136)), "key": fake((2, 7, 2, 136)), "value": fake((2, 7, 2, 136))},
    {"lengths": fake((2,), "float32")},
    {"starts": fake((2,), "int64", device=1)},
], ids=["integers", "mixed", "value_type", "host", "device", "axes", "wide", "length_type", "start_device"])
def test_declined(ops, change):
    with pytest.raises(mod("tensor").DeclinedError):
        call(ops, **change)


@pytest.mark.parametrize("change,message", [
    ({"value": fake((2, 8, 2, 16))}, "differ in shape"),
    ({"key": fake((3, 7, 2, 16)), "value": fake((3, 7, 2, 16))}, "sequences"),
    ({"key": fake((2, 7, 2, 24)), "value": fake((2, 7, 2, 24))}, "heads of"),
    ({"key": fake((2, 7, 3, 16)), "value": fake((2, 7, 3, 16))}, "share"),
    ({"key": fake((2, 7, 0, 16)), "value": fake((2, 7, 0, 16))}, "share"),
    ({"sinks": -1}, "sinks"),
    ({"scale": 0.0}, "scale"), ({"scale": -1.0}, "scale"), ({"scale": float("nan")}, "scale"),
    ({"scale": float("inf")}, "scale"), ({"scale": 3e38}, "scale"), ({"scale": 1e-60}, "scale"),
    ({"lengths": fake((3,), "int32")}, "lengths"),
    ({"starts": fake((2, 1), "int32")}, "starts"),
    ({"key": fake((2, 1 << 30, 2, 16)), "value": fake((2, 1 << 30, 2, 16))}, "2\\^30"),
])
def test_refused(ops, change, message):
    with pytest.raises(mod("tensor").DeviceError, match=message):
        call(ops, **change)


@pytest.mark.parametrize("change,error", [
    ({0: fake((2, 5, 4, 8))}, "DeviceError"),
    ({0: fake((2, 5, 4, 16), "float32")}, "DeclinedError"),
    ({4: fake((2, 5, 2, 16))}, "DeviceError"),
    ({5: fake((2, 5, 4), "float32")}, "DeviceError"),
    ({5: fake((2, 4, 5), "bfloat16")}, "DeclinedError"),
], ids=["gradient_shape", "gradient_type", "out_shape", "lse_shape", "lse_type"])
def test_backward_refused(ops, change, error):
    a = [fake((2, 5, 4, 16)), fake((2, 5, 4, 16)), fake((2, 7, 2, 16)), fake((2, 7, 2, 16)), fake((2, 5, 4, 16)),
         fake((2, 4, 5), "float32")]
    for i, t in change.items():
        a[i] = t
    with pytest.raises(getattr(mod("tensor"), error)):
        ops.sliding_window_attention_backward(*a, window=4)


@pytest.mark.parametrize("query,error", [(None, "DeviceError"), (fake(()), "DeclinedError"), (fake((16,)), "DeclinedError")],
                         ids=["none", "scalar", "one_axis"])
def test_refused_without_a_scale(ops, query, error):
    """The default scale asks a query for its last axis: one that has none is
    refused as it is with a scale."""
    t = mod("tensor")
    with pytest.raises(getattr(t, error)) as given:
        call(ops, query=query, scale=0.25)
    with pytest.raises(getattr(t, error)) as default:
        call(ops, query=query)
    assert str(default.value) == str(given.value)


@pytest.mark.parametrize("n,want", [(5, 5), (-1, -1), (2 ** 63 - 1, 2 ** 63 - 1), (2 ** 63, 2 ** 63 - 1), (2 ** 70, 2 ** 63 - 1),
                                    (-2 ** 70, -2 ** 63)])
def test_numbers_of_tokens_past_64_bits(ops, n, want):
    """They do not come around: 2^70 is no window of 0."""
    assert ops._tokens(n) == want
