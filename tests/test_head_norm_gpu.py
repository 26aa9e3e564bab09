"""The norm and rotation of each head's query and key on the GPU against
float64.

Tolerances, u = 2^-24.  A row's sum of squares is a chain of at most 16
fused steps a lane and 6 exchanges, all terms positive: at most 22 u, halved
by the root, which with the division and the sum's scaling makes r right to
14 u.  n takes two more roundings, the turn three: y is within 20 u of
|a| + |b|, its pair's magnitudes.  Backward: g has 3 u of |a| + |b|, u and
m one each, their mean 23 u of the mean of |u m|, dx two more: 32 u of the
magnitudes covers it.  dw is a chain of the rows one group takes, 32 or
fewer groups and the blocks: never more than (rows + 40) u of the sum of its
terms' magnitudes.  Then one rounding to the type.
"""

import numpy as np
import pytest

from _attention import (BF16, F16, F32, U, assert_within, head_norm, head_norm_backward, mod, put, sample, table_of, wide)

pytestmark = pytest.mark.gpu

DTYPES = [F32, F16, BF16]
IDS = ["fp32", "fp16", "bf16"]
SIZES = [(128, 128), (64, 64), (80, 40), (96, 96), (256, 64), (2, 2), (6, 4), (33, 16), (7, 0), (130, 130), (1024, 1024),
         (1000, 500), (136, 128), (40, 32)]


def check(ops, dtype, q, k, dq_, dk_, table, pos, qw, kw, interleaved, eps=1e-6, views=None, pos_dev=None):
    """Forward and backward of both sides against float64; ``views`` are the
    device operands when they are not plain copies."""
    dev = views or [put(x, dtype) for x in (q, k, dq_, dk_)]
    dqw, dkw = (None if w is None else put(w, dtype) for w in (qw, kw))
    tab = put(table)
    pos_dev = pos_dev if pos_dev is not None else put(pos)
    got = ops.qk_norm_rope(dev[0], dev[1], tab, pos_dev, dqw, dkw, eps, interleaved)
    grads = ops.qk_norm_rope_backward(dev[2], dev[3], dev[0], dev[1], tab, pos_dev, got[2], got[3], dqw, dkw, interleaved)
    p = np.broadcast_to(pos, q.shape[:-2])
    for s, (x, w, dy, name) in enumerate([(q, qw, dq_, "query"), (k, kw, dk_, "key")]):
        x64, dy64 = wide(x, dtype), wide(dy, dtype)
        w64 = np.ones(x.shape[-1]) if w is None else wide(w, dtype)
        y, r, mag = head_norm(x64, w64, table, p, eps, interleaved)
        assert got[s].is_contiguous() and got[s].shape == x.shape and got[2 + s].shape == x.shape[:-1]
        assert_within(got[s].numpy(), y, 20 * U * mag, dtype, name)
        assert_within(got[2 + s].numpy(), r, 14 * U * r, F32, name + " rstd")
        r32 = got[2 + s].numpy().astype(np.float64)
        dx, dw, mag, total = head_norm_backward(dy64, x64, r32, w64, table, p, interleaved)
        rows = x[..., 0].size
        assert_within(grads[s].numpy(), dx, 32 * U * mag, dtype, "d" + name)
        assert_within(grads[2 + s].numpy(), dw, (rows + 40) * U * total, dtype, "weight of " + name)
    return got, grads


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("dim,rotary", SIZES)
def test_sizes(dev, ops, dtype, dim, rotary, interleaved):
    b, t, h, hk = 2, 5, 6, 2
    q, k = sample((b, t, h, dim), dtype, 1, 1.5, 0.2), sample((b, t, hk, dim), dtype, 2, 0.7)
    dq, dk = sample((b, t, h, dim), dtype, 3), sample((b, t, hk, dim), dtype, 4)
    pos = np.random.default_rng(5).integers(0, 300, (b, t))
    check(ops, dtype, q, k, dq, dk, table_of(300, rotary), pos, sample((dim,), dtype, 6, 0.2, 1.0),
          sample((dim,), dtype, 7, 0.2, 1.0), interleaved)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1,), (1, 1), (3, 1), (1, 777), (2, 3, 41), ()], ids=str)
def test_token_axes_and_no_weights(dev, ops, dtype, shape):
    h, hk, dim = 5, 3, 64
    q, k = sample((*shape, h, dim), dtype, 11), sample((*shape, hk, dim), dtype, 12)
    dq, dk = sample((*shape, h, dim), dtype, 13), sample((*shape, hk, dim), dtype, 14)
    pos = np.random.default_rng(15).integers(0, 100, shape[-1:]).astype(np.int32)
    check(ops, dtype, q, k, dq, dk, table_of(100, dim), pos, None, None, False)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("lead", [0, 1, 3])
def test_views_of_a_packed_projection(dev, ops, dtype, lead):
    """Query and key as views of one projection's output that starts at any
    element; gradients that lie heads first; positions of every other token."""
    b, t, h, hk, dim = 3, 7, 4, 2, 80
    width = (h + 2 * hk) * dim
    flat = sample((b * t * width + lead,), dtype, 21)
    packed = flat[lead:].reshape(b, t, width)
    dpacked = put(flat, dtype)[lead:].view(b, t, width)

    def heads(x, first, n):
        if isinstance(x, np.ndarray):
            return x[..., first * dim: (first + n) * dim].reshape(b, t, n, dim)
        part = x[:, :, first * dim: (first + n) * dim]
        return part._view([b, t, n, dim], [part.strides[0], part.strides[1], dim, 1])

    dq, dk = sample((b, h, t, dim), dtype, 22), sample((b, hk, t, dim), dtype, 23)
    pos = np.random.default_rng(24).integers(0, 64, (2 * t,))
    check(ops, dtype, heads(packed, 0, h), heads(packed, h, hk), dq.transpose(0, 2, 1, 3), dk.transpose(0, 2, 1, 3),
          table_of(64, dim), pos[::2], sample((dim,), dtype, 25, 0.2, 1.0), sample((dim,), dtype, 26, 0.2, 1.0), True,
          views=[heads(dpacked, 0, h), heads(dpacked, h, hk), put(dq, dtype).transpose(1, 2), put(dk, dtype).transpose(1, 2)],
          pos_dev=put(pos)[::2])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_layouts_that_are_copied(dev, ops, dtype):
    """A strided last axis, and token axes that do not merge into two."""
    shape = (2, 2, 3, 4, 24)
    big = sample((2, 2, 3, 4, 48), dtype, 31)
    turned = sample((2, 3, 2, 4, 24), dtype, 32)
    q, k = np.ascontiguousarray(big[..., ::2]), np.ascontiguousarray(turned.transpose(0, 2, 1, 3, 4))
    dq, dk = sample(shape, dtype, 33), sample(shape, dtype, 34)
    views = [put(big, dtype)[:, :, :, :, ::2], put(turned, dtype).permute(0, 2, 1, 3, 4), put(dq, dtype), put(dk, dtype)]
    pos = np.arange(3)
    check(ops, dtype, q, k, dq, dk, table_of(8, 24), pos, None, sample((24,), dtype, 35), False, views=views)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_many_rows(dev, ops, dtype):
    """More rows than the backward's groups: each walks several."""
    b, t, h, hk, dim = 2, 1501, 16, 2, 128
    q, k = sample((b, t, h, dim), dtype, 41), sample((b, t, hk, dim), dtype, 42)
    dq, dk = sample((b, t, h, dim), dtype, 43), sample((b, t, hk, dim), dtype, 44)
    got, grads = check(ops, dtype, q, k, dq, dk, table_of(2000, dim), np.arange(t) + 400, sample((dim,), dtype, 45, 0.2, 1.0),
                       sample((dim,), dtype, 46, 0.2, 1.0), False)
    # the same call gives the same bits, and outputs masked off leave the others alone
    dev_ = [put(x, dtype) for x in (dq, dk, q, k)]
    pos, tab = put(np.arange(t) + 400), put(table_of(2000, dim))
    ws = [put(sample((dim,), dtype, s, 0.2, 1.0), dtype) for s in (45, 46)]
    for mask in [(True,) * 4, (False, True, True, False), (True, False, False, True), (False,) * 4]:
        again = ops.qk_norm_rope_backward(*dev_, tab, pos, got[2], got[3], *ws, output_mask=mask)
        for want, a, first in zip(mask, again, grads):
            assert (a is not None) == want
            assert a is None or np.array_equal(a.numpy(), first.numpy())


def test_positions_outside_the_table(dev, ops):
    """Rows of NaN and no read, whatever the position; the others as ever."""
    q, k = sample((8, 3, 64), BF16, 51), sample((8, 1, 64), BF16, 52)
    pos = np.array([0, 9, 10, -1, 1 << 40, -(1 << 62), 3, 2 ** 31])
    y, ky, r, kr = ops.qk_norm_rope(put(q, BF16), put(k, BF16), put(table_of(10, 32)), put(pos))
    for got, x in ((y, q), (ky, k)):
        want, _, mag = head_norm(wide(x, BF16), np.ones(64), table_of(10, 32), pos, 1e-6, False)
        assert_within(got.numpy(), want, np.nan_to_num(20 * U * mag), BF16)
    assert np.isfinite(r.numpy()).all() and np.isfinite(kr.numpy()).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_rows_of_zeros_and_of_extremes(dev, ops, dtype):
    """A row of zeros stays zero (eps keeps r finite); an infinity makes its
    row NaN or zero as the formula does, and no other row."""
    q = sample((4, 2, 64), F32, 61)
    q[1] = 0.0
    q = orc_from(q, dtype)
    q[2, 1, 5] = orc_from(np.array([np.inf], np.float32), dtype)[0]
    y, _, r, _ = ops.qk_norm_rope(put(q, dtype), put(q, dtype), put(table_of(10, 64)), put(np.zeros(1, np.int64)))
    y64, r64 = wide(y.numpy(), dtype), r.numpy()
    assert (y64[1] == 0).all() and np.allclose(r64[1], 1e3, rtol=1e-6)
    assert r64[2, 1] == 0 and np.isnan(y64[2, 1, 5]) and np.isfinite(y64[2, 0]).all() and np.isfinite(y64[3]).all()


def orc_from(x, dtype):
    from oracle import binding
    return binding.from_float(x, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_no_tokens(dev, ops, dtype):
    """Empty results, and zero gradients of the weights."""
    q, k = put(sample((0, 4, 32), dtype), dtype), put(sample((0, 1, 32), dtype), dtype)
    w = put(sample((32,), dtype, 1), dtype)
    tab, pos = put(table_of(4, 32)), put(np.zeros((0,), np.int64))
    y, ky, r, kr = ops.qk_norm_rope(q, k, tab, pos, w, w)
    assert y.shape == (0, 4, 32) and ky.shape == (0, 1, 32) and r.shape == (0, 4) and kr.shape == (0, 1)
    dq, dk, dqw, dkw = ops.qk_norm_rope_backward(q, k, q, k, tab, pos, r, kr, w, w)
    assert dq.shape == (0, 4, 32) and dk.shape == (0, 1, 32)
    assert (wide(dqw.numpy(), dtype) == 0).all() and (wide(dkw.numpy(), dtype) == 0).all()


def test_recorded_and_replayed(dev, ops):
    """Forward and backward in a recording, replayed on new inputs between
    eager calls: the eager bits each time."""
    graph, runtime = mod("graph"), mod("runtime")
    shape, dim = (2, 65, 4, 64), 64
    x = [put(sample(shape, BF16, s), BF16) for s in (71, 72, 73, 74)]
    w, tab, pos = put(sample((dim,), BF16, 75, 0.2, 1.0), BF16), put(table_of(65, dim)), put(np.arange(65))

    def step():
        y, ky, r, kr = ops.qk_norm_rope(x[0], x[1], tab, pos, w, w)
        return [y, ky, r, kr, *ops.qk_norm_rope_backward(x[2], x[3], x[0], x[1], tab, pos, r, kr, w, w)]

    g = graph.Graph()
    try:
        results = g.capture(step)
        for i in range(4):
            for s, t in enumerate(x):
                ops.copy_(t, sample(shape, F32, 80 + 10 * i + s))
            g.replay()
            runtime.synchronize()
            for a, b in zip(results, step()):
                assert np.array_equal(a.numpy(), b.numpy())
    finally:
        g.reset()


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("dim,rotary", [(64, 0), (80, 48), (64, 32), (33, 16), (7, 0), (256, 64)])
def test_an_element_that_does_not_turn_stays_by_itself(dev, ops, dtype, dim, rotary, interleaved):
    """Elements past the rotated ones have no partner: where the weight or the
    gradient of one is infinite, the others' results and weight gradients are as
    without it."""
    h = 3
    q, k, dq, dk = (sample((2, 5, h, dim), dtype, 90 + i) for i in range(4))
    tab, pos = table_of(20, rotary), np.arange(10).reshape(2, 5)
    at = rotary
    others = np.arange(dim) != at
    w = sample((dim,), dtype, 95, 0.2, 1.0)
    w[at] = orc_from(np.array([np.inf], np.float32), dtype)[0]
    y, ky, r, kr = ops.qk_norm_rope(put(q, dtype), put(k, dtype), put(tab), put(pos), put(w, dtype), put(w, dtype), interleaved=interleaved)
    w64 = np.where(others, wide(w, dtype), 0.0)
    for got, x in ((y, q), (ky, k)):
        want, _, mag = head_norm(wide(x, dtype), w64, tab, pos, 1e-6, interleaved)
        assert_within(got.numpy()[..., others], want[..., others], 20 * U * mag[..., others], dtype)
        assert np.isinf(wide(got.numpy(), dtype)[..., at]).all()
    dq[1, 2, 1, at] = orc_from(np.array([np.inf], np.float32), dtype)[0]
    _, _, r, kr = ops.qk_norm_rope(put(q, dtype), put(k, dtype), put(tab), put(pos), interleaved=interleaved)
    grads = ops.qk_norm_rope_backward(put(dq, dtype), put(dk, dtype), put(q, dtype), put(k, dtype), put(tab), put(pos), r, kr,
                                      interleaved=interleaved)
    dy = wide(dq, dtype)
    dy[1, 2, 1, at] = 0.0
    _, dw, _, total = head_norm_backward(dy, wide(q, dtype), r.numpy().astype(np.float64), np.ones(dim), tab, pos, interleaved)
    assert_within(grads[2].numpy()[others], dw[others], 70 * U * total[others], dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_gradients_of_positions_outside_the_table(dev, ops, dtype):
    """NaN in such a token's rows and in the weights' gradients, whatever the
    gradient; the other tokens' rows as ever."""
    q, k, dq, dk = (sample((6, 2, 48), dtype, 100 + i) for i in range(4))
    pos, tab = np.array([0, 3, -1, 9, 10, 4]), table_of(10, 32)
    outside = (pos < 0) | (pos >= 10)
    dq[outside] = 0
    _, _, r, kr = ops.qk_norm_rope(put(q, dtype), put(k, dtype), put(tab), put(pos))
    grads = ops.qk_norm_rope_backward(put(dq, dtype), put(dk, dtype), put(q, dtype), put(k, dtype), put(tab), put(pos), r, kr)
    for got, weight, x, dy, stat in ((grads[0], grads[2], q, dq, r), (grads[1], grads[3], k, dk, kr)):
        dx, _, mag, _ = head_norm_backward(wide(dy, dtype), wide(x, dtype), stat.numpy().astype(np.float64), np.ones(48), tab, pos, False)
        assert np.isnan(dx[outside]).all()
        assert_within(got.numpy(), dx, np.nan_to_num(32 * U * mag), dtype)
        assert np.isnan(wide(weight.numpy(), dtype)).all()
