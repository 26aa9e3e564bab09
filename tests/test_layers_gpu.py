"""Dropout without a mask, the join of a block to its residual stream, and log
probabilities of tokens on the GPU against float64.  Bounds: `_layers.py`."""

import math

import numpy as np
import pytest

from oracle import binding as orc

from _attention import BF16, F16, F32, U, assert_within, mod, put, wide
from _attention import sample as sample_flat
from _layers import Join, Probs, kept

pytestmark = pytest.mark.gpu

DTYPES = [F32, F16, BF16]
IDS = ["fp32", "fp16", "bf16"]
SEED = (0x1234567 << 32) + 0x89ABCDEF


def sample(shape, *args, **kwargs):
    """Of no axes too (the oracle's bfloat16 has one at least)."""
    return sample_flat(shape, *args, **kwargs).reshape(shape)


def bits(x, dtype):
    return orc.from_float(np.asarray(x, np.float32), dtype)


# ---- dropout ------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1,), (3,), (7, 1), (8,), (1000,), (257, 33), (64, 4096), (2, 3, 5, 7), ()], ids=str)
def test_dropout_has_native_dropouts_bits(dev, ops, dtype, shape):
    x = sample(shape, dtype, 1, 2.0)
    for p in (0.1, 0.5, 0.93):
        want, mask = ops.native_dropout(put(x, dtype), p, True, SEED)
        got = ops.seeded_dropout(put(x, dtype), p, SEED)
        back = ops.seeded_dropout_backward(put(x, dtype), p, SEED)
        assert got.shape == shape and got.is_contiguous()
        assert np.array_equal(got.numpy(), want.numpy()) and np.array_equal(back.numpy(), want.numpy())
        assert np.array_equal(mask.numpy(), kept(p, SEED, shape))


def dropped(x, dtype, p, keep):
    """The float32 product with 1 / (1 - p), rounded to the type."""
    return bits(np.where(keep, wide(x, dtype).astype(np.float32) * np.float32(1.0 / (1.0 - p)), np.float32(0)), dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_dropout_offsets_and_seeds_in_memory(dev, ops, dtype):
    x = sample((513,), dtype, 2)
    seeds = put(np.array([5, -7, SEED], np.int64))
    for i, seed in enumerate((5, (1 << 64) - 7, SEED)):
        for offset in (0, 1, (3 << 32) + 9):
            keep = kept(0.4, seed, x.shape, offset)
            want = dropped(x, dtype, 0.4, keep)
            for s in (seed, seeds[i], seeds[i: i + 1]):
                got = ops.seeded_dropout(put(x, dtype), 0.4, s, offset).numpy()
                assert np.array_equal(got, want) and ((wide(got, dtype) != 0) <= keep).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_dropout_of_none_and_of_all(dev, ops, dtype):
    x = sample((37, 5), dtype, 3)
    x[3, 2], x[4, 1] = bits([np.nan], dtype)[0], bits([np.inf], dtype)[0]
    none, all_ = ops.seeded_dropout(put(x, dtype), 0.0, 1).numpy(), ops.seeded_dropout(put(x, dtype), 1.0, 1).numpy()
    assert np.array_equal(wide(none, dtype), wide(x, dtype), equal_nan=True)
    assert (wide(all_, dtype) == 0).all()
    # what is not finite goes where it is dropped
    keep = kept(0.5, 11, x.shape)
    got = wide(ops.seeded_dropout(put(x, dtype), 0.5, 11).numpy(), dtype)
    assert np.isnan(got[3, 2]) == keep[3, 2] and np.isinf(got[4, 1]) == keep[4, 1]
    assert (got[~keep] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_dropout_of_views(dev, ops, dtype):
    """Elements count in row-major order of the view, wherever it starts."""
    x = sample((9, 14), dtype, 4)
    d = put(x, dtype)
    for view, host in ((d.t(), x.T), (d[1:, 3:], x[1:, 3:]), (d[:, ::2], x[:, ::2]), (d[2], x[2]), (d[2, 1:], x[2, 1:])):
        want = dropped(host, dtype, 0.3, kept(0.3, 9, host.shape))
        assert np.array_equal(ops.seeded_dropout(view, 0.3, 9).numpy(), want)


def test_dropout_of_nothing(dev, ops):
    assert ops.seeded_dropout(put(np.zeros((0, 4), np.float32)), 0.5, 1).shape == (0, 4)


# ---- the join --------------------------------------------------------------------------

# gate, branch's norm, its weight, norm, its weight, p, scales
FORMS = {
    "plain": (None, False, False, True, True, 0.0, (1.0, 1.0)),
    "both_norms": (None, True, True, True, True, 0.0, (1.0, 0.3)),
    "no_weights": (None, True, False, True, False, 0.0, (0.8, 1.0)),
    "no_norm": ("channel", False, False, False, False, 0.3, (1.0, 1.0)),
    "branch_norm_only": ("token", True, True, False, False, 0.0, (0.9, -1.2)),
    "channel": ("channel", True, True, True, True, 0.1, (0.9, 0.4)),
    "sequence": ("sequence", True, True, True, True, 0.2, (1.0, 1.0)),
    "sequence_one": ("sequence_one", False, False, True, True, 0.0, (1.0, 0.5)),
    "token": ("token", True, True, True, True, 0.5, (1.0, 1.0)),
    "full": ("full", True, True, True, True, 0.1, (1.0, 1.0)),
    "one": ("one", False, False, True, True, 0.1, (1.0, 1.0)),
    "scalar": ("scalar", True, True, True, True, 0.0, (1.0, 1.0)),
    "all_dropped": ("channel", True, True, True, True, 1.0, (1.0, 1.0)),
}


def gate_shape(kind, shape):
    b, d = shape[0], shape[-1]
    ones = (1,) * (len(shape) - 2)
    return {"channel": (d,), "sequence": (b, *ones, d), "sequence_one": (b, *ones, 1), "token": (*shape[:-1], 1), "full": shape,
            "one": (1,), "scalar": ()}[kind]


def check_join(ops, dtype, shape, form, seed=0, views=None, grads=(True, True), mask=None):
    """Forward and backward of one form against float64; ``views`` turns a
    host array into the device operand."""
    kind, norm1, has1, norm2, has2, p, (a, b) = FORMS[form]
    dim = shape[-1]
    x, y = sample(shape, dtype, seed + 1, 1.5, 0.1), sample(shape, dtype, seed + 2, 0.7)
    dz, dh = sample(shape, dtype, seed + 3), sample(shape, dtype, seed + 4)
    gate = None if kind is None else sample(gate_shape(kind, shape), dtype, seed + 5, 0.4, 0.9)
    w1 = sample((dim,), dtype, seed + 6, 0.2, 1.0) if has1 else None
    w2 = sample((dim,), dtype, seed + 7, 0.2, 1.0) if has2 else None
    place = views or (lambda v: put(v, dtype))
    dx_, dy_, ddz, ddh = (place(v) for v in (x, y, dz, dh))
    dgate, dw1, dw2 = (None if v is None else put(v, dtype) for v in (gate, w1, w2))
    eps1, eps2 = 1e-5 if norm1 else None, 1e-6 if norm2 else None
    key = SEED + seed
    got = ops.residual_norm(dx_, dy_, dgate, dw1, dw2, a, b, eps1, eps2, p, key)
    back = ops.residual_norm_backward(ddz if grads[0] else None, ddh if norm2 and grads[1] else None, dx_, dy_, got[2], got[3], dgate, dw1,
                                      dw2, a, b, p, key)
    wide_ = [None if v is None else wide(v, dtype).reshape(v.shape) for v in (x, y, gate, w1, w2)]
    j = Join(*wide_, a=float(np.float32(a)), b=float(np.float32(b)), eps1=eps1, eps2=eps2, keep=kept(p, key, shape), p=p)
    assert got[0].shape == shape and got[0].is_contiguous()
    assert_within(got[0].numpy(), j.z, j.z_bound, dtype, "sum")
    assert (got[1] is None) == (got[3] is None) == (not norm2) and (got[2] is None) == (not norm1)
    if norm1:
        assert_within(got[2].numpy(), j.r1, j.r1_bound, F32, "branch_rstd")
    if norm2:
        assert_within(got[1].numpy(), j.h, j.h_bound, dtype, "normed")
        assert_within(got[3].numpy(), j.r2, j.r2_bound, F32, "rstd")
    r1, r2 = (None if t is None else t.numpy().astype(np.float64) for t in got[2:])
    want, bound = j.backward(wide(dz, dtype) if grads[0] else None, wide(dh, dtype) if norm2 and grads[1] else None, r1, r2)
    for g, name in zip(back, ("dx", "dy", "dgate", "dw1", "dw2")):
        assert (g is not None) == (name in want), name
        if g is not None:
            assert g.shape == want[name].shape and g.is_contiguous()
            assert_within(np.atleast_1d(g.numpy()), np.atleast_1d(want[name]), np.atleast_1d(bound[name]), dtype, name)
    return got, back


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(3, 5, 64), (2, 7, 1001), (4, 1, 2), (2, 3, 3, 72)], ids=str)
def test_join_forms(dev, ops, dtype, shape, form):
    check_join(ops, dtype, shape, form)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("dim", [1, 2, 7, 8, 9, 16, 63, 100, 256, 257, 504, 512, 513, 520, 1024, 2047, 4096, 4100, 5000, 8192, 8193,
                                 9999, 16383, 16384])
def test_join_widths(dev, ops, dtype, dim):
    for i, form in enumerate(("both_norms", "channel", "token", "full")):
        check_join(ops, dtype, (2, 3, dim), form, seed=10 * i)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("form", ["channel", "sequence", "sequence_one", "one", "token"])
@pytest.mark.parametrize("shape", [(1, 1, 128), (1, 3000, 72), (700, 3, 40), (5, 401, 1100), (1500, 1, 16), (40, 33, 520)], ids=str)
def test_join_many_rows(dev, ops, dtype, form, shape):
    """More rows than blocks, more groups than blocks, groups of a few rows."""
    check_join(ops, dtype, shape, form)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("form", ["plain", "both_norms", "no_norm", "channel", "full"])
@pytest.mark.parametrize("dim", [129, 191, 193, 257, 267, 383, 384, 385, 513, 601, 767, 768, 769, 1025, 1100, 1535, 1536, 1537])
def test_join_many_rows_between_powers_of_two(dev, ops, dtype, form, dim):
    check_join(ops, dtype, (13, 47, dim), form)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(64,), (5, 64), (2, 2, 2, 2, 2, 2, 2, 24)], ids=str)
def test_join_axes(dev, ops, dtype, shape):
    for form in ("plain", "no_norm", "scalar"):
        check_join(ops, dtype, shape, form)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_join_of_views(dev, ops, dtype):
    """Rows some distance apart that start at any element, read in place; and
    layouts that are copied."""
    def spaced(v):
        big = sample((v.shape[0], v.shape[1], v.shape[2] + 11), dtype, 99)
        big[..., 3: 3 + v.shape[2]] = v
        return put(big, dtype)[:, :, 3: 3 + v.shape[2]]

    def turned(v):
        return put(np.ascontiguousarray(v.transpose(1, 0, 2)), dtype).transpose(0, 1)

    def strided(v):
        return put(np.repeat(v, 2, axis=2), dtype)[:, :, ::2]

    for place in (spaced, turned, strided):
        for shape in ((3, 4, 100), (2, 5, 1003)):
            check_join(ops, dtype, shape, "channel", views=place)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("dim", [48, 1004])
def test_join_gates_as_views(dev, ops, dtype, dim):
    """A gate that is a slice, a transposed one, an expanded one."""
    b, t = 3, 4
    x, y, dz, dh = (sample((b, t, dim), dtype, 30 + i) for i in range(4))
    wide_gate = sample((b, 1, 3 * dim + 1), dtype, 35)
    turned = sample((t, b, dim), dtype, 36)
    one = sample((b, 1, 1), dtype, 37)
    for host, view in ((wide_gate[..., dim + 1: 2 * dim + 1], put(wide_gate, dtype)[:, :, dim + 1: 2 * dim + 1]),
                       (np.ascontiguousarray(turned.transpose(1, 0, 2)), put(turned, dtype).transpose(0, 1)),
                       (np.broadcast_to(one, (b, t, dim)), put(one, dtype).expand(b, t, dim))):
        d = [put(v, dtype) for v in (x, y, dz, dh)]
        z, h, r1, r2 = ops.residual_norm(d[0], d[1], view)
        j = Join(wide(x, dtype), wide(y, dtype), wide(np.ascontiguousarray(host), dtype))
        assert_within(z.numpy(), j.z, j.z_bound, dtype)
        assert_within(h.numpy(), j.h, j.h_bound, dtype)
        grads = ops.residual_norm_backward(d[2], d[3], d[0], d[1], r1, r2, view)
        want, bound = j.backward(wide(dz, dtype), wide(dh, dtype), None, r2.numpy().astype(np.float64))
        for g, name in zip(grads, ("dx", "dy", "dgate")):
            assert_within(g.numpy(), want[name], bound[name], dtype, name)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(6, 96), (3, 2, 1500)], ids=str)
def test_norm_alone(dev, ops, dtype, shape):
    x, dz, dh = (sample(shape, dtype, 40 + i) for i in range(3))
    w = sample(shape[-1:], dtype, 44, 0.2, 1.0)
    none, h, r1, r2 = ops.residual_norm(put(x, dtype), weight=put(w, dtype))
    assert none is None and r1 is None
    j = Join(wide(x, dtype), w2=wide(w, dtype))
    assert_within(h.numpy(), j.h, j.h_bound, dtype)
    for first in (None, dz):
        grads = ops.residual_norm_backward(None if first is None else put(first, dtype), put(dh, dtype), put(x, dtype), rstd=r2,
                                           weight=put(w, dtype))
        want, bound = j.backward(None if first is None else wide(first, dtype), wide(dh, dtype), None, r2.numpy().astype(np.float64))
        assert [g is not None for g in grads] == [True, False, False, False, True]
        assert_within(grads[0].numpy(), want["dx"], bound["dx"], dtype)
        assert_within(grads[4].numpy(), want["dw2"], bound["dw2"], dtype)


@pytest.mark.parametrize("grads", [(True, False), (False, True)], ids=["sum", "normed"])
@pytest.mark.parametrize("form", ["channel", "token"])
def test_join_with_one_gradient(dev, ops, form, grads):
    for shape in ((3, 4, 200), (2, 3, 1200)):
        _, back = check_join(ops, BF16, shape, form, grads=grads)
        if not grads[1]:
            assert (wide(back[4].numpy(), BF16) == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("form", ["channel", "sequence", "full", "token"])
def test_join_outputs_masked_off(dev, ops, dtype, form):
    """The same bits every time, whichever of them are asked for."""
    kind, _, _, _, _, p, (a, b) = FORMS[form]
    shape = (4, 33, 264)
    x, y, dz, dh = (put(sample(shape, dtype, i), dtype) for i in range(4))
    gate = put(sample(gate_shape(kind, shape), dtype, 5), dtype)
    w1, w2 = (put(sample(shape[-1:], dtype, i, 0.2, 1.0), dtype) for i in (6, 7))
    _, _, r1, r2 = ops.residual_norm(x, y, gate, w1, w2, a, b, 1e-6, 1e-6, p, SEED)
    first = None
    for mask in [(True,) * 5, (False, True, False, True, False), (True, False, True, False, True), (False, False, True, False, False),
                 (False, False, False, False, True), (False,) * 5]:
        again = ops.residual_norm_backward(dz, dh, x, y, r1, r2, gate, w1, w2, a, b, p, SEED, output_mask=mask)
        first = first or again
        for want, got, all_ in zip(mask, again, first):
            assert (got is not None) == want
            assert got is None or np.array_equal(got.numpy(), all_.numpy())


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(0, 4, 32), (3, 0, 32), (0, 2048)], ids=str)
def test_join_of_no_rows(dev, ops, dtype, shape):
    x, dim = put(np.zeros(shape, np.float32)[..., :] if dtype == F32 else sample(shape, dtype), dtype), shape[-1]
    w, gate = put(sample((dim,), dtype, 1), dtype), put(sample((dim,), dtype, 2), dtype)
    z, h, r1, r2 = ops.residual_norm(x, x, gate, w, w, branch_eps=1e-6)
    assert z.shape == h.shape == shape and r1.shape == r2.shape == shape[:-1]
    grads = ops.residual_norm_backward(x, x, x, x, r1, r2, gate, w, w)
    assert grads[0].shape == grads[1].shape == shape
    assert all(g.shape == (dim,) and (wide(g.numpy(), dtype) == 0).all() for g in grads[2:])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("dim", [72, 1032])
def test_join_rows_stay_by_themselves(dev, ops, dtype, dim):
    """Rows of zeros stay finite by eps; what is not finite stays in its row,
    and out of it where it is dropped."""
    shape = (6, dim)
    x, y, dz, dh = (sample(shape, dtype, 50 + i) for i in range(4))
    x[0] = y[0] = 0
    keep = kept(0.5, 3, shape)
    at_kept, at_dropped = int(np.flatnonzero(keep[1])[0]), int(np.flatnonzero(~keep[2])[0])
    y[1, at_kept], y[2, at_dropped] = bits([np.inf], dtype)[0], bits([np.nan], dtype)[0]
    d = [put(v, dtype) for v in (x, y, dz, dh)]
    z, h, _, r2 = ops.residual_norm(d[0], d[1], p=0.5, seed=3)
    j = Join(wide(x, dtype), wide(y, dtype), keep=keep, p=0.5)
    assert_within(z.numpy(), j.z, np.nan_to_num(j.z_bound), dtype)
    rows = [0, 2, 3, 4, 5]
    assert_within(h.numpy()[rows], j.h[rows], j.h_bound[rows], dtype)
    assert np.isinf(j.z[1, at_kept]) and r2.numpy()[1] == 0
    dx, dy, _, _, _ = ops.residual_norm_backward(d[2], d[3], d[0], d[1], None, r2, p=0.5, seed=3)
    with np.errstate(invalid="ignore"):
        want, bound = j.backward(wide(dz, dtype), wide(dh, dtype), None, r2.numpy().astype(np.float64))
    for got, name in ((dx, "dx"), (dy, "dy")):
        assert_within(got.numpy()[rows], want[name][rows], bound[name][rows], dtype)
    assert (wide(dy.numpy(), dtype)[~keep] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("dim", [36, 1028, 1031])
def test_join_drops_infinite_gradients(dev, ops, dtype, dim):
    """A gradient that is not finite at a dropped element does not reach the
    branch's norm by it."""
    shape = (3, dim)
    x, y, dz = (sample(shape, dtype, 60 + i) for i in range(3))
    keep = kept(0.5, 4, shape)
    dz[1, int(np.flatnonzero(~keep[1])[0])] = bits([np.inf], dtype)[0]
    d = [put(v, dtype) for v in (x, y, dz)]
    _, _, r1, _ = ops.residual_norm(d[0], d[1], branch_eps=1e-6, eps=None, p=0.5, seed=4)
    _, dy, _, _, _ = ops.residual_norm_backward(d[2], None, d[0], d[1], r1, p=0.5, seed=4)
    finite = np.where(np.isfinite(wide(dz, dtype)), wide(dz, dtype), 0.0)
    j = Join(wide(x, dtype), wide(y, dtype), eps1=1e-6, eps2=None, keep=keep, p=0.5)
    want, bound = j.backward(finite, None, r1.numpy().astype(np.float64))
    assert_within(dy.numpy(), want["dy"], bound["dy"], dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("gate", [None, "channel", "token"])
@pytest.mark.parametrize("branch_norm", [False, True], ids=["", "branch_norm"])
@pytest.mark.parametrize("dim", [36, 1028, 9000])
def test_join_without_a_gradient_of_its_norm(dev, ops, dtype, dim, branch_norm, gate):
    """No gradient comes through the sum then: what is not finite in the residual,
    in the norm's weight, or elsewhere in a row of the branch, reaches none."""
    shape = (5, dim)
    x, y, dz = (sample(shape, dtype, 70 + i) for i in range(3))
    x[1, 3], x[2, dim - 1] = bits([np.inf], dtype)[0], bits([np.nan], dtype)[0]
    y[3, 5], y[4, 0] = bits([np.inf], dtype)[0], bits([np.nan], dtype)[0]
    w2 = sample((dim,), dtype, 74, 0.2, 1.0)
    w2[7] = bits([np.inf], dtype)[0]
    g = None if gate is None else sample(gate_shape(gate, shape), dtype, 75, 0.4, 0.9)
    d = [None if v is None else put(v, dtype) for v in (x, y, g, w2, dz)]
    eps1 = 1e-6 if branch_norm else None
    for weight in (None, d[3]):
        _, _, r1, r2 = ops.residual_norm(d[0], d[1], d[2], None, weight, 0.5, 0.75, eps1, None if weight is None else 1e-6)
        back = ops.residual_norm_backward(d[4], None, d[0], d[1], r1, r2, d[2], None, weight, 0.5, 0.75)
        # two products, and the rounding to the type
        assert_within(back[0].numpy(), 0.5 * wide(dz, dtype), 2.0 ** -22 * np.abs(wide(dz, dtype)), dtype, "dx")
        dy = 0.75 * wide(dz, dtype) * (1.0 if g is None else wide(g, dtype))
        if not branch_norm:
            assert_within(back[1].numpy(), dy, 2.0 ** -22 * np.abs(dy), dtype, "dy")
        gate3 = None if g is None else wide(g, dtype)[:3] if gate == "token" else wide(g, dtype)
        j = Join(np.zeros((3, dim)), wide(y, dtype)[:3], gate3, a=0.5, b=0.75, eps1=eps1, eps2=None)
        want, bound = j.backward(wide(dz, dtype)[:3], None, r1.numpy()[:3].astype(np.float64) if branch_norm else None)
        assert_within(back[1].numpy()[:3], want["dy"], bound["dy"], dtype, "dy")
        if gate == "token":
            assert_within(back[2].numpy()[:3], want["dgate"], bound["dgate"], dtype, "dgate")
        if weight is not None:
            assert (wide(back[4].numpy(), dtype) == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("gate", ["channel", "sequence", "sequence_one", "token", "full", "one"])
@pytest.mark.parametrize("dim", [5, 36, 1028, 9000])
def test_join_gate_of_dropped_elements_that_are_not_finite(dev, ops, dtype, gate, dim):
    """A dropped element of the branch has no part in the gate's gradient,
    whatever it holds."""
    shape = (3, 4, dim)
    x, y, dz, dh = (sample(shape, dtype, 80 + i) for i in range(4))
    g, keep = sample(gate_shape(gate, shape), dtype, 84, 0.4, 0.9), kept(0.5, 6, shape)
    out = np.flatnonzero(~keep)
    for i, value in enumerate((np.inf, np.nan, -np.inf)):
        y.reshape(-1)[out[i::7]] = bits([value], dtype)[0]
    d = [put(v, dtype) for v in (x, y, g, dz, dh)]
    z, h, _, r2 = ops.residual_norm(d[0], d[1], d[2], p=0.5, seed=6)
    j = Join(wide(x, dtype), wide(y, dtype), wide(g, dtype).reshape(g.shape), keep=keep, p=0.5)
    assert_within(z.numpy(), j.z, j.z_bound, dtype)
    assert_within(h.numpy(), j.h, j.h_bound, dtype)
    for grad_normed in (d[4], None):
        got = ops.residual_norm_backward(d[3], grad_normed, d[0], d[1], None, r2, d[2], p=0.5, seed=6)
        want, bound = j.backward(wide(dz, dtype), None if grad_normed is None else wide(dh, dtype), None, r2.numpy().astype(np.float64))
        for a, name in zip(got, ("dx", "dy", "dgate")):
            assert_within(a.numpy(), want[name], bound[name], dtype, name)
        assert (wide(got[1].numpy(), dtype)[~keep] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("branch_norm", [False, True], ids=["", "branch_norm"])
@pytest.mark.parametrize("dim", [5, 36, 1028, 9000])
def test_join_infinite_gate_of_dropped_elements(dev, ops, dtype, dim, branch_norm):
    """Nor has a dropped element a gradient by a gate or a weight that is not
    finite."""
    shape = (3, 4, dim)
    x, y, dz = (sample(shape, dtype, 90 + i) for i in range(3))
    w, infinite = sample((dim,), dtype, 93, 0.2, 1.0), bits([np.inf], dtype)[0]
    eps1, weight = (1e-6, put(w, dtype)) if branch_norm else (None, None)
    d = [put(v, dtype) for v in (x, y, dz)]
    # a gate of its own for every element, infinite where that is dropped
    g, keep = sample(shape, dtype, 94, 0.4, 0.9), kept(0.5, 7, shape)
    hidden = g.copy()
    hidden.reshape(-1)[np.flatnonzero(~keep)[::5]] = infinite
    r1 = ops.residual_norm(d[0], d[1], put(hidden, dtype), weight, None, 1.0, 1.0, eps1, None, 0.5, 7)[2]
    got = ops.residual_norm_backward(d[2], None, d[0], d[1], r1, None, put(hidden, dtype), weight, p=0.5, seed=7)
    j = Join(wide(x, dtype), wide(y, dtype), wide(g, dtype), wide(w, dtype) if branch_norm else None, eps1=eps1, eps2=None, keep=keep, p=0.5)
    want, bound = j.backward(wide(dz, dtype), None, None if r1 is None else r1.numpy().astype(np.float64))
    for a, name in zip(got, ("dx", "dy", "dgate", "dw1")):
        assert (a is not None) == (name in want)
        if a is not None:
            assert_within(a.numpy(), want[name], bound[name], dtype, name)
    # every element dropped: no gradient at all but the residual's
    w[dim // 2] = infinite
    weight = put(w, dtype) if branch_norm else None
    for kind in ("channel", "sequence", "sequence_one", "token", "full", "one"):
        g = np.full(gate_shape(kind, shape), infinite)
        got = ops.residual_norm_backward(d[2], None, d[0], d[1], r1, None, put(g, dtype), weight, p=1.0, seed=7)
        assert_within(got[0].numpy(), wide(dz, dtype), 0.0, dtype, "dx")
        for a in got[1:]:
            assert a is None or (wide(a.numpy(), dtype) == 0).all(), kind


# ---- log probabilities --------------------------------------------------------------------


def rows_of_logits(rows, vocab, dtype, seed, std=2.5):
    x = sample((rows, vocab), dtype, seed, std)
    return x


def check_probs(ops, dtype, x, targets, scale=1.0, top=0, ignore=-100, view=None, entropy=True, back=True, lanes=256):
    logits = view if view is not None else put(x, dtype)
    t = None if targets is None else put(targets)
    got = ops.token_log_probs(logits, t, scale, top, entropy, ignore)
    x64 = wide(x, dtype)
    want = Probs(x64, None if targets is None else targets.astype(np.int64), float(np.float32(scale)), ignore, lanes)
    assert (got[0] is None) == (targets is None) and (got[1] is None) == (not entropy)
    assert (got[3] is None) == (got[4] is None) == (top == 0)
    if targets is not None:
        lp, bound = want.given()
        assert_within(got[0].numpy(), lp, bound, F32, "logprob")
    if entropy:
        assert_within(got[1].numpy(), want.h, np.nan_to_num(np.where(want.skipped, 0, want.h_bound)), F32, "entropy")
    stats = got[2].numpy()
    assert np.array_equal(stats[:, 0], want.m.astype(np.float32), equal_nan=True)
    fine = np.isfinite(want.ls)
    assert_within(stats[fine, 1], want.ls[fine], np.where(want.skipped, 0, want.ls_bound)[fine], F32, "sum")
    if top:
        order, values, bound = want.top(top)
        assert np.array_equal(got[4].numpy(), order)
        assert_within(got[3].numpy(), values, bound, F32, "alternatives")
    if back:
        rng = np.random.default_rng(17)
        da, db = (rng.standard_normal(len(x)).astype(np.float32) for _ in range(2))
        for a, b in ((da, None), (None, db), (da, db)):
            if (a is not None and targets is None) or (b is not None and not entropy):
                continue
            dx = ops.token_log_probs_backward(None if a is None else put(a), None if b is None else put(b), logits, t, got[2], got[1], scale,
                                              ignore)
            d, bound = want.backward(a, b)
            assert dx.shape == x.shape and dx.is_contiguous()
            assert_within(dx.numpy(), d, bound, dtype, "gradient")
    return got


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 65, 1000, 2047, 2048, 2049, 4099, 8192, 8200, 20011, 50001])
def test_log_probs_sizes(dev, ops, dtype, vocab):
    x = rows_of_logits(3, vocab, dtype, vocab)
    rng = np.random.default_rng(vocab)
    check_probs(ops, dtype, x, rng.integers(0, vocab, 3), top=min(vocab, 5))
    check_probs(ops, dtype, x, rng.integers(0, vocab, 3).astype(np.int32), scale=0.7, top=0)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,vocab", [(1, 32000), (1, 128003), (2, 512), (600, 3001), (1500, 64), (33, 9000), (257, 20000)])
def test_log_probs_rows(dev, ops, dtype, rows, vocab):
    """Rows split over many blocks, a block a row, and between."""
    x = rows_of_logits(rows, vocab, dtype, rows)
    t = np.random.default_rng(rows).integers(0, vocab, rows)
    check_probs(ops, dtype, x, t, scale=1.3, top=20, back=rows * vocab < 2e6)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("top", [1, 2, 3, 4, 5, 31, 63, 64])
def test_alternatives(dev, ops, dtype, top):
    for rows, vocab in ((2, 64), (4, 3000), (700, 9001)):
        x = rows_of_logits(rows, vocab, dtype, top)
        check_probs(ops, dtype, x, None, top=top, back=False, entropy=False)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,vocab", [(2, 50), (3, 5000), (2, 40000), (700, 20000)])
def test_alternatives_of_equal_and_ordered_logits(dev, ops, dtype, rows, vocab):
    """Equal logits, few different ones, rising and falling rows, a few allowed
    tokens: the lowest indices first, whatever the order of the row."""
    rng = np.random.default_rng(5)
    step = np.arange(vocab) * (40.0 / vocab) - 20.0
    few = np.full(vocab, -np.inf)
    few[rng.permutation(vocab)[:7]] = rng.standard_normal(7)
    last = np.zeros(vocab)
    last[-9:] = np.arange(9)
    for row in (np.zeros(vocab), rng.integers(0, 3, vocab) - 1.0, step, -step, few, last, np.where(np.arange(vocab) % 2, 0.0, -0.0),
                np.where(np.arange(vocab) < 10, -np.inf, 1.0)):
        x = bits(np.broadcast_to(row, (rows, vocab)), dtype)
        check_probs(ops, dtype, np.ascontiguousarray(x), np.full(rows, vocab - 1), top=20, back=False)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("top", [1, 4, 16, 17, 64])
@pytest.mark.parametrize("rows,vocab", [(2, 700), (3, 5000), (2, 40000), (700, 20000)])
def test_alternatives_of_rising_and_equal_logits(dev, ops, dtype, rows, vocab, top):
    rng = np.random.default_rng(15)
    step = np.arange(vocab) * (40.0 / vocab) - 20.0
    for row in (np.zeros(vocab), step, -step, rng.integers(0, 3, vocab) - 1.0, np.where(np.arange(vocab) % 64 == 63, step, -20.0),
                np.where(np.arange(vocab) < 10, 1.0, -np.inf), np.where(rng.random(vocab) < 0.01, np.nan, step)):
        x = bits(np.broadcast_to(row, (rows, vocab)), dtype)
        check_probs(ops, dtype, np.ascontiguousarray(x), np.full(rows, vocab - 1), top=top, back=False)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("top", [1, 5, 17])
def test_alternatives_of_many_long_rows(dev, ops, dtype, top):
    """Rows enough for a wave each."""
    rows, vocab = 4099, 9001 if dtype == F32 else 17001
    x = rows_of_logits(64, vocab, dtype, top)
    x = np.ascontiguousarray(np.concatenate([x] * 65)[:rows])  # (only 64 of them differ)
    x[7, 100:] = bits([-np.inf], dtype)[0]
    x[4098] = x[4098][::-1]
    t = np.random.default_rng(top).integers(0, vocab, rows)
    check_probs(ops, dtype, x, t, top=top, back=False, lanes=64)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,vocab", [(1, 300), (9, 300), (9, 12000), (1100, 2500)])
def test_log_probs_of_what_is_not_finite(dev, ops, dtype, rows, vocab):
    """Masked tokens, the type's lowest value, NaN, +inf, rows with nothing
    left; each by itself."""
    x = wide(rows_of_logits(rows, vocab, dtype, 3), dtype)
    low = {F32: -3.4028234663852886e38, F16: -65504.0, BF16: -3.3895313892515355e38}[dtype]
    t = np.random.default_rng(6).integers(0, vocab, rows)
    cases = [lambda r: None, lambda r: r.__setitem__(slice(1, None, 2), -np.inf), lambda r: r.__setitem__(slice(0, -1), low),
             lambda r: r.__setitem__(slice(None), low), lambda r: r.__setitem__(slice(None), -np.inf), lambda r: r.__setitem__(vocab // 2, np.nan),
             lambda r: r.__setitem__(slice(0, vocab, 37), np.nan), lambda r: r.__setitem__(vocab - 1, np.inf), lambda r: r.__setitem__(0, -np.inf)]
    for first in range(0, len(cases), rows):
        for i, change in enumerate(cases[first: first + rows]):
            change(x[i])
        host = orc.from_float(x.astype(np.float32), dtype)
        check_probs(ops, dtype, host, t, top=5)
        check_probs(ops, dtype, host, t, scale=0.5)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,vocab", [(8, 100), (8, 30000), (1000, 700)])
def test_skipped_and_unknown_targets(dev, ops, dtype, rows, vocab):
    """A skipped row is not read (NaN in it changes nothing), a target outside
    the vocabulary reads nothing and gives NaN."""
    x = wide(rows_of_logits(rows, vocab, dtype, 8), dtype)
    t = np.random.default_rng(9).integers(0, vocab, rows)
    t[1], t[2], t[3], t[4], t[5] = -100, vocab, -1, 1 << 40, -(1 << 62)
    x[1] = np.nan
    host = orc.from_float(x.astype(np.float32), dtype)
    got = check_probs(ops, dtype, host, t, top=3)
    assert got[0].numpy()[1] == 0 and got[1].numpy()[1] == 0 and (got[4].numpy()[1] == -1).all()
    assert np.isnan(got[0].numpy()[2:6]).all()
    t[:] = 7
    x[1] = 0
    check_probs(ops, dtype, orc.from_float(x.astype(np.float32), dtype), t, ignore=7)  # every row
    check_probs(ops, dtype, orc.from_float(x.astype(np.float32), dtype), t, ignore=8)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("vocab", [1, 7, 65, 1001, 2049])
def test_log_probs_of_many_short_rows(dev, ops, dtype, vocab):
    """Rows enough for a wave each, the last block's not all there; some skipped,
    some of unknown targets, some with masked tokens, NaN or nothing left."""
    rows = 4099
    x = wide(rows_of_logits(rows, vocab, dtype, vocab + 1), dtype)
    t = np.random.default_rng(vocab).integers(0, vocab, rows)
    t[3::50], t[4098], t[7::300], t[8::300] = -100, -100, vocab, -(1 << 40)
    x[9::90, ::2] = -np.inf
    x[11::200, vocab // 2], x[13::200], x[15::200, vocab - 1] = np.nan, -np.inf, np.inf
    host = orc.from_float(x.astype(np.float32), dtype)
    check_probs(ops, dtype, host, t, lanes=64)
    check_probs(ops, dtype, host, t.astype(np.int32) if vocab == 7 else t, scale=0.7, entropy=False, back=vocab < 100, lanes=64)
    check_probs(ops, dtype, host, t, top=min(3, vocab), back=False, lanes=64)
    check_probs(ops, dtype, host, None, back=False, lanes=64)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("vocab", [200, 4001])
def test_log_probs_of_views(dev, ops, dtype, vocab):
    """The last token of every sequence, rows that start at any element, a
    transposed matrix, several row axes; targets as a view."""
    b, t = 5, 3
    big = sample((b, t, vocab + 3), dtype, 21, 2.0)
    d = put(big, dtype)
    targets = np.random.default_rng(1).integers(0, vocab, b)
    check_probs(ops, dtype, np.ascontiguousarray(big[:, -1, 1: vocab + 1]), targets, top=4, view=d[:, -1, 1: vocab + 1])
    turned = sample((vocab, b), dtype, 22, 2.0)
    check_probs(ops, dtype, np.ascontiguousarray(turned.T), targets, top=4, view=put(turned, dtype).t())
    x = sample((2, 3, 4, vocab), dtype, 23, 2.0)
    wide_t = np.random.default_rng(2).integers(0, vocab, (2, 3, 8))
    got = ops.token_log_probs(put(x, dtype), put(wide_t)[:, :, ::2], top=2)
    assert [g.shape for g in got] == [(2, 3, 4), (2, 3, 4), (2, 3, 4, 2), (2, 3, 4, 2), (2, 3, 4, 2)]
    want = Probs(wide(x, dtype).reshape(24, vocab), wide_t[:, :, ::2].reshape(24))
    lp, bound = want.given()
    assert_within(got[0].numpy().reshape(24), lp, bound, F32)
    assert np.array_equal(got[4].numpy().reshape(24, 2), want.top(2)[0])
    # one row without a row axis
    one = ops.token_log_probs(put(x[0, 0, 0], dtype), put(wide_t[0, 0, :1])[0], top=1)
    assert one[0].shape == () and one[4].shape == (1,)
    assert_within(one[0].numpy().reshape(1), lp[:1], bound[:1], F32)


def test_log_probs_of_no_rows(dev, ops):
    got = ops.token_log_probs(put(np.zeros((0, 9), np.float32)), put(np.zeros(0, np.int64)), top=3)
    assert [g.shape for g in got] == [(0,), (0,), (0, 2), (0, 3), (0, 3)]
    dx = ops.token_log_probs_backward(put(np.zeros(0, np.float32)), None, put(np.zeros((0, 9), np.float32)), put(np.zeros(0, np.int64)), got[2])
    assert dx.shape == (0, 9)


@pytest.mark.parametrize("rows,vocab", [(4, 20000), (900, 5000)])
def test_log_probs_agree_with_the_library(dev, ops, rows, vocab):
    """log_softmax and nll_loss give the same."""
    x = rows_of_logits(rows, vocab, F32, 30)
    t = np.random.default_rng(31).integers(0, vocab, rows)
    lp = ops.token_log_probs(put(x), put(t))[0].numpy()
    other, _ = ops.nll_loss(ops.log_softmax(put(x), -1), put(t), reduction=0)
    p = Probs(x.astype(np.float64), t)
    # both are within this of the definition
    assert (np.abs(lp + other.numpy()) <= 2 * p.given()[1] + 2 * U * np.abs(lp)).all()


# ---- together ---------------------------------------------------------------------------


def test_recorded_and_replayed(dev, ops):
    """A run of all of them in a recording, replayed on new inputs and a new
    seed between eager calls: the eager bits each time."""
    graph, runtime = mod("graph"), mod("runtime")
    shape, dim, vocab = (2, 65, 264), 264, 4001
    x, y, gate = (put(sample(s, BF16, i), BF16) for i, s in ((1, shape), (2, shape), (3, (2, 1, dim))))
    w, head = put(sample((dim,), BF16, 4, 0.2, 1.0), BF16), put(sample((vocab, dim), BF16, 5, 0.1), BF16)
    t = put(np.random.default_rng(6).integers(0, vocab, shape[:2]))
    da, db = (put(sample(shape[:2], F32, i)) for i in (7, 8))
    dz, seed = put(sample(shape, BF16, 9), BF16), put(np.array([77], np.int64))

    def step():
        x1 = ops.seeded_dropout(x, 0.1, seed)
        z, h, r1, r2 = ops.residual_norm(x1, y, gate, w, w, 1.0, 0.5, 1e-6, 1e-6, 0.2, seed, 1)
        logits = ops.linear(h, head)
        lp, entropy, stats, values, indices = ops.token_log_probs(logits, t, 0.8, 7)
        dlogits = ops.token_log_probs_backward(da, db, logits, t, stats, entropy, 0.8)
        dh = ops.matmul(dlogits, head)
        grads = ops.residual_norm_backward(dz, dh, x1, y, r1, r2, gate, w, w, 1.0, 0.5, 0.2, seed, 1)
        return [z, lp, entropy, values, indices, *grads, ops.seeded_dropout_backward(grads[0], 0.1, seed)]

    g = graph.Graph()
    try:
        results = g.capture(step)
        seen = []
        for i in range(4):
            ops.copy_(x, sample(shape, F32, 100 + i))
            ops.copy_(seed, np.array([1000 * i + 5], np.int64))
            g.replay()
            runtime.synchronize()
            for a, b in zip(results, step()):
                assert np.array_equal(a.numpy(), b.numpy())
            seen.append(results[-1].numpy())
        assert not np.array_equal(seen[0] == 0, seen[1] == 0)
    finally:
        g.reset()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_entropy_of_a_sure_row(dev, ops, dtype):
    """Never below 0, whatever rounding makes of a row with one likely token."""
    x = sample((64, 3001), dtype, 50)
    x[np.arange(64), np.arange(64) * 7] = bits(np.linspace(10, 60, 64), dtype)
    h = ops.token_log_probs(put(x, dtype))[1].numpy()
    want = Probs(wide(x, dtype))
    assert (h >= 0).all()
    assert_within(h, want.h, want.h_bound, F32)


@pytest.mark.parametrize("shape", [(2, 0, 3), (0, 2), (2, 3, 0)], ids=str)
def test_token_axes_without_a_token(dev, ops, shape):
    """An axis of no tokens anywhere among the others."""
    x = put(np.zeros((*shape, 16), np.float32))
    z, h, _, r = ops.residual_norm(x, x)
    assert z.shape == h.shape == (*shape, 16) and r.shape == shape
    got = ops.token_log_probs(x, put(np.zeros(shape, np.int64)))
    assert got[0].shape == shape and got[2].shape == (*shape, 2)
    q = put(np.zeros((*shape, 4, 16), np.float32))
    table = put(np.ones((5, 16), np.float32))
    out = ops.qk_norm_rope(q, q, table, put(np.zeros(shape[-1:], np.int64)))
    assert out[0].shape == (*shape, 4, 16) and out[2].shape == (*shape, 4)
