"""Where the attention layer's operators meet what is not finite, not small or
not large: each case against float64 or against the same call without it.

Bounds are those of ``_attention.Attention``; where a test needs a closer one
it is derived beside the test.
"""

import numpy as np
import pytest

from _attention import BF16, F16, F32, FLUSH, HALF, TINY, U, Attention, assert_within, mod, put, sample, wide
from oracle import binding as orc

pytestmark = pytest.mark.gpu

DTYPES = [F32, F16, BF16]
IDS = ["fp32", "fp16", "bf16"]


def make(dtype, b, tq, tk, h, hk, d, seed=0):
    return [sample(s, dtype, seed + i) for i, s in enumerate(((b, tq, h, d), (b, tk, hk, d), (b, tk, hk, d), (b, tq, h, d)))]


def one(value, dtype):
    return orc.from_float(np.array([value], np.float32), dtype)[0]


# ---- NaN among the scores -------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("tq", [1, 5, 70, 400])
def test_a_query_that_is_nan(dev, ops, dtype, tq):
    """Its own row is NaN, whichever kernel takes it; the others are as ever."""
    host = make(dtype, 2, tq, 400, 4, 2, 64, 10)
    a = Attention(dtype, *[wide(x, dtype) for x in host[:3]])
    host[0][1, tq // 2, 2] = one(np.nan, dtype)
    out, lse = ops.sliding_window_attention(*[put(x, dtype) for x in host[:3]])
    o, l = wide(out.numpy(), dtype), lse.numpy()
    assert np.isnan(o[1, tq // 2, 2]).all() and np.isnan(l[1, 2, tq // 2])
    want, bound = a.tokens(a.out).copy(), a.tokens(a.out_bound).copy()
    want[1, tq // 2, 2], bound[1, tq // 2, 2] = np.nan, 0.0
    assert_within(out.numpy(), want, bound, dtype, "out")
    a.lse[1, 2, tq // 2] = np.nan
    assert_within(l, a.lse, np.nan_to_num(a.lse_bound), F32, "lse")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("tk,first,count", [(33, 32, 1), (2, 1, 1), (1, 0, 1), (64, 32, 32), (5000, 3200, 1000), (5000, 4999, 1), (5000, 0, 5000)])
@pytest.mark.parametrize("tq", [1, 40])
def test_keys_that_are_nan(dev, ops, dtype, tq, tk, first, count):
    """Every query that sees one is NaN, also where a wave or a split meets no
    other key; queries before the first of them are as ever."""
    host = make(dtype, 2, tq, tk, 4, 2, 64, 20)
    a = Attention(dtype, *[wide(x, dtype) for x in host[:3]])
    host[1][0, first:first + count, 1] = one(np.nan, dtype)
    out, lse = ops.sliding_window_attention(*[put(x, dtype) for x in host[:3]])
    struck = np.zeros((2, tq, 4), bool)
    struck[0, :, 2:] = (tk - tq + np.arange(tq) >= first)[:, None]
    want = np.where(struck[..., None], np.nan, a.tokens(a.out))
    assert_within(out.numpy(), want, a.tokens(a.out_bound), dtype, "out")
    struck = struck.transpose(0, 2, 1)
    assert_within(lse.numpy(), np.where(struck, np.nan, a.lse), a.lse_bound, F32, "lse")


# ---- gradients of every size in float16 -----------------------------------------


def close_bounds(a, do, dtype):
    """The backward's results and bounds of an ``Attention`` whose dS and P are
    scaled by powers of two before they are rounded to 16 bits: of dS in a sum
    the largest so far lies at 2^7 or above, so that an element is off by half a
    step, relative, and by 2^-25, half of float16's smallest step, over 2^7 of
    the sum's largest; P is scaled by 2^12."""
    want, bounds = a.backward(do, dtype)
    if dtype != F16:
        return want, bounds
    do = np.where(~a.see.any(-1)[..., None], 0.0, do.transpose(0, 2, 1, 3))
    dp = do @ a.v.swapaxes(-1, -2)
    ds = np.abs(a.p * (dp - (do * a.out).sum(-1, keepdims=True)))
    see = np.broadcast_to(a.see, a.p.shape)
    t, k, q = TINY[F16], np.abs(a.k), np.abs(a.q)
    row = ds.max(-1, keepdims=True) * 2.0 ** -7 - 1.0
    # a key's sum runs over all query heads that share it
    b, h, tq, tk = ds.shape
    column = np.repeat(ds.reshape(b, h // a.group, -1, tk).max(2), a.group, 1)[:, :, None] * 2.0 ** -7 - 1.0
    more = (a.tokens(a.scale * t * (row * see) @ k), a.shared(a.scale * t * (column * see).swapaxes(-1, -2) @ q),
            a.shared(t * (2.0 ** -12 - 1.0) * see.swapaxes(-1, -2) @ np.abs(do)))
    return want, tuple(x + y for x, y in zip(bounds, more))


@pytest.mark.parametrize("shape", [(1, 512, 512, 2, 1, 128), (1, 200, 200, 256, 256, 64), (1, 130, 700, 64, 32, 96), (1, 300, 300, 6, 2, 32)], ids=str)
@pytest.mark.parametrize("size", [1e-5, 1e-4, 1e-3, 1.0, 300.0, 8000.0])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS[1:])
def test_gradients_of_every_size(dev, ops, dtype, size, shape):
    """dS as large as the gradients passes float16's range, and as small falls
    among its subnormals: neither shows in dq, dk or dv."""
    host = make(dtype, *shape, 30)
    # (large ones beside small queries and keys, so that the results stay in range)
    for i, by in enumerate((0.25, 0.25, 2.0, size) if size > 1000 else (1.0, 1.0, 1.0, size)):
        host[i] = orc.from_float((wide(host[i], dtype) * by).astype(np.float32), dtype)
    w = [wide(x, dtype) for x in host]
    a = Attention(dtype, *w[:3], window=250, sinks=2)
    want, bounds = close_bounds(a, w[3], dtype)
    assert all(np.abs(x).max() < 6e4 for x in want), "the results themselves have to be in range"
    q, k, v, do = (put(x, dtype) for x in host)
    out, lse = ops.sliding_window_attention(q, k, v, 250, 2)
    for g, x, bound, name in zip(ops.sliding_window_attention_backward(do, q, k, v, out, lse, 250, 2), want, bounds, ("dq", "dk", "dv")):
        assert_within(g.numpy(), x, bound, dtype, name)


@pytest.mark.parametrize("down", [False, True], ids=["growing", "shrinking"])
@pytest.mark.parametrize("shape", [(1, 400, 400, 2, 1, 64), (1, 200, 200, 256, 256, 64)], ids=str)
def test_gradients_that_change_size_along_a_sum(dev, ops, shape, down):
    """Values grow by 2^20 along the keys and the gradients along the queries:
    the scale of a sum's dS is left again and again."""
    host = make(F16, *shape, 40)
    for i in (2, 3):
        grow = 2.0 ** np.linspace(-14 + 2 * i, 2 + 2 * i, host[i].shape[1])[:: -1 if down else 1]
        host[i] = orc.from_float((wide(host[i], F16) * grow[:, None, None]).astype(np.float32), F16)
    w = [wide(x, F16) for x in host]
    a = Attention(F16, *w[:3])
    want, bounds = close_bounds(a, w[3], F16)
    assert all(np.abs(x).max() < 6e4 for x in want), "the results themselves have to be in range"
    q, k, v, do = (put(x, F16) for x in host)
    out, lse = ops.sliding_window_attention(q, k, v)
    for g, x, bound, name in zip(ops.sliding_window_attention_backward(do, q, k, v, out, lse), want, bounds, ("dq", "dk", "dv")):
        assert_within(g.numpy(), x, bound, F16, name)


def test_dv_of_small_probabilities(dev, ops):
    """302292 keys of one score: each probability lies midway between two of
    float16's subnormals.  With keys of zero every sum of exponentials is a
    whole number under 2^24 and exact; l = ln n is off by 2 u of itself, its
    product with log2 e by 2 u more and the power by 4 u: under 2^-18 of P
    together.  A sum of 8 heads' and queries' terms adds 2^-20."""
    tk, tq, heads, kv, d = 302292, 4, 2, 1, 8
    q, k, v, do = make(F16, 1, tq, tk, heads, kv, d, 50)
    k[:] = 0
    do = orc.from_float(np.sign(wide(do, F16)).astype(np.float32) * 512 + np.abs(wide(do, F16)).astype(np.float32), F16)
    dq_, dk_, dv_, ddo = (put(x, F16) for x in (q, k, v, do))
    out, lse = ops.sliding_window_attention(dq_, dk_, dv_)
    dv = ops.sliding_window_attention_backward(ddo, dq_, dk_, dv_, out, lse)[2].numpy()
    n = tk - tq + 1 + np.arange(tq)
    terms = (wide(do, F16)[0] / n[:, None, None]).reshape(tq, kv, heads // kv, d).sum(2)
    want = np.cumsum(terms[::-1], 0)[::-1]  # key tk - tq + i: by queries i and on
    want = np.concatenate([np.broadcast_to(want[:1], (tk - tq + 1, kv, d)), want[1:]])
    size = np.abs(wide(do, F16)[0] / n[:, None, None]).reshape(tq, kv, heads // kv, d).sum((0, 2))
    assert_within(dv[0], want, (HALF[F16] + 2.0 ** -17) * size, F16, "dv")


# ---- rows without a sum -----------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("tq,heads,kv", [(1, 1, 1), (200, 1, 1), (200, 128, 64)])
def test_rows_whose_scores_are_minus_infinity(dev, ops, dtype, tq, heads, kv):
    """Sequence 0's keys give every score -inf: zeros, an l of -inf and
    gradients of zero, and sequence 1 is as ever."""
    host = make(dtype, 2, tq, 200, heads, kv, 16, 60)
    host[0][:, :, :, 3] = one(1.0, dtype)
    w = [wide(x, dtype) for x in host]
    a = Attention(dtype, *w[:3])
    want, bounds = a.backward(w[3], dtype)
    host[1][0, :, :, 3] = one(-np.inf, dtype)
    q, k, v, do = (put(x, dtype) for x in host)
    out, lse = ops.sliding_window_attention(q, k, v)
    grads = ops.sliding_window_attention_backward(do, q, k, v, out, lse)
    assert (wide(out.numpy(), dtype)[0] == 0).all() and (lse.numpy()[0] == -np.inf).all()
    for g, x, bound, name in zip(grads, want, bounds, ("dq", "dk", "dv")):
        x, bound = x.copy(), bound.copy()
        x[0] = bound[0] = 0.0
        assert_within(g.numpy(), x, bound, dtype, name)
        assert (wide(g.numpy(), dtype)[0] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("heads,kv", [(1, 1), (256, 128)])
@pytest.mark.parametrize("where", ["query", "gradient", "out"])
def test_rows_given_as_without_a_sum(dev, ops, dtype, heads, kv, where):
    """A query whose l is handed in as -inf has no gradient and takes no part
    in the keys', whatever it, its result and its gradient hold."""
    host = make(dtype, 1, 150, 150, heads, kv, 32, 65)
    q, k, v, do = (put(x, dtype) for x in host)
    out, lse = ops.sliding_window_attention(q, k, v, 60, 1)
    o, l = out.numpy().copy(), lse.numpy().copy()
    without = [0, 70, 71, 149]
    l[:, :, without] = -np.inf
    clean = [x.numpy() for x in ops.sliding_window_attention_backward(do, q, k, v, put(o, dtype), put(l), 60, 1)]
    for x in clean:
        assert np.isfinite(wide(x, dtype)).all()
    assert (wide(clean[0], dtype)[:, without] == 0).all()
    struck = {"query": host[0], "gradient": host[3], "out": o}[where]
    struck[:, without] = one(np.inf, dtype)
    struck[:, without[1]] = one(np.nan, dtype)
    q, do = put(host[0], dtype), put(host[3], dtype)
    for x, y in zip(ops.sliding_window_attention_backward(do, q, k, v, put(o, dtype), put(l), 60, 1), clean):
        # the rows' part is summed in another order where it is left out
        assert_within(x.numpy(), wide(y, dtype), 2.0 ** -7 * np.abs(wide(y, dtype)).max(), dtype)


# ---- memory of the parts ------------------------------------------------------------


def test_sums_of_few_first_tokens_beside_many_keys(dev, ops):
    """Only the first tokens' walks are cut: the keys behind them write their
    gradients themselves and have no room among the parts."""
    runtime = mod("runtime")
    t, h, d, window, sinks = 16384, 8, 64, 256, 4
    q, k, v, do = (put(x, BF16) for x in make(BF16, 1, t, t, h, h, d, 70))
    out, lse = ops.sliding_window_attention(q, k, v, window, sinks)
    runtime.synchronize()
    runtime.reset_peak_memory_stats()
    before = runtime.memory_allocated()
    grads = ops.sliding_window_attention_backward(do, q, k, v, out, lse, window, sinks)
    runtime.synchronize()
    # a block of 128 keys walks 64 queries a step: the first block all of
    # them, in parts no shorter than the others' walk of at least 6 steps
    parts = h * (t // 64 // 6 + 1)
    bound = parts * 2 * 128 * d * 4 + 3 * t * h * d * 2 + 2 * t * h * 4
    assert runtime.max_memory_allocated() - before <= 1.1 * bound
    # head 3 against float64, a run of keys at either end
    w = [wide(x.numpy(), BF16)[:, :, 3:4] for x in (q, k, v, do)]
    n = 700
    for cut in (slice(0, n), slice(t - n, t)):
        if cut.start == 0:
            continue
        low = t - n - window
        part = [np.concatenate([x[:, :sinks], x[:, low:]], 1) for x in w[1:3]]
        a = Attention(BF16, w[0][:, low + window:], *part, window=window, sinks=sinks)
        want, bounds = a.backward(w[3][:, low + window:], BF16)
        assert_within(grads[0].numpy()[:, t - n:, 3:4], want[0], bounds[0], BF16, "dq")
        for i, name in ((1, "dk"), (2, "dv")):
            last = n - window  # keys whose queries are all among these
            assert_within(grads[i].numpy()[:, t - last:, 3:4], want[i][:, -last:], bounds[i][:, -last:], BF16, name)


@pytest.mark.parametrize("heads,sinks,window", [(256, 2048, 600), (8, 300, 900), (40, 130, 40)])
def test_which_walks_are_cut(dev, ops, heads, sinks, window):
    """The first tokens' walks, the others', both: the heads are all one, and
    each has the gradients that float64 gives it."""
    t, d = 2176, 8
    host = make(F32, 1, t, t, 1, 1, d, 75)
    w = [wide(x, F32) for x in host]
    a = Attention(F32, *w[:3], window=window, sinks=sinks)
    want, bounds = a.backward(w[3], F32)
    q, k, v, do = (put(x).expand(1, t, heads, d) for x in host)
    out, lse = ops.sliding_window_attention(q, k, v, window, sinks)
    for g, x, bound, name in zip(ops.sliding_window_attention_backward(do, q, k, v, out, lse, window, sinks), want, bounds, ("dq", "dk", "dv")):
        g = g.numpy()
        assert (g == g[:, :, :1]).all(), name
        assert_within(g[:, :, :1], x, bound, F32, name)


# ---- D of rows that see few keys ------------------------------------------------------


@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS[1:])
@pytest.mark.parametrize("shape,rule", [
    ((1, 500, 500, 2, 1, 64), dict(window=16)),
    ((1, 500, 500, 2, 2, 128), dict(window=100, sinks=28)),
    ((2, 300, 300, 32, 16, 32), dict(window=33, sinks=3)),
    ((1, 500, 500, 2, 1, 64), dict(window=0, sinks=128)),
    ((1, 128, 128, 3, 3, 64), dict()),
    ((1, 100, 160, 2, 1, 64), dict()),
    ((1, 90, 190, 2, 2, 128), dict(sinks=3, window=170)),
], ids=str)
def test_gradients_of_rows_that_see_few_keys(dev, ops, dtype, shape, rule):
    """Values far from zero: D = do . out with out rounded to 16 bits is off by
    more than what dP - D leaves of it.  Rows of at most 128 keys, and those in a
    block with one, have it as the sum of P dP, off by eps of P and by dP's own
    error: the bound here has no rounding of out in it.  (The closer bound of dP - D takes half a step of the
    difference, not of its two parts.)"""
    host = make(dtype, *shape, 80)
    host[2] = orc.from_float((wide(host[2], dtype) + 50.0).astype(np.float32), dtype)
    w = [wide(x, dtype) for x in host]
    a = Attention(dtype, *w[:3], **rule)
    want, _ = a.backward(w[3], dtype)
    do = w[3].transpose(0, 2, 1, 3)
    d, n = do.shape[-1], a.see.sum(-1, keepdims=True)
    assert n.min() <= 128 and (n.max() <= 128 or shape[1] <= 128)
    eps = a.eps + a.lse_bound[..., None] + n * U
    dp = do @ a.v.swapaxes(-1, -2)
    e_dp = (d + 8) * U * (np.abs(do) @ np.abs(a.v).swapaxes(-1, -2))
    delta = (a.p * dp).sum(-1, keepdims=True)
    e_delta = (a.p * (np.abs(dp) * (2 * eps + n * U) + e_dp)).sum(-1, keepdims=True)
    off = a.p * (np.abs(dp - delta) * (a.h + 2 * eps) + e_dp + e_delta) * (1 + a.h)
    off = off + FLUSH * a.see * (1 + np.abs(dp) + np.abs(delta))
    if dtype == F16:  # half of the smallest step, at a scale that leaves the sum's largest at 2^7 or above
        ds = np.abs(a.p * (dp - delta))
        b, h, tq, tk = ds.shape
        column = np.repeat(ds.reshape(b, h // a.group, -1, tk).max(2), a.group, 1)[:, :, None]
        off = off + TINY[F16] * 2.0 ** -7 * a.see * np.maximum(ds.max(-1, keepdims=True), column)
    # the sums over a row's keys, and over the queries and heads a key has
    sums = (2 * n.max() * a.group + 400) * U
    bq = a.scale * ((off + sums * np.abs(a.p * (dp - delta))) @ np.abs(a.k))
    bk = a.scale * ((off + sums * np.abs(a.p * (dp - delta))).swapaxes(-1, -2) @ np.abs(a.q))
    q, k, v, g = (put(x, dtype) for x in host)
    out, lse = ops.sliding_window_attention(q, k, v, **rule)
    dq, dk, _ = ops.sliding_window_attention_backward(g, q, k, v, out, lse, **rule)
    assert_within(dq.numpy(), want[0], a.tokens(bq), dtype, "dq")
    assert_within(dk.numpy(), want[1], a.shared(bk), dtype, "dk")


# ---- what is not finite stays with those that see it ------------------------------------


CROSS = [((1, 200, 200, 2, 1, 64), dict(window=40, sinks=3), 150),
         ((2, 40, 90, 4, 2, 32), dict(), 70),
         ((1, 300, 300, 3, 3, 128), dict(window=33), 100),
         ((1, 6, 500, 8, 2, 96), dict(window=100, sinks=2), 496),
         ((2, 200, 200, 128, 64, 40), dict(window=70, sinks=1), 130)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("what", ["key", "value"])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf], ids=["nan", "inf", "-inf"])
@pytest.mark.parametrize("shape,rule,at", CROSS, ids=str)
def test_keys_and_values_reach_their_queries_only(dev, ops, dtype, what, value, shape, rule, at):
    """Key ``at`` of key head 0 or its value is not finite: queries that do not
    see it, and keys that none of its queries sees, are as without it."""
    host = make(dtype, *shape, 90)
    w = [wide(x, dtype) for x in host]
    a = Attention(dtype, *w[:3], **rule)
    want, bounds = a.backward(w[3], dtype)
    group = shape[3] // shape[4]
    struck = host[1 if what == "key" else 2]
    struck[0, at, 0, 5] = one(value, dtype)
    q, k, v, do = (put(x, dtype) for x in host)
    out, lse = ops.sliding_window_attention(q, k, v, **rule)
    grads = ops.sliding_window_attention_backward(do, q, k, v, out, lse, **rule)
    rows = np.zeros(a.lse.shape, bool)  # [B, H, Tq]: those that see it
    rows[0, :group] = a.see[0, 0][:, at]
    assert rows.any() and not rows.all()
    keys = np.zeros((shape[0], shape[4], shape[2]), bool)  # seen by one of those
    keys[0, 0] = a.see[0, 0][rows[0, 0]].any(0)
    r, c = rows.transpose(0, 2, 1)[..., None], keys.transpose(0, 2, 1)[..., None]
    o = wide(out.numpy(), dtype)
    if what == "value":
        assert not np.isfinite(o[0, rows[0, 0], 0, 5]).any()
        fine = r & (np.arange(shape[5]) != 5)
        assert np.isfinite(o[np.broadcast_to(fine, o.shape)]).all()
    elif value != value:
        assert np.isnan(o[np.broadcast_to(r, o.shape)]).all()

    def clean(x, x64, bound, mask, name):
        x = wide(x, dtype if x.ndim == 4 else F32)
        mask = np.broadcast_to(mask, x.shape)
        kept = np.where(mask, 0.0, x)
        store = orc.from_float(kept.astype(np.float32), dtype) if x.ndim == 4 else kept.astype(np.float32)
        assert_within(store, np.where(mask, 0.0, x64), np.where(mask, 0.0, bound), dtype if x.ndim == 4 else F32, name)

    clean(out.numpy(), a.tokens(a.out), a.tokens(a.out_bound), r, "out")
    clean(lse.numpy(), a.lse, a.lse_bound, rows, "lse")
    for g, x, bound, m, name in zip(grads, want, bounds, (r, c, c), ("dq", "dk", "dv")):
        clean(g.numpy(), x, bound, m, name)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("what", ["query", "gradient"])
@pytest.mark.parametrize("value", [np.nan, np.inf], ids=["nan", "inf"])
@pytest.mark.parametrize("shape,rule,at", CROSS, ids=str)
def test_queries_and_gradients_reach_their_keys_only(dev, ops, dtype, what, value, shape, rule, at):
    """One query of head 0 or its gradient is not finite: keys that it does not
    see are as without it, and so is every other query."""
    host = make(dtype, *shape, 95)
    w = [wide(x, dtype) for x in host]
    a = Attention(dtype, *w[:3], **rule)
    want, bounds = a.backward(w[3], dtype)
    i = shape[1] // 2
    struck = host[0 if what == "query" else 3]
    struck[0, i, 0, 5] = one(value, dtype)
    q, k, v, do = (put(x, dtype) for x in host)
    out, lse = ops.sliding_window_attention(q, k, v, **rule)
    grads = ops.sliding_window_attention_backward(do, q, k, v, out, lse, **rule)
    seen = a.see[0, 0, i]
    for g, x, bound, name in zip(grads, want, bounds, ("dq", "dk", "dv")):
        g64, x, bound = wide(g.numpy(), dtype), x.copy(), bound.copy()
        at_ = (0, i, 0) if name == "dq" else (0, seen, 0)
        g64[at_] = x[at_] = bound[at_] = 0.0
        assert_within(orc.from_float(g64.astype(np.float32), dtype), x, bound, dtype, name)
    dv = wide(grads[2].numpy(), dtype)[0, seen, 0]
    assert not np.isfinite(dv[:, 5]).any()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("tq,heads", [(3, 2), (200, 2), (200, 256)])
def test_keys_that_no_query_sees(dev, ops, dtype, tq, heads):
    """A window of none leaves the first tokens alone: NaN in every other key
    and value reaches nothing, and their own gradients are zeros."""
    host = make(dtype, 1, tq, 200, heads, heads, 32, 99)
    w = [wide(x, dtype) for x in host]
    a = Attention(dtype, *w[:3], window=0, sinks=4)
    want, bounds = a.backward(w[3], dtype)
    for x in host[1:3]:
        x[:, 4:] = one(np.nan, dtype)
    q, k, v, do = (put(x, dtype) for x in host)
    out, lse = ops.sliding_window_attention(q, k, v, 0, 4)
    assert_within(out.numpy(), a.tokens(a.out), a.tokens(a.out_bound), dtype, "out")
    for g, x, bound, name in zip(ops.sliding_window_attention_backward(do, q, k, v, out, lse, 0, 4), want, bounds, ("dq", "dk", "dv")):
        assert_within(g.numpy(), x, bound, dtype, name)


# ---- many small probabilities ---------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("tq,tk,heads", [(1, 4097, 2), (1, 70001, 2), (40, 4097, 2), (130, 2200, 64)])
@pytest.mark.parametrize("first", [True, False], ids=["first", "last"])
def test_many_keys_far_below_the_largest(dev, ops, dtype, tq, tk, heads, first):
    """One key stands 17 above all others, whose probabilities of 2^-24.5 are
    what the result is made of.  float16 has them as subnormals: a probability
    is rounded at 2^7 times its size against the row's bound, so it is off by
    half of the smallest step, 2^-25, over 2^7, besides its half step."""
    d = 16
    q, k, v, _ = (wide(x, dtype) for x in make(dtype, 1, tq, tk, heads, heads, d, 110))
    q[:], k[:] = 0.0, 0.0
    q[..., 0] = 1.0
    k[:, 0 if first else tk - tq, :, 0] = 17.0
    v = np.abs(v)
    v[:, 0 if first else tk - tq] = 0.0
    host = [orc.from_float(x.astype(np.float32), dtype) for x in (q, k, v)]
    a = Attention(dtype, *[wide(x, dtype) for x in host], scale=1.0)
    out, lse = ops.sliding_window_attention(*[put(x, dtype) for x in host], scale=1.0)
    bound = a.out_bound + (2.0 ** -32 * (a.see @ np.abs(a.v)) if dtype == F16 else 0.0)
    assert_within(out.numpy(), a.tokens(a.out), a.tokens(bound), dtype, "out")
    assert_within(lse.numpy(), a.lse, a.lse_bound, F32, "lse")


# ---- numbers of tokens past 64 bits -----------------------------------------------------


def test_windows_past_64_bits(dev, ops):
    """A window of 2^70 is none, and 2^63 first tokens are all of them.  (The same
    keys in tiles of another order: P is off by under 2^-16 of itself, its sums
    over 40 keys by no more, and dS is a difference of two such sums.)"""
    q, k, v, do = (put(x, F32) for x in make(F32, 1, 9, 40, 2, 1, 16, 120))
    want = ops.sliding_window_attention(q, k, v)
    grads = ops.sliding_window_attention_backward(do, q, k, v, *want)
    for rule in (dict(window=2 ** 70), dict(window=2, sinks=2 ** 63), dict(window=-2 ** 70)):
        got = ops.sliding_window_attention(q, k, v, **rule)
        assert_within(got[0].numpy(), want[0].numpy(), 2.0 ** -15 * np.abs(want[0].numpy()).max(), F32, str(rule))
        for g, w in zip(ops.sliding_window_attention_backward(do, q, k, v, *got, **rule), grads):
            assert_within(g.numpy(), w.numpy(), 2.0 ** -13 * np.abs(w.numpy()).max(), F32, str(rule))


# ---- several values that are not finite --------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1, 200, 200, 2, 1, 64), (1, 6, 500, 4, 2, 96), (2, 200, 200, 128, 64, 40)], ids=str)
def test_each_element_has_its_own(dev, ops, dtype, shape):
    """Two values are infinite, in elements 5 and 9: a query that sees the first
    alone is infinite in 5 and as ever in 9.  The same of two gradients and dv."""
    b, tq, tk, h, hk, d = shape
    host = make(dtype, *shape, 130)
    w = [wide(x, dtype) for x in host]
    a = Attention(dtype, *w[:3])
    want, bounds = a.backward(w[3], dtype)
    group, last = h // hk, tk - 3
    at = ((tk - tq, 5), (last, 9))  # every query sees the first, two see the second
    v = host[2].copy()
    for key, e in at:
        v[0, key, 0, e] = one(np.inf, dtype)
    q, k, dv_ = put(host[0], dtype), put(host[1], dtype), put(host[2], dtype)
    out, _ = ops.sliding_window_attention(q, k, put(v, dtype))
    o, o64, bound = wide(out.numpy(), dtype), a.tokens(a.out).copy(), a.tokens(a.out_bound).copy()
    for key, e in at:
        rows = tk - tq + np.arange(tq) >= key
        assert np.isposinf(o[0, rows, :group, e]).all()
        for x in (o, o64, bound):
            x[0, rows, :group, e] = 0.0
    assert_within(orc.from_float(o.astype(np.float32), dtype), o64, bound, dtype, "out")
    # query 1 sees keys up to tk - tq + 1, the last one all keys
    do = host[3].copy()
    at = ((1, 5), (tq - 1, 9))
    for i, e in at:
        do[0, i, 0, e] = one(np.inf, dtype)
    out, lse = ops.sliding_window_attention(q, k, dv_)
    dv = wide(ops.sliding_window_attention_backward(put(do, dtype), q, k, dv_, out, lse)[2].numpy(), dtype)
    v64, bound = want[2].copy(), bounds[2].copy()
    for i, e in at:
        keys = np.arange(tk) <= tk - tq + i
        assert np.isposinf(dv[0, keys, 0, e]).all()
        for x in (dv, v64, bound):
            x[0, keys, 0, e] = 0.0
    assert_within(orc.from_float(dv.astype(np.float32), dtype), v64, bound, dtype, "dv")
