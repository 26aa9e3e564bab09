"""Attention with a sliding window and first tokens on the GPU against
float64, forward and backward.

Tolerances (``_attention.Attention``), u = 2^-24 and h half a step of the
type.  A score is off by (D + 8) u of the sum of its products' magnitudes and
4 u of its size; a probability by twice that, relative, and (2 n + 16) u for
the sum of n of them; rounding it to 16 bits adds h.  Out and dv are sums of
probabilities times what they multiply, dq and dk of dS = P (dP - D), where
D carries the rounding of out.  Every error is taken at its largest, with no
luck among the terms; then one rounding to the type.
"""

import numpy as np
import pytest

from _attention import BF16, F16, F32, Attention, assert_within, mod, put, sample, wide

pytestmark = pytest.mark.gpu

DTYPES = [F32, F16, BF16]
IDS = ["fp32", "fp16", "bf16"]


def make(dtype, b, tq, tk, h, hk, d, seed=0):
    return [sample(s, dtype, seed + i) for i, s in enumerate(((b, tq, h, d), (b, tk, hk, d), (b, tk, hk, d), (b, tq, h, d)))]


def check(ops, dtype, host, rule, views=None, backward=True):
    """One call and its backward against float64; ``host`` holds q, k, v, do
    as stored, ``views`` the device operands when not plain copies."""
    wide_ = [wide(x, dtype) for x in host]
    a = Attention(dtype, *wide_[:3], **rule)
    dev = views or [put(x, dtype) for x in host]
    given = {n: put(np.asarray(x)) if n in ("lengths", "starts") and x is not None else x for n, x in rule.items()}
    out, lse = ops.sliding_window_attention(*dev[:3], **given)
    assert out.is_contiguous() and out.shape == host[0].shape and lse.shape == a.lse.shape
    assert_within(out.numpy(), a.tokens(a.out), a.tokens(a.out_bound), dtype, "out")
    assert_within(lse.numpy(), a.lse, a.lse_bound, F32, "lse")
    if not backward:
        return out, lse
    grads = ops.sliding_window_attention_backward(dev[3], *dev[:3], out, lse, **given)
    want, bounds = a.backward(wide_[3], dtype)
    for g, w, bound, name in zip(grads, want, bounds, ("dq", "dk", "dv")):
        assert g.is_contiguous()
        assert_within(g.numpy(), w, bound, dtype, name)
    return out, lse, *grads


RULES = [
    dict(),
    dict(window=1),
    dict(window=2, sinks=1),
    dict(window=33, sinks=4),
    dict(window=64),
    dict(window=100, sinks=70),
    dict(window=0, sinks=5),
    dict(window=0),
    dict(window=1000, sinks=3),
    dict(window=17, sinks=10 ** 12),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rule", RULES, ids=str)
def test_rules(dev, ops, dtype, rule):
    check(ops, dtype, make(dtype, 2, 200, 200, 4, 2, 64), rule)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("tq,tk", [(1, 1), (1, 2), (1, 33), (1, 300), (3, 130), (31, 31), (32, 32), (33, 64), (64, 65), (127, 127),
                                   (128, 128), (129, 129), (130, 257), (257, 400)])
def test_lengths_of_axes(dev, ops, dtype, tq, tk):
    check(ops, dtype, make(dtype, 1, tq, tk, 3, 3, 128, 10), dict(window=70, sinks=2))
    check(ops, dtype, make(dtype, 1, tq, tk, 2, 1, 32, 20), dict())


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("dim", [1, 2, 5, 8, 16, 24, 33, 40, 64, 72, 80, 96, 100, 104, 120, 128])
def test_head_sizes(dev, ops, dtype, dim):
    """Among them sizes that are no whole number of packets (copied)."""
    check(ops, dtype, make(dtype, 2, 70, 90, 4, 2, dim, 30), dict(window=40, sinks=2))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 1), (6, 2), (8, 1), (12, 12), (40, 2)])
def test_shared_heads(dev, ops, dtype, heads, kv):
    check(ops, dtype, make(dtype, 2, 65, 140, heads, kv, 48, 40), dict(window=90, sinks=1))
    check(ops, dtype, make(dtype, 2, 1, 140, heads, kv, 48, 40), dict(window=90, sinks=1))


@pytest.mark.parametrize("index", [np.int32, np.int64], ids=["i32", "i64"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("tq", [1, 4, 60, 150])
def test_padded_batches(dev, ops, dtype, tq, index):
    """Sequences of every length, none and more than the keys among them;
    queries before their sequence's first position and behind its last."""
    tk = 150
    lengths = np.array([150, 149, 65, 64, 1, 0, -5, 2000, 100, 3], index)
    host = make(dtype, len(lengths), tq, tk, 4, 2, 64, 50)
    check(ops, dtype, host, dict(window=50, sinks=3, lengths=lengths))
    starts = np.array([0, 10, -3, 63, 0, 0, 1, 149, 99, -2 ** 31], index)
    check(ops, dtype, host, dict(window=50, sinks=3, lengths=lengths, starts=starts))
    check(ops, dtype, host, dict(starts=np.array([0, 2 ** 31 - 1, 149, -149, 1, 5, 30, 70, 90, 100], index)))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("tq", [1, 90])
def test_memory_nobody_sees(dev, ops, dtype, tq):
    """NaN past a sequence's end, between the first tokens and the window, and
    in rows of queries outside their sequence is not read."""
    b, tk, h, hk, d = 4, 200, 4, 2, 64
    lengths = np.array([200, 131, 64, 20])
    host = make(dtype, b, tq, tk, h, hk, d, 60)
    rule = dict(window=40, sinks=3, lengths=lengths)
    a = Attention(dtype, *[wide(x, dtype) for x in host[:3]], **rule)
    nan = {F32: np.float32(np.nan), F16: np.float16(np.nan), BF16: np.uint16(0x7FC0)}[dtype]
    unseen, dead = ~a.see.any((1, 2)), ~a.see.any(-1)[:, 0]
    for x in host[1:3]:
        x[unseen] = nan
    for x in (host[0], host[3]):
        x[dead] = nan
    for x, y in zip(check(ops, dtype, host, rule), (None, None, dead, unseen, unseen)):
        x64 = wide(x.numpy(), dtype if x.ndim == 4 else F32)
        assert not np.isnan(x64).any() and (y is None or (x64[y] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_layouts(dev, ops, dtype):
    """Heads before tokens, a packed projection, a cache longer than its
    view, a token shared by stride 0, rows that begin anywhere."""
    b, tq, tk, h, hk, d = 2, 70, 100, 4, 2, 64
    host = make(dtype, b, tq, tk, h, hk, d, 70)
    rule = dict(window=50, sinks=2)

    def heads_first(x):
        return put(np.ascontiguousarray(x.transpose(0, 2, 1, 3)), dtype).transpose(1, 2)

    check(ops, dtype, host, rule, [heads_first(x) for x in host])

    def in_cache(x):
        big = sample((b + 1, x.shape[1] + 9, x.shape[2] + 1, d), dtype, 71)
        big[1:, 5:5 + x.shape[1], :x.shape[2]] = x
        return put(big, dtype)[1:, 5:5 + x.shape[1], :x.shape[2]]

    check(ops, dtype, host, rule, [in_cache(x) for x in host])

    def off_by_one(x):
        flat = np.concatenate([x.reshape(-1)[:1], x.reshape(-1)])
        return put(flat, dtype)[1:].view(*x.shape)

    check(ops, dtype, host, rule, [off_by_one(x) for x in host])

    def wide_last(x):
        return put(np.repeat(x, 2, -1), dtype)[:, :, :, ::2]

    check(ops, dtype, host, rule, [wide_last(x) for x in host])
    one = [x[:, :1] for x in host[1:3]]
    same = [host[0], *[np.repeat(x, tk, 1) for x in one], host[3]]
    views = [put(x, dtype) for x in same]
    views[1:3] = [put(np.ascontiguousarray(x), dtype).expand(b, tk, hk, d) for x in one]
    check(ops, dtype, same, rule, views)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("tq", [1, 130])
def test_large_scores(dev, ops, dtype, tq):
    """Scores in the thousands, growing along the keys: the running bound is
    passed again and again, and nothing overflows."""
    host = make(dtype, 1, tq, 300, 2, 1, 64, 80)
    grow = np.linspace(0.1, 30.0, 300)[None, :, None, None]
    from oracle import binding
    host[1] = binding.from_float((wide(host[1], dtype) * grow).astype(np.float32), dtype)
    out, lse, *grads = check(ops, dtype, host, dict(scale=1.5))
    assert np.abs(lse.numpy()).max() > 100
    host[1] = binding.from_float((-wide(host[1], dtype)[:, ::-1]).astype(np.float32), dtype)
    check(ops, dtype, host, dict(scale=1.5, window=100, sinks=4))


@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS[1:])
@pytest.mark.parametrize("tq", [1, 40])
def test_values_that_are_not_finite(dev, ops, dtype, tq):
    """A key that every query sees: NaN or +inf in it or in its value shows in
    every row, and one score of -inf takes its key out."""
    host = make(dtype, 1, tq, 50, 2, 2, 32, 90)
    inf, nan = {F16: (0x7C00, 0x7E00), BF16: (0x7F80, 0x7FC0)}[dtype]
    bits = [x.view(np.uint16) for x in host]
    bits[2][0, 3, 0, 5] = inf
    bits[1][0, 2, 1, 7] = nan
    out, lse = ops.sliding_window_attention(*[put(x, dtype) for x in host[:3]])
    o, l = wide(out.numpy(), dtype), lse.numpy()
    assert np.isposinf(o[0, :, 0, 5]).all() and np.isfinite(np.delete(o[0, :, 0], 5, -1)).all()
    assert np.isnan(o[0, :, 1]).all() and np.isnan(l[0, 1]).all() and np.isfinite(l[0, 0]).all()
    host = make(dtype, 1, tq, 50, 1, 1, 32, 95)
    host[0].view(np.uint16)[..., 4] = {F16: 0x3C00, BF16: 0x3F80}[dtype]  # 1
    host[1].view(np.uint16)[0, 6, 0, 4] = inf | 0x8000
    out, lse = ops.sliding_window_attention(*[put(x, dtype) for x in host[:3]])
    keep = np.delete(np.arange(50), 6)
    q, k, v = (wide(x, dtype) for x in host[:3])
    k[0, 6] = 0
    s = np.einsum("id,jd->ij", q[0, :, 0], k[0, :, 0]) * 32 ** -0.5
    s[np.arange(50)[None] > np.arange(50 - tq, 50)[:, None]] = -np.inf
    p = np.exp(s[:, keep])
    assert np.allclose(wide(out.numpy(), dtype)[0, :, 0], p @ v[0, keep, 0] / p.sum(1, keepdims=True), rtol=0, atol=0.05)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_walks_in_parts(dev, ops, dtype):
    """First tokens that thousands of queries see, and few heads of many keys:
    the gradients' sums come in parts.  Twice the same bits."""
    host = make(dtype, 1, 1500, 1500, 2, 1, 64, 100)
    first = check(ops, dtype, host, dict(window=64, sinks=130))
    again = check(ops, dtype, host, dict(window=64, sinks=130))
    for x, y in zip(first, again):
        assert np.array_equal(x.numpy(), y.numpy())
    check(ops, dtype, host, dict())


def test_sums_of_many_first_tokens_stay_small(dev, ops):
    """Thousands of first tokens beside a short window: the parts of their
    walks are bounded by the device's blocks, not by the walks' length."""
    runtime = mod("runtime")
    t, h, d = 8192, 4, 128
    q, k, v, do = (put(x, BF16) for x in make(BF16, 1, t, t, h, h, d, 180))
    out, lse = ops.sliding_window_attention(q, k, v, 1, 4096)
    runtime.synchronize()
    runtime.reset_peak_memory_stats()
    before = runtime.memory_allocated()
    dq, dk, dv = ops.sliding_window_attention_backward(do, q, k, v, out, lse, 1, 4096)
    runtime.synchronize()
    # parts: at most 4 rounds of 4 blocks a CU and one more a block of first
    # tokens, of 2 x 32 rows of float32; results and statistics beside them
    blocks = 16 * runtime.compute_units() + h * 4096 // 32
    bound = blocks * 2 * 32 * d * 4 + 3 * t * h * d * 2 + 2 * t * h * 4
    assert runtime.max_memory_allocated() - before <= 1.1 * bound
    # the rows of dv add up to do: every row of P adds up to 1 (each P rounded
    # to bf16, 8192 rows of do's size, and dv's own rounding)
    d64 = wide(do.numpy(), BF16)[0].sum(0)
    v64 = wide(dv.numpy(), BF16)[0]
    assert (np.abs(v64.sum(0) - d64) <= 2.0 ** -8 * (np.abs(wide(do.numpy(), BF16)[0]).sum(0) + np.abs(v64).sum(0)) + 1e-2).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rule", RULES, ids=str)
def test_many_heads(dev, ops, dtype, rule):
    """Work enough for blocks of several waves on every kernel's side, of heads
    that share keys and of heads that do not."""
    check(ops, dtype, make(dtype, 2, 131, 131, 128, 32, 40, 150), rule)
    check(ops, dtype, make(dtype, 2, 70, 140, 128, 128, 24, 160), rule)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("tq,dim", [(150, 64), (290, 128)])
def test_many_heads_padded(dev, ops, dtype, tq, dim):
    """The same, and long walks in parts, over sequences of every length."""
    lengths, starts = np.array([290, 130, 0, 1]), np.array([140, -3, 0, 289 - tq])
    for heads, kv in ((32, 32), (32, 1)):
        host = make(dtype, 4, tq, 290, heads, kv, dim, 170)
        check(ops, dtype, host, dict(lengths=lengths, starts=starts))
        check(ops, dtype, host, dict(window=129, sinks=5, lengths=lengths))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("batch,tq,heads,kv", [(1, 1, 8, 8), (1, 1, 8, 1), (3, 2, 6, 2), (5, 9, 8, 2), (64, 1, 4, 2), (2, 33, 4, 1)])
def test_long_caches(dev, ops, dtype, batch, tq, heads, kv):
    """A few queries over a long cache: the keys are split over blocks."""
    tk = 5000
    lengths = np.maximum(tk - 613 * np.arange(batch) % tk, 1)
    host = make(dtype, batch, tq, tk, heads, kv, 64, 110)
    check(ops, dtype, host, dict(lengths=lengths), backward=False)
    check(ops, dtype, host, dict(window=1777, sinks=65, lengths=lengths), backward=False)


@pytest.mark.parametrize("shape", [(0, 3, 5, 2, 1), (2, 0, 5, 2, 1), (2, 3, 0, 2, 1), (2, 3, 5, 0, 1)], ids=["batch", "queries", "keys", "heads"])
def test_empty(dev, ops, shape):
    b, tq, tk, h, hk = shape
    q, k, v, do = (put(x, F32) for x in make(F32, b, tq, tk, h, hk, 16))
    out, lse = ops.sliding_window_attention(q, k, v, 4, 1)
    assert out.shape == (b, tq, h, 16) and (out.numpy() == 0).all() and (lse.numpy() == -np.inf).all()
    grads = ops.sliding_window_attention_backward(do, q, k, v, out, lse, 4, 1)
    for g, x in zip(grads, (q, k, v)):
        assert g.shape == x.shape and (g.numpy() == 0).all()


def test_a_layer_recorded_and_replayed(dev, ops):
    """Projection, head norm with rotation, attention, output projection and
    the way back through all of them, as a layer has them, in a recording that
    is replayed on new inputs between eager steps; and a decode step over the
    cache the layer's keys make."""
    graph, runtime = mod("graph"), mod("runtime")
    b, t, h, hk, d = 2, 150, 4, 2, 64
    width = (h + 2 * hk) * d
    from _attention import table_of
    x = put(sample((b * t, 128), BF16, 1), BF16)
    w_in, w_out = put(sample((width, 128), BF16, 2, 128 ** -0.5), BF16), put(sample((128, h * d), BF16, 3, (h * d) ** -0.5), BF16)
    norm = put(sample((d,), BF16, 4, 0.2, 1.0), BF16)
    tab, pos, dy = put(table_of(t, d)), put(np.arange(t)), put(sample((b * t, 128), BF16, 5), BF16)
    rule = dict(window=40, sinks=3)

    def heads(packed, first, n):
        part = packed.view(b, t, width)[:, :, first * d: (first + n) * d]
        return part._view([b, t, n, d], [part.strides[0], part.strides[1], d, 1])

    def step():
        packed = ops.linear(x, w_in)
        q, k, v = heads(packed, 0, h), heads(packed, h, hk), heads(packed, h + hk, hk)
        qr, kr, sq, sk = ops.qk_norm_rope(q, k, tab, pos, norm, norm)
        out, lse = ops.sliding_window_attention(qr, kr, v, **rule)
        y = ops.linear(out.view(b * t, h * d), w_out)
        dout = ops.mm(dy, w_out).view(b, t, h, d)
        dq, dk, dv = ops.sliding_window_attention_backward(dout, qr, kr, v, out, lse, **rule)
        gq, gk, wq, wk = ops.qk_norm_rope_backward(dq, dk, q, k, tab, pos, sq, sk, norm, norm)
        last = qr[:, t - 1:]
        one, _ = ops.sliding_window_attention(last, kr, v, **rule)
        return [packed, qr, kr, out, lse, y, gq, gk, dv, wq, wk, one]

    g = graph.Graph()
    try:
        results = g.capture(step)
        for i in range(4):
            ops.copy_(x, sample((b * t, 128), F32, 20 + i))
            g.replay()
            runtime.synchronize()
            eager = step()
            for a, c in zip(results, eager):
                assert np.array_equal(a.numpy(), c.numpy())
    finally:
        g.reset()
    packed, qr, kr, out = eager[:4]
    a = Attention(BF16, wide(qr.numpy(), BF16), wide(kr.numpy(), BF16), wide(heads(packed, h + hk, hk).numpy(), BF16), **rule)
    assert_within(out.numpy(), a.tokens(a.out), a.tokens(a.out_bound), BF16, "out")
    assert_within(eager[11].numpy(), a.tokens(a.out)[:, -1:], a.tokens(a.out_bound)[:, -1:], BF16, "one token")


@pytest.mark.parametrize("tq", [1, 130], ids=["split", "wide"])
def test_offsets_past_32_bits(dev, ops, tq):
    """A cache of more than 2^31 elements: the first tokens and the window's
    are at its two ends."""
    h, d, tk = 64, 128, 270000
    k, v = ops.empty((1, tk, h, d), "bfloat16"), ops.empty((1, tk, h, d), "bfloat16")
    assert k.numel() > 2 ** 31
    near, sinks, window = 260, 3, 100
    q, *tail = make(BF16, 1, tq, near, h, h, d, 120)[:3]
    head = make(BF16, 1, 1, sinks, h, h, d, 130)[1:3]
    for cache, a, b in zip((k, v), head, tail):
        ops.zero_(cache)
        ops.copy_(cache[:, :sinks], put(a, BF16))
        ops.copy_(cache[:, tk - near:], put(b, BF16))
    out, lse = ops.sliding_window_attention(put(q, BF16), k, v, window, sinks)
    # the same rows with what lies between left out: nobody sees it
    short = [np.concatenate([a, b], 1) for a, b in zip(head, tail)]
    a = Attention(BF16, wide(q, BF16), *[wide(x, BF16) for x in short], window=window, sinks=sinks)
    assert_within(out.numpy(), a.tokens(a.out), a.tokens(a.out_bound), BF16, "out")
    assert_within(lse.numpy(), a.lse, a.lse_bound, F32, "lse")


def test_more_rows_than_a_launch_has(dev, ops):
    """2^24 sequences' blocks of 256 threads are 2^32 threads: refused."""
    one = put(np.zeros((1, 1, 1, 8), np.float16)).expand(1 << 24, 1, 1, 8)
    with pytest.raises(mod("tensor").DeviceError, match="too many rows"):
        ops.sliding_window_attention(one, one, one)


@pytest.mark.parametrize("tq", [1, 200])
def test_scores_of_minus_infinity_only(dev, ops, tq):
    """A row whose every score is -inf has no sum: zeros, -inf, no gradient."""
    q, k, v, do = make(F32, 1, tq, 200, 1, 1, 16, 140)
    q[:, :, :, 3], k[0, :, 0, 3] = 1.0, -np.inf
    q, k, v, do = (put(x) for x in (q, k, v, do))
    out, lse = ops.sliding_window_attention(q, k, v)
    assert (out.numpy() == 0).all() and (lse.numpy() == -np.inf).all()
    dv = ops.sliding_window_attention_backward(do, q, k, v, out, lse)[2]
    assert (dv.numpy() == 0).all()
