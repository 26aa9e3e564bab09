"""Dropout of more elements than 2^34: their generator's blocks have numbers
past 32 bits.  The join's operands are one row expanded, so that only its
result takes memory.  The join's backward and the log probabilities past 2^31
elements.  More rows than one launch takes: 2^24 - 1 a block each, 2^26 - 4 a
wave each."""

import numpy as np
import pytest

from oracle import binding as orc

from _attention import BF16, F32, assert_within, put, sample, wide
from _layers import Join, Probs

pytestmark = pytest.mark.gpu

DIM, ROWS = 16384, (1 << 20) + 3  # element 2^34 begins row 2^20
SEED, P = (99 << 32) + 1234, 0.4


def kept_row(row, width, offset=0):
    """Which elements of a row the generator keeps, block by block."""
    first = row * width
    key = np.array([SEED & 0xFFFFFFFF, SEED >> 32], np.uint32)
    words = []
    for block in range(first // 4, (first + width + 3) // 4):
        ctr = np.array([block & 0xFFFFFFFF, block >> 32, offset & 0xFFFFFFFF, offset >> 32], np.uint32)
        words.append(orc.philox4x32_10(ctr, key))
    words = np.concatenate(words)[first % 4: first % 4 + width]
    return (words >> 8) >= np.ceil(P * 2 ** 24)


@pytest.fixture
def memory(amd):
    yield
    amd.load().tp_mlu_empty_cache()


@pytest.mark.parametrize("width,rows", [(DIM, [0, 5, (1 << 20) - 1, 1 << 20, ROWS - 1]), (DIM - 1, [7, (1 << 20) + 63, (1 << 20) + 64, (1 << 20) + 66])],
                         ids=["whole_blocks", "blocks_across_rows"])
def test_join(dev, ops, memory, width, rows):
    count = max(rows) + 1
    x, y = sample((1, width), BF16, 1), sample((1, width), BF16, 2)
    z, h, _, _ = ops.residual_norm(put(x, BF16).expand(count, width), put(y, BF16).expand(count, width), eps=None, p=P, seed=SEED)
    assert h is None and z.shape == (count, width)
    for r in rows:
        got = wide(z[r].numpy(), BF16)
        # kept: two roundings of the product and the sum in float32, one to bfloat16
        x64, u = wide(x[0], BF16), np.where(kept_row(r, width), wide(y[0], BF16) / (1 - P), 0.0)
        assert (np.abs(got - (x64 + u)) <= 2.0 ** -8 * np.abs(x64 + u) + 2.0 ** -21 * (np.abs(x64) + np.abs(u))).all(), r


def test_dropout(dev, ops, memory):
    x = sample((1, DIM), BF16, 3)
    out = ops.seeded_dropout(put(x, BF16).expand(ROWS, DIM), P, SEED)
    for r in (0, (1 << 20) - 1, 1 << 20, ROWS - 1):
        want = np.where(kept_row(r, DIM), wide(x[0], BF16).astype(np.float32) * np.float32(1 / (1 - P)), np.float32(0))
        assert np.array_equal(out[r].numpy(), orc.from_float(want, BF16)), r


def test_join_backward(dev, ops, memory):
    """More than 2^31 elements a tensor; rows differ by what dropout left of them."""
    width, rows = 4096, (1 << 19) + 9
    x = ops.seeded_dropout(put(sample((1, width), BF16, 4), BF16).expand(rows, width), P, SEED)
    y, dz = (put(sample((1, width), BF16, i), BF16).expand(rows, width) for i in (5, 6))
    z, h, r1, r2 = ops.residual_norm(x, y, branch_eps=1e-6, p=P, seed=SEED, offset=1)
    dx, dy, _, _, _ = ops.residual_norm_backward(dz, h, x, y, r1, r2, p=P, seed=SEED, offset=1)
    for r in (0, (1 << 19) - 1, 1 << 19, rows - 1):
        row = [wide(t[r: r + 1].numpy(), BF16) for t in (x, y, dz, h)]
        j = Join(row[0], row[1], eps1=1e-6, keep=kept_row(r, width, 1)[None], p=P)
        assert_within(z[r: r + 1].numpy(), j.z, j.z_bound, BF16, "sum")
        assert_within(h[r: r + 1].numpy(), j.h, j.h_bound, BF16, "normed")
        want, bound = j.backward(row[2], row[3], *(t[r: r + 1].numpy().astype(np.float64) for t in (r1, r2)))
        assert_within(dx[r: r + 1].numpy(), want["dx"], bound["dx"], BF16, "dx")
        assert_within(dy[r: r + 1].numpy(), want["dy"], bound["dy"], BF16, "dy")


def test_log_probs(dev, ops, memory):
    """More than 2^31 logits."""
    vocab, rows = 32000, 70001
    x = ops.seeded_dropout(put(sample((1, vocab), BF16, 7), BF16).expand(rows, vocab), P, SEED)
    t = np.random.default_rng(8).integers(0, vocab, rows)
    da, db = (np.random.default_rng(i).standard_normal(rows).astype(np.float32) for i in (9, 10))
    lp, h, stats, top, index = ops.token_log_probs(x, put(t), top=3, entropy=True)
    dx = ops.token_log_probs_backward(put(da), put(db), x, put(t), stats, h)
    for r in (0, (1 << 31) // vocab, (1 << 31) // vocab + 1, rows - 1):
        want = Probs(wide(x[r: r + 1].numpy(), BF16), t[r: r + 1])
        given, bound = want.given()
        assert_within(lp[r: r + 1].numpy(), given, bound, F32, "logprob")
        assert_within(h[r: r + 1].numpy(), want.h, want.h_bound, F32, "entropy")
        order, values, bound = want.top(3)
        assert np.array_equal(index[r: r + 1].numpy(), order)
        assert_within(top[r: r + 1].numpy(), values, bound, F32, "alternatives")
        grad, bound = want.backward(da[r: r + 1], db[r: r + 1])
        assert_within(dx[r: r + 1].numpy(), grad, bound, BF16, "gradient")


def test_log_probs_of_more_rows_than_a_launch_takes(dev, ops, memory):
    vocab, rows, block = 5, (1 << 26) + 5, (1 << 24) - 1
    x = ops.seeded_dropout(put(sample((1, vocab), BF16, 11), BF16).expand(rows, vocab), P, SEED)
    t = np.random.default_rng(12).integers(0, vocab, rows, np.int32)
    t[block], t[-1] = -100, vocab
    da = np.random.default_rng(13).standard_normal(rows, np.float32)
    lp, h, stats, top, index = ops.token_log_probs(x, put(t), top=2)
    dx = ops.token_log_probs_backward(put(da), put(da), x, put(t), stats, h)
    for first in (0, block - 3, 2 * block - 3, 4 * block - 3, (1 << 26) - 7, rows - 7):
        at = slice(first, first + 7)
        want = Probs(wide(x[at].numpy(), BF16), t[at].astype(np.int64), lanes=64)
        given, bound = want.given()
        assert_within(lp[at].numpy(), given, bound, F32, "logprob")
        assert_within(h[at].numpy(), want.h, np.where(want.skipped, 0, want.h_bound), F32, "entropy")
        order, values, bound = want.top(2)
        assert np.array_equal(index[at].numpy(), order)
        assert_within(top[at].numpy(), values, bound, F32, "alternatives")
        grad, bound = want.backward(da[at], da[at])
        assert_within(dx[at].numpy(), grad, bound, BF16, "gradient")


def test_norm_of_more_rows_than_a_launch_takes(dev, ops, memory):
    """64 lanes a row: 2^26 - 4 rows a launch."""
    width, rows, launch = 264, (1 << 26) + 5, (1 << 26) - 4
    base = sample((1, width), BF16, 14)
    _, h, _, r = ops.residual_norm(put(base, BF16).expand(rows, width))
    j = Join(wide(base, BF16))
    for first in (0, launch - 3, rows - 7):
        at = slice(first, first + 7)
        assert_within(h[at].numpy(), np.broadcast_to(j.h, (7, width)), j.h_bound, BF16, "normed")
        assert_within(r[at].numpy(), np.broadcast_to(j.r2, 7), j.r2_bound, F32, "rstd")
