"""Dropout of more elements than 2^34: their generator's blocks have numbers
past 32 bits.  The join's operands are one row expanded, so that only its
result takes memory."""

import numpy as np
import pytest

from oracle import binding as orc

from _attention import BF16, mod, put, sample, wide

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
