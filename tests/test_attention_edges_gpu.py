"""Where the attention layer's operators meet what is not finite, not small or
not large: each case against float64 or against the same call without it.

Bounds are those of ``_attention.Attention``; where a test needs a closer one
it is derived beside the test.
"""

import numpy as np
import pytest

from _attention import BF16, F16, F32, Attention, assert_within, put, sample, wide
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
