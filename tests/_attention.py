"""The attention layer's operators in float64 numpy, from their definitions,
and the operands the tests hand to the library."""

from __future__ import annotations

import importlib

import numpy as np

from oracle import binding as orc

F32, F16, BF16 = orc.F32, orc.F16, orc.BF16
#: half a step of each type, relative to the value, and its smallest step's half
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -134}
U = 2.0 ** -24


def mod(name):
    return importlib.import_module("tensorplay-mlu_amd." + name)


def sample(shape, dtype, seed=0, std=1.0, shift=0.0):
    x = np.random.default_rng(seed).standard_normal(shape).astype(np.float32)
    return orc.from_float(x * np.float32(std) + np.float32(shift), dtype)


def wide(x, dtype):
    return orc.to_float(x, dtype).astype(np.float64)


def put(x, dtype=None):
    return mod("tensor").DeviceTensor.from_numpy(x, dtype=dtype)


def fake(shape, dtype="bfloat16", device=0, strides=None):
    """A view of device memory that is not there: for calls that have to be
    refused before anything is read."""
    abi, tensor = mod("_abi"), mod("tensor")
    ref = abi.Tensor()
    ref.data, ref.ctx, ref.ndim = 1 << 20, None, len(shape)
    strides = strides if strides is not None else tensor.contiguous_strides(shape)
    for i, (n, s) in enumerate(zip(shape, strides)):
        ref.sizes[i], ref.strides[i] = n, s
    ref.dtype, ref.device = tensor.dtype_code(dtype), device
    return tensor.DeviceTensor(ref, owner=object())


def assert_within(got, want, bound, dtype, what=""):
    """|got - want| <= bound + the rounding of want + bound to ``dtype``; NaN
    and infinities in the same places."""
    g, w = wide(got, dtype), np.asarray(want, np.float64)
    assert g.shape == w.shape, (what, g.shape, w.shape)
    assert np.array_equal(np.isnan(g), np.isnan(w)), f"{what}: NaN in other places"
    inf = np.isinf(w)
    assert np.array_equal(g[inf], w[inf]), f"{what}: infinities differ"
    fine = np.isfinite(w)
    b = np.broadcast_to(np.asarray(bound, np.float64), w.shape)
    with np.errstate(invalid="ignore"):
        off = np.abs(g - w)
        allowed = b + HALF[dtype] * (np.abs(w) + b) + TINY[dtype]
    bad = fine & ~(off <= allowed)
    if bad.any():
        i = np.unravel_index(int(np.flatnonzero(bad)[0]), w.shape)
        raise AssertionError(f"{what}: {int(bad.sum())} of {w.size} beyond the bound; first at {i}: got {g[i]!r} want "
                             f"{w[i]!r} allowed {allowed[i]!r}; worst {float(np.max(off[bad] / allowed[bad])):.3g} times")


# ---- norm and rotation ---------------------------------------------------------


def table_of(rows, rotary, base=10000.0):
    """float32 [rows, rotary]: cosines, then sines."""
    angle = np.arange(rows)[:, None] * base ** -(np.arange(rotary // 2) * 2.0 / max(rotary, 1))
    return np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)


def pair_index(dim, rotary, interleaved):
    j = np.arange(rotary // 2)
    return (2 * j, 2 * j + 1) if interleaved else (j, j + rotary // 2)


def turn(x, table, positions, interleaved, back=False):
    """Rows [tokens..., heads, D] turned by their position's angles."""
    rotary = table.shape[1]
    a, b = pair_index(x.shape[-1], rotary, interleaved)
    known = (positions >= 0) & (positions < table.shape[0])
    row = table.astype(np.float64)[np.where(known, positions, 0)][..., None, :]
    c, s = row[..., : rotary // 2], row[..., rotary // 2:] * (-1 if back else 1)
    y = x.copy()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    y[~known] = np.nan
    return y


def pair_sum(x, rotary, interleaved):
    """|a| + |b| at both elements of every pair, |x| past them."""
    a, b = pair_index(x.shape[-1], rotary, interleaved)
    y = np.abs(x)
    y[..., a] = y[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    return y


def head_norm(x, weight, table, positions, eps, interleaved):
    """(y, r, the magnitude that y's terms have)."""
    r = 1.0 / np.sqrt((x * x).mean(-1) + eps)
    n = x * r[..., None] * weight
    return turn(n, table, positions, interleaved), r, pair_sum(n, table.shape[1], interleaved)


def head_norm_backward(dy, x, r, weight, table, positions, interleaved):
    """(dx, dw, magnitudes of dx's terms, sum of |terms| of dw)."""
    g = turn(dy, table, positions, interleaved, back=True)
    m, u = x * r[..., None], g * weight
    dx = r[..., None] * (u - m * (u * m).mean(-1, keepdims=True))
    size = pair_sum(dy, table.shape[1], interleaved)
    au = size * np.abs(weight)
    mag = r[..., None] * (au + np.abs(m) * (au * np.abs(m)).mean(-1, keepdims=True))
    axes = tuple(range(x.ndim - 1))
    return dx, (g * m).sum(axes), mag, (size * np.abs(m)).sum(axes)


# ---- attention ---------------------------------------------------------------------

#: v_exp_f32 gives 0 for a result under 2^-126.  A row's running bound lies at most
#: 2^8 above its largest exponential, so a probability (at least 2^-8 of what
#: v_exp_f32 formed, over a sum of at least 2^-8) is off by up to 2^-118 besides its
#: relative error; the backward forms it against l itself, off by 2^-126.
FLUSH = 2.0 ** -118


def seen(queries, keys, window, sinks, length=None, start=None):
    """[queries, keys] booleans: which keys each query sees."""
    length = keys if length is None else min(max(int(length), 0), keys)
    start = length - queries if start is None else int(start)
    p = start + np.arange(queries, dtype=np.float64)[:, None]
    j = np.arange(keys)[None, :]
    s = (p >= 0) & (p < length) & (j <= p)
    return s & ((j > p - window) | (j < sinks)) if window >= 0 else s


class Attention:
    """Forward and backward in float64 of operands rounded to ``dtype``, with
    the bounds a pass in float32 with P and dS rounded to ``dtype`` keeps."""

    def __init__(self, dtype, q, k, v, window=-1, sinks=0, scale=None, lengths=None, starts=None):
        b, tq, h, d = q.shape
        tk, hk = k.shape[1:3]
        self.scale = d ** -0.5 if scale is None else scale
        self.h = 0.0 if dtype == F32 else HALF[dtype]
        self.q, self.do = q.transpose(0, 2, 1, 3), None
        self.group = h // hk
        self.k, self.v = (np.repeat(x.transpose(0, 2, 1, 3), self.group, 1) for x in (k, v))
        self.see = np.stack([seen(tq, tk, window, sinks, None if lengths is None else lengths[i],
                                  None if starts is None else starts[i]) for i in range(b)])[:, None]
        dead = ~self.see.any(-1)
        self.q = np.where(dead[..., None], 0.0, self.q)
        unseen = ~self.see.any((1, 2))[:, None, :, None]
        self.k, self.v = (np.where(unseen, 0.0, x) for x in (self.k, self.v))
        with np.errstate(invalid="ignore", divide="ignore"):
            s = self.scale * (self.q @ self.k.swapaxes(-1, -2))
            s = np.where(self.see, s, -np.inf)
            m = s.max(-1, initial=-np.inf, keepdims=True)
            e = np.exp(s - np.where(np.isfinite(m), m, 0.0))
            t = e.sum(-1, keepdims=True)
            self.p = np.where(t > 0, e / np.where(t > 0, t, 1.0), 0.0)
            self.lse = np.where(t > 0, m + np.log(t), -np.inf)[..., 0]
        self.out = self.p @ self.v
        n = self.see.sum(-1, keepdims=True)
        # a score is a sum of d products in float32, then scaled and shifted
        terms = self.scale * np.where(self.see, np.abs(self.q) @ np.abs(self.k).swapaxes(-1, -2), 0.0).max(-1, initial=0.0, keepdims=True)
        size = np.where(self.see, np.abs(s), 0.0).max(-1, initial=0.0, keepdims=True)
        self.ds = (d + 8) * U * terms + 4 * U * size
        self.eps = 2 * self.ds + (2 * n + 16) * U  # of a probability, relative
        self.out_bound = (self.p @ np.abs(self.v)) * (self.h + self.eps) + FLUSH * (self.see @ np.abs(self.v))
        with np.errstate(invalid="ignore"):
            self.lse_bound = np.where(dead, 0.0, (self.ds + (n + 8) * U)[..., 0] + 4 * U * np.abs(np.where(dead, 0, self.lse)))

    @staticmethod
    def tokens(x):
        return x.transpose(0, 2, 1, 3)

    def shared(self, x):
        b, h, t, d = x.shape
        return self.tokens(x.reshape(b, h // self.group, self.group, t, d).sum(2))

    def backward(self, do, dtype):
        """(dq, dk, dv) and their bounds, tokens first."""
        d, n = do.shape[-1], self.see.shape[2] * self.group + self.see.shape[3]
        do = np.where(~self.see.any(-1)[..., None], 0.0, do.transpose(0, 2, 1, 3))
        dp = do @ self.v.swapaxes(-1, -2)
        delta = (do * self.out).sum(-1, keepdims=True)
        ds = self.p * (dp - delta)
        dq, dk = self.scale * (ds @ self.k), self.scale * (ds.swapaxes(-1, -2) @ self.q)
        dv = self.p.swapaxes(-1, -2) @ do
        eps = self.eps + self.lse_bound[..., None] + n * U
        rounded = HALF[dtype] * np.abs(self.out) + self.out_bound
        e_delta = (np.abs(do) * rounded).sum(-1, keepdims=True) + (d + 8) * U * (np.abs(do) * np.abs(self.out)).sum(-1, keepdims=True)
        e_dp = (d + 8) * U * (np.abs(do) @ np.abs(self.v).swapaxes(-1, -2))
        off = self.p * ((np.abs(dp) + np.abs(delta)) * (2 * eps + self.h) + e_dp + e_delta) * (1 + self.h)
        off = off + FLUSH * self.see * (1 + np.abs(dp) + np.abs(delta))
        bq, bk = self.scale * (off @ np.abs(self.k)), self.scale * (off.swapaxes(-1, -2) @ np.abs(self.q))
        bv = (self.p * (eps + self.h) + FLUSH * self.see).swapaxes(-1, -2) @ np.abs(do)
        # a 16-bit dS below the smallest normal value is off by a step of its own
        if dtype == F16:
            bq = bq + self.scale * TINY[F16] * (self.see @ np.abs(self.k))
            bk = bk + self.scale * TINY[F16] * (self.see.swapaxes(-1, -2) @ np.abs(self.q))
            bv = bv + TINY[F16] * (np.broadcast_to(self.see, self.p.shape).swapaxes(-1, -2) @ np.abs(do))
        return ((self.tokens(dq), self.shared(dk), self.shared(dv)),
                (self.tokens(bq), self.shared(bk), self.shared(bv)))
