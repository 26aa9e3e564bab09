"""The operators between a model's products in float64 numpy, from their
definitions, with the bounds a pass in float32 keeps.

u = 2^-24.  A row's sums are chains of at most 16 fused steps a thread, 6
exchanges in a wave and 16 waves: 38 u of the sum of their terms' magnitudes,
each bound below rounds that up with its terms' own errors.
"""

from __future__ import annotations

import math

import numpy as np

from oracle import binding as orc

from _attention import F32, U


def kept(p, seed, shape, offset=0):
    """Which elements of a dense tensor the generator keeps."""
    if p == 0:
        return np.ones(shape, bool)
    if p == 1:
        return np.zeros(shape, bool)
    return orc.dropout(F32, np.ones(math.prod(shape), np.float32), p, seed, offset)[1].astype(bool).reshape(shape)


# ---- the join of a block to its residual stream ----------------------------------


class Join:
    """sum, normed and their statistics, gradients, and bounds of each."""

    def __init__(self, x, y=None, gate=None, w1=None, w2=None, a=1.0, b=1.0, eps1=None, eps2=1e-6, keep=None, p=0.0):
        self.x, self.y, self.a, self.b, self.w1, self.w2, self.eps1, self.eps2 = x, y, a, b, w1, w2, eps1, eps2
        self.gate = gate
        self.g = np.ones(1) if gate is None else gate
        self.scale = 1.0 if keep is None or p == 1 else 1.0 / (1.0 - p)
        self.keep = np.ones(x.shape, bool) if keep is None else keep
        self.one1, self.one2 = (np.ones(x.shape[-1]) if w is None else w for w in (w1, w2))
        with np.errstate(invalid="ignore", over="ignore"):
            self.forward()

    def branch(self, r1):
        """b drop(n), its factor without g and n's own, from given statistics."""
        m1 = self.y * (1.0 if r1 is None else r1[..., None])
        n = m1 * (self.one1 if r1 is not None else 1.0)
        return m1, self.b * np.where(self.keep, n * self.scale, 0.0)

    def forward(self):
        x, y = self.x, self.y
        self.r1 = None if self.eps1 is None else 1.0 / np.sqrt((y * y).mean(-1) + self.eps1)
        self.r1_bound = None if self.r1 is None else 24 * U * self.r1
        part = self.g * self.branch(self.r1)[1] if y is not None else 0.0
        self.z = self.a * x + part if y is not None else x
        mag = np.abs(self.a * x) + np.abs(part)
        self.z_bound = 33 * U * mag if y is not None else 0.0 * mag
        if self.eps2 is None:
            return
        mean = (self.z * self.z).mean(-1) + self.eps2
        self.r2 = 1.0 / np.sqrt(mean)
        ratio = np.sqrt((mag * mag).mean(-1) / np.where(mean > 0, mean, 1.0))
        rel = (24 + 33 * ratio) * U
        self.r2_bound = rel * self.r2
        self.h = self.z * self.r2[..., None] * self.one2
        self.h_bound = np.abs(self.r2[..., None] * self.one2) * self.z_bound + np.abs(self.h) * (rel[..., None] + 3 * U)

    def backward(self, dz, dh, r1=None, r2=None):
        """({name: gradient}, {name: bound}) from the statistics given, which
        count as exact."""
        x, y, w1, w2 = self.x, self.y, self.one1, self.one2
        rows = math.prod(x.shape[:-1])
        dz = np.zeros(x.shape) if dz is None else dz
        R2 = np.zeros(x.shape[:-1] + (1,)) if dh is None else r2[..., None]
        dh = np.zeros(x.shape) if dh is None else dh
        z, mag = self.x, np.abs(self.x)
        if y is not None:
            m1, u = self.branch(r1)
            z = self.a * x + self.g * u
            mag = np.abs(self.a * x) + np.abs(self.g * u)
        m2, mag2, v = z * R2, mag * R2, dh * w2
        c, cm = (v * m2).mean(-1, keepdims=True), (np.abs(v) * mag2).mean(-1, keepdims=True)
        G = dz + R2 * (v - m2 * c)
        gm = np.abs(dz) + R2 * np.abs(v) + cm * R2 * mag2
        grads, bounds = {"dx": self.a * G}, {"dx": 67 * U * abs(self.a) * gm}
        if self.w2 is not None:
            axes = tuple(range(x.ndim - 1))
            grads["dw2"], bounds["dw2"] = (dh * m2).sum(axes), (rows + 80) * U * (np.abs(dh) * mag2).sum(axes)
        if y is None:
            return grads, bounds
        f = np.abs(np.where(self.keep, self.b * self.g * self.scale, 0.0))
        q = np.where(self.keep, self.b * self.g * self.scale * G, 0.0)
        grads["dy"], bounds["dy"] = q, 72 * U * f * gm
        if r1 is not None:
            R1 = r1[..., None]
            c1, cm1 = (q * w1 * m1).mean(-1, keepdims=True), (f * np.abs(w1 * m1) * gm).mean(-1, keepdims=True)
            grads["dy"] = R1 * (q * w1 - m1 * c1)
            bounds["dy"] = 120 * U * R1 * (f * np.abs(w1) * gm + np.abs(m1) * cm1)
            if self.w1 is not None:
                grads["dw1"], bounds["dw1"] = (q * m1).sum(axes_of(x)), (rows + 140) * U * (f * np.abs(m1) * gm).sum(axes_of(x))
        if self.gate is not None:
            n = (u * G).size // max(self.gate.size, 1)
            grads["dgate"] = fold_to(u * G, self.gate.shape)
            bounds["dgate"] = (n + 140) * U * fold_to(np.abs(u) * gm, self.gate.shape)
        return grads, bounds


def axes_of(x):
    return tuple(range(x.ndim - 1))


def fold_to(x, shape):
    """Summed over what broadcasting repeated."""
    lead = x.ndim - len(shape)
    x = x.sum(tuple(range(lead))) if lead else x
    axes = tuple(d for d in range(len(shape)) if shape[d] == 1)
    return x.sum(axes, keepdims=True) if axes else x


# ---- log probabilities of tokens ----------------------------------------------------

#: v_exp_f32 gives 0 for a result under 2^-126
FLUSH = 2.0 ** -125


class Probs:
    """Rows [R, V] of logits (float64 of their type), summed by `lanes` at least."""

    def __init__(self, x, targets=None, scale=1.0, ignore=-100, lanes=256):
        self.x, self.t, self.scale = x, targets, scale
        rows, v = x.shape
        self.skipped = np.zeros(rows, bool) if targets is None else targets == ignore
        with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
            self.m = x.max(1)
            d = (x - self.m[:, None]) * scale
            e = np.exp(d)
            self.s = e.sum(1)
            self.ls = np.log(self.s)
            self.log_p = d - self.ls[:, None]
            self.p = np.exp(self.log_p)
            self.h = self.ls - np.where(e > 0, e * d, np.where(np.isnan(d), np.nan, 0.0)).sum(1) / self.s
            far = np.where(np.isfinite(d), -d, 0.0)
            # weights fall as e^d, so e^d |d| sums to what the entropy's own terms do
            size = np.where(np.isfinite(d), e * far, 0.0).sum(1) / self.s
            chain = 1.25 * v / lanes + 80
            srel = (chain + 10 * size) * U
            self.ls_bound = srel + 3 * U * np.abs(self.ls)
            spread = np.where(np.isfinite(d), e * far * far, 0.0).sum(1) / self.s
            self.h_bound = self.ls_bound + size * (2 * chain + 20 * size + 8) * U + 10 * U * spread + 2 * U * np.abs(self.h)
            self.lp_bound = self.ls_bound[:, None] + 4 * U * (far + np.abs(self.ls[:, None]))
        for a in (self.m, self.ls, self.h):
            a[self.skipped] = 0.0

    def given(self):
        """(log probability of the targets, bound)."""
        v = self.x.shape[1]
        known = (self.t >= 0) & (self.t < v)
        at = np.where(known, self.t, 0)[:, None]
        lp = np.take_along_axis(self.log_p, at, 1)[:, 0]
        bound = np.take_along_axis(self.lp_bound, at, 1)[:, 0]
        return np.where(self.skipped, 0.0, np.where(known, lp, np.nan)), np.nan_to_num(np.where(known & ~self.skipped, bound, 0.0))

    def top(self, k):
        """(indices, log probabilities, bounds): falling, of equal ones the lower index first, NaN first of all."""
        key = np.where(np.isnan(self.x), np.inf, self.x)
        order = np.lexsort((np.broadcast_to(np.arange(self.x.shape[1]), self.x.shape), -key, ~np.isnan(self.x)), axis=-1)[:, :k]
        values, bounds = np.take_along_axis(self.log_p, order, 1), np.take_along_axis(self.lp_bound, order, 1)
        order[self.skipped], values[self.skipped] = -1, 0.0
        return order, values, np.nan_to_num(bounds)

    def backward(self, da=None, db=None):
        """(dlogits, bound)."""
        rows, v = self.x.shape
        with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
            a = np.zeros(rows) if da is None else da.astype(np.float64)
            b = np.zeros(rows) if db is None else db.astype(np.float64)
            known = np.zeros(rows, bool) if self.t is None else (self.t >= 0) & (self.t < v)
            if self.t is not None:
                a = np.where(known, a, np.nan)
            log_p = np.where(self.p > 0, self.log_p, np.where(np.isnan(self.log_p), np.nan, 0.0))
            g = a[:, None] + b[:, None] * (log_p + self.h[:, None])
            delta = np.zeros_like(self.x)
            if self.t is not None:
                delta[known, self.t[known]] = 1.0
            dx = self.scale * (np.where(delta > 0, a[:, None], 0.0) - self.p * g)
            far = np.where(np.isfinite(self.log_p), np.abs(self.log_p), 0.0) + 2 * np.abs(self.ls[:, None])
            p_rel = 6 * U * far + 4 * U + self.ls_bound[:, None]
            part = np.abs(b)[:, None] * (self.lp_bound + self.h_bound[:, None] + 3 * U * (far + np.abs(self.h[:, None])))
            size = np.abs(a)[:, None] + np.abs(b)[:, None] * (np.abs(log_p) + np.abs(self.h[:, None]))
            bound = self.scale * (self.p * (size * (p_rel + 6 * U) + part) + 3 * U * delta * np.abs(a)[:, None] + FLUSH * size)
        dx[self.skipped] = 0.0
        return dx, np.nan_to_num(bound)
