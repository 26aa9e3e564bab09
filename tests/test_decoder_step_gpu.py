"""A training step of a small decoder layer made of the library's operators, as
they are used together: embedding, dropout, the first norm, attention with its
head norm, the joins of both blocks, the head and the log probabilities of the
next tokens with their entropy -- and back to every weight.  Against the same
step differentiated in float64."""

import numpy as np
import pytest
import torch

from _attention import put, table_of
from _layers import kept

pytestmark = pytest.mark.gpu

B, T, D, H, HK, DH, F, V = 2, 37, 96, 6, 2, 16, 160, 331
SEED, P, EPS, SCALE, COST = (7 << 33) + 5, 0.2, 1e-6, 0.9, 0.01


def weights():
    rng = np.random.default_rng(3)

    def normal(*shape, std, mean=0.0):
        return (rng.standard_normal(shape) * std + mean).astype(np.float32)

    return {"embed": normal(V, D, std=1.0), "w0": normal(D, std=0.1, mean=1.0), "qkv": normal((H + 2 * HK) * DH, D, std=D ** -0.5),
            "qw": normal(DH, std=0.1, mean=1.0), "kw": normal(DH, std=0.1, mean=1.0), "out": normal(D, H * DH, std=(H * DH) ** -0.5),
            "a1": normal(D, std=0.1, mean=1.0), "g1": normal(B, 1, D, std=0.2, mean=0.8), "w1": normal(D, std=0.1, mean=1.0),
            "up": normal(F, D, std=D ** -0.5), "down": normal(D, F, std=F ** -0.5), "a2": normal(D, std=0.1, mean=1.0),
            "g2": normal(D, std=0.2, mean=0.8), "w2": normal(D, std=0.1, mean=1.0), "head": normal(V, D, std=D ** -0.5)}


def inputs():
    rng = np.random.default_rng(4)
    ids, targets = rng.integers(0, V, (B, T)), rng.integers(0, V, (B, T))
    targets[1, 30:] = -100  # the second sequence is shorter
    return ids, targets


def step64(w, ids, targets):
    """(loss, gradients) in float64 on the host."""
    t = {n: torch.from_numpy(x).double().requires_grad_() for n, x in w.items()}
    drop = [torch.from_numpy(kept(P, SEED, (B, T, D), i)) for i in range(3)]

    def norm(x, weight):
        return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * weight

    def dropped(x, i):
        return torch.where(drop[i], x / (1 - P), 0.0)

    def turned(x):  # [B, T, heads, DH], halves
        row = torch.from_numpy(table_of(T, DH)).double()[None, :, None]
        c, s, a, b = row[..., : DH // 2], row[..., DH // 2:], x[..., : DH // 2], x[..., DH // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    x = dropped(t["embed"][torch.from_numpy(ids)], 0)
    packed = norm(x, t["w0"]) @ t["qkv"].T
    q, k, v = (packed.view(B, T, H + 2 * HK, DH)[:, :, a:b] for a, b in ((0, H), (H, H + HK), (H + HK, H + 2 * HK)))
    q, k = turned(norm(q, t["qw"])), turned(norm(k, t["kw"]))
    k, v = (m.repeat_interleave(H // HK, 2) for m in (k, v))
    scores = torch.einsum("bihd,bjhd->bhij", q, k) * DH ** -0.5
    scores = scores.masked_fill(torch.ones(T, T).triu(1).bool(), -torch.inf)
    y = torch.einsum("bhij,bjhd->bihd", scores.softmax(-1), v).reshape(B, T, H * DH) @ t["out"].T
    x = 0.9 * x + 0.5 * t["g1"] * dropped(norm(y, t["a1"]), 1)
    y = torch.nn.functional.silu(norm(x, t["w1"]) @ t["up"].T) @ t["down"].T
    x = x + t["g2"] * dropped(norm(y, t["a2"]), 2)
    log_p = torch.log_softmax(SCALE * (norm(x, t["w2"]) @ t["head"].T), -1)
    used = torch.from_numpy(targets != -100)
    lp = log_p.gather(-1, torch.from_numpy(targets).clamp(min=0)[..., None])[..., 0]
    entropy = -(log_p.exp() * log_p).sum(-1)
    loss = -((lp + COST * entropy) * used).sum() / used.sum()
    names = list(t)
    return loss.item(), dict(zip(names, torch.autograd.grad(loss, [t[n] for n in names])))


def step(ops, w, ids, targets):
    d = {n: put(x) for n, x in w.items()}
    table, positions, t = put(table_of(T, DH)), put(np.arange(T)), put(targets)
    used = int((targets != -100).sum())

    def rows(x):
        return x.view(B * T, x.shape[-1])

    def back(dy, x, weight):  # of linear: (dx, dweight)
        return ops.matmul(dy, d[weight]), ops.mm(rows(dy).t(), rows(x))

    e = ops.embedding(d["embed"], put(ids))
    x0 = ops.seeded_dropout(e, P, SEED)
    _, h0, _, r0 = ops.residual_norm(x0, weight=d["w0"], eps=EPS)
    packed = ops.linear(h0, d["qkv"]).view(B, T, H + 2 * HK, DH)
    q, k, v = packed[:, :, :H], packed[:, :, H: H + HK], packed[:, :, H + HK:]
    qt, kt, qr, kr = ops.qk_norm_rope(q, k, table, positions, d["qw"], d["kw"], EPS)
    o, lse = ops.sliding_window_attention(qt, kt, v)
    y1 = ops.linear(o.view(B, T, H * DH), d["out"])
    x1, h1, b1, r1 = ops.residual_norm(x0, y1, d["g1"], d["a1"], d["w1"], 0.9, 0.5, EPS, EPS, P, SEED, 1)
    u = ops.linear(h1, d["up"])
    s = ops.silu(u)
    y2 = ops.linear(s, d["down"])
    x2, h2, b2, r2 = ops.residual_norm(x1, y2, d["g2"], d["a2"], d["w2"], 1.0, 1.0, EPS, EPS, P, SEED, 2)
    logits = ops.linear(h2, d["head"])
    lp, entropy, stats, best, best_ids = ops.token_log_probs(logits, t, SCALE, top=3)
    loss = -float((lp.numpy().astype(np.float64) + COST * entropy.numpy()).sum()) / used

    g = {}
    dlogits = ops.token_log_probs_backward(put(np.full((B, T), -1.0 / used, np.float32)), put(np.full((B, T), -COST / used, np.float32)),
                                           logits, t, stats, entropy, SCALE)
    dh2, g["head"] = back(dlogits, h2, "head")
    dx1, dy2, g["g2"], g["a2"], g["w2"] = ops.residual_norm_backward(None, dh2, x1, y2, b2, r2, d["g2"], d["a2"], d["w2"], p=P, seed=SEED,
                                                                     offset=2)
    ds, g["down"] = back(dy2, s, "down")
    dh1, g["up"] = back(ops.silu_backward(ds, u), h1, "up")
    dx0, dy1, g["g1"], g["a1"], g["w1"] = ops.residual_norm_backward(dx1, dh1, x0, y1, b1, r1, d["g1"], d["a1"], d["w1"], 0.9, 0.5, P, SEED, 1)
    do, g["out"] = back(dy1, o.view(B, T, H * DH), "out")
    dqt, dkt, dv = ops.sliding_window_attention_backward(do.view(B, T, H, DH), qt, kt, v, o, lse)
    dq, dk, g["qw"], g["kw"] = ops.qk_norm_rope_backward(dqt, dkt, q, k, table, positions, qr, kr, d["qw"], d["kw"])
    dpacked = ops.empty((B, T, H + 2 * HK, DH))
    for part, grad in ((dpacked[:, :, :H], dq), (dpacked[:, :, H: H + HK], dk), (dpacked[:, :, H + HK:], dv)):
        ops.copy_(part, grad)
    dh0, g["qkv"] = back(dpacked.view(B, T, (H + 2 * HK) * DH), h0, "qkv")
    # the residual flows on beside its norm
    dx0, _, _, _, g["w0"] = ops.residual_norm_backward(dx0, dh0, x0, rstd=r0, weight=d["w0"])
    g["embed"] = ops.embedding_dense_backward(ops.seeded_dropout_backward(dx0, P, SEED), put(ids), V)
    return loss, {n: x.numpy() for n, x in g.items()}, (lp.numpy(), best.numpy(), best_ids.numpy())


def test_step_against_float64(dev, ops):
    """About 24 operators in a row, each of which is off by at most a few dozen
    u = 2^-24 of its result's norm: 24 x 70 u = 1e-4."""
    w, (ids, targets) = weights(), inputs()
    want_loss, want = step64(w, ids, targets)
    loss, grads, (lp, best, best_ids) = step(ops, w, ids, targets)
    assert abs(loss - want_loss) < 1e-4 * abs(want_loss)
    assert set(grads) == set(want)
    for n, g in grads.items():
        x = want[n].numpy()
        assert g.shape == x.shape
        assert np.linalg.norm(g - x) < 1e-4 * np.linalg.norm(x), n
    used = targets != -100
    assert (lp[~used] == 0).all() and (best_ids[~used] == -1).all()
    # a target among the alternatives has their log probability
    rank = best_ids == targets[..., None]
    assert np.array_equal(best[rank & used[..., None]], np.broadcast_to(lp[..., None], rank.shape)[rank & used[..., None]])
