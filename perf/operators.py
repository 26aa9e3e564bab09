"""Performance cases of the attention layer's operators: the norm and position
rotation of each head's query and key, and causal attention with a sliding
window and a few first tokens that stay visible, in training and in serving.

A pass calls the public operators of the package's ``ops`` (``own`` true) or
computes the same in elementary torch operations in float32 (``own`` false)
and returns every result whole: forward results, saved statistics, gradients.
Inputs are torch tensors the operators read in place; results come back as
torch views of the library's own memory, alive until the state's next pass.

``work`` counts each input read once and each result written once (of a
cache: the keys and values some query sees), and two operations per
multiply-add of the products over the visible pairs of query and key.

Kinds of case, and what each stands for:

rope            queries and keys of a packed projection normed and rotated on
                their way to attention (prompt, or one token a sequence)
rope_train      the same in a training step: forward and backward, gradients
                of both norms' weights among the results
prefill         attention of a prompt, or of a chunk of one behind the tokens
                that a cache holds already; a padded batch has its lengths
train           attention of a training step, forward and backward
decode          one new token (or a few drafted ones) a sequence against a
                cache filled to different lengths
"""

from __future__ import annotations

import importlib
import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
EPS = 1e-6


# ---- the cases -----------------------------------------------------------------


def listed():
    return [
        # One new token for each of eight sequences: bound by latency.
        {"name": "rope_decode_8x1", "kind": "rope", "batch": 8, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "far": 131072, "dtype": "bfloat16"},
        # A long prompt of a model with the benchmark's 4096-wide layers.
        {"name": "rope_prompt_1x8192", "kind": "rope", "batch": 1, "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "far": 32768, "dtype": "bfloat16"},
        # A training batch of the same layer.
        {"name": "rope_train_4x2048", "kind": "rope_train", "batch": 4, "tokens": 2048, "heads": 32, "kv_heads": 8,
         "dim": 128, "rotary": 128, "interleaved": False, "far": 2048, "dtype": "bfloat16"},
        # A small model in float32 on a ragged number of tokens, rotating a part of each head in neighbouring pairs.
        {"name": "rope_train_1x3001_f32", "kind": "rope_train", "batch": 1, "tokens": 3001, "heads": 12, "kv_heads": 12,
         "dim": 80, "rotary": 40, "interleaved": True, "far": 4096, "dtype": "float32"},
        # One token of one sequence, its window full: bound by latency.
        {"name": "decode_1x1_w1024", "kind": "decode", "batch": 1, "queries": 1, "keys": 4096, "heads": 32, "kv_heads": 8,
         "dim": 128, "window": 1024, "sinks": 4, "dtype": "bfloat16"},
        # Many sequences over long caches without a window: bound by the cache's bytes.
        {"name": "decode_64x1_16384", "kind": "decode", "batch": 64, "queries": 1, "keys": 16384, "heads": 32, "kv_heads": 8,
         "dim": 128, "window": -1, "sinks": 0, "dtype": "bfloat16"},
        # Four drafted tokens a sequence to verify, in float16, heads of an odd multiple of 16.
        {"name": "decode_16x4_w2000", "kind": "decode", "batch": 16, "queries": 4, "keys": 5001, "heads": 24, "kv_heads": 4,
         "dim": 80, "window": 2000, "sinks": 8, "dtype": "float16"},
        # A long prompt under a window.
        {"name": "prefill_1x8192_w1024", "kind": "prefill", "batch": 1, "queries": 8192, "keys": 8192, "heads": 32,
         "kv_heads": 8, "dim": 128, "window": 1024, "sinks": 4, "padded": False, "dtype": "bfloat16"},
        # A padded batch of prompt chunks behind what their caches hold.
        {"name": "prefill_4x777_chunk", "kind": "prefill", "batch": 4, "queries": 777, "keys": 4001, "heads": 16,
         "kv_heads": 4, "dim": 96, "window": 1500, "sinks": 16, "padded": True, "dtype": "float16"},
        # The benchmark's batched products as the attention they come from, all earlier tokens visible.
        {"name": "train_1x512_64heads", "kind": "train", "batch": 1, "queries": 512, "keys": 512, "heads": 64,
         "kv_heads": 64, "dim": 128, "window": -1, "sinks": 0, "dtype": "bfloat16"},
        # A training batch of the 4096-wide layer under a window.
        {"name": "train_2x4096_w1024", "kind": "train", "batch": 2, "queries": 4096, "keys": 4096, "heads": 32,
         "kv_heads": 8, "dim": 128, "window": 1024, "sinks": 4, "dtype": "bfloat16"},
        # A small model in float32 on a ragged number of tokens.
        {"name": "train_1x1001_f32", "kind": "train", "batch": 1, "queries": 1001, "keys": 1001, "heads": 12,
         "kv_heads": 12, "dim": 64, "window": 256, "sinks": 1, "dtype": "float32"},
    ]


def draw(rng):
    def size(low, high, step=1):
        """Log-uniform in [low, high]; half of them a multiple of ``step``."""
        n = math.exp(rng.uniform(math.log(low), math.log(high)))
        if step > 1 and rng.random() < 0.5:
            n = step * max(1, round(n / step))
        return int(min(high, max(low, round(n))))

    kind = rng.choice(["rope", "rope_train", "prefill", "train", "decode"])
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    heads = kv_heads * rng.choice([1, 1, 2, 4, 6, 8])
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": rng.choice([64, 64, 80, 96, 128, 128]),
            "dtype": rng.choice(["bfloat16", "bfloat16", "float16", "float32"])}
    if kind in ("rope", "rope_train"):
        case["batch"] = size(1, 64)
        most = (1 << 18) // (heads + kv_heads)  # rows of one batch entry at most
        case["tokens"] = size(1, max(1, min(8192, most // case["batch"] * 4)), 64)
        case["rotary"] = rng.choice([case["dim"], case["dim"], case["dim"] // 2])
        case["interleaved"] = rng.random() < 0.4
        case["far"] = max(case["tokens"], rng.choice([4096, 32768, 131072]))
        return case
    case["window"] = rng.choice([-1, size(16, 8192, 64), size(16, 4096, 64)])
    case["sinks"] = 0 if case["window"] < 0 else rng.choice([0, 1, 4, size(1, 200)])
    if kind == "decode":
        case["batch"] = size(1, 128)
        case["queries"] = rng.choice([1, 1, 1, 2, size(1, 16)])
        bytes_of = 2 * kv_heads * case["dim"] * (4 if case["dtype"] == "float32" else 2)
        case["keys"] = max(case["queries"], size(64, max(64, min(65536, (2 << 30) // (case["batch"] * bytes_of))), 64))
        return case
    case["batch"] = size(1, 8)
    # scores of the plain form, and so its time and memory
    most = int(math.sqrt((1 << (28 if kind == "train" else 29)) / (case["batch"] * heads)))
    case["queries"] = size(16, max(16, min(8192, most)), 64)
    if kind == "train":
        case["keys"] = case["queries"]
    else:
        case["keys"] = case["queries"] + rng.choice([0, size(1, 4096)])
        case["padded"] = rng.random() < 0.5
    return case


def _lengths(case):
    """Keys each sequence holds: the first all of them, the others evenly fewer, never less than its queries."""
    b, n, q = case["batch"], case["keys"], case["queries"]
    if case["kind"] == "train" or (case["kind"] == "prefill" and not case["padded"]):
        return [n] * b
    return [max(min(q, n), n - (n * i) // (2 * b)) for i in range(b)]


# ---- inputs -----------------------------------------------------------------------


def _inputs(case, seed):
    """The case's inputs as torch tensors on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0):
        # in slices: a cache's float32 draw would be twice its size
        out = torch.empty(shape, dtype=dtype, device="cuda")
        for part in out if len(shape) > 1 else [out]:
            part.copy_(torch.randn(part.shape, generator=g, device="cuda").mul_(scale).add_(shift))
        return out

    b, h, hk, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] in ("rope", "rope_train"):
        t, r, far = case["tokens"], case["rotary"], case["far"]
        angle = torch.arange(far, dtype=torch.float64)[:, None] * 10000.0 ** -(torch.arange(r // 2, dtype=torch.float64) * 2 / r)
        table = torch.cat([angle.cos(), angle.sin()], 1).float().cuda()
        first = torch.randint(far - t + 1, (b, 1), generator=g, device="cuda")
        packed = normal(b, t, (h + 2 * hk) * d)  # the projection's output: queries, keys, values
        out = {"packed": packed, "table": table, "positions": first + torch.arange(t, device="cuda"),
               "qw": normal(d, scale=0.1, shift=1.0), "kw": normal(d, scale=0.1, shift=1.0)}
        if case["kind"] == "rope_train":
            out.update(dq=normal(b, t, h, d), dk=normal(b, t, hk, d))
        return out
    tq, tk = case["queries"], case["keys"]
    out = {"q": normal(b, tq, h, d), "k": normal(b, tk, hk, d), "v": normal(b, tk, hk, d)}
    if case["kind"] == "train":
        out["do"] = normal(b, tq, h, d)
    else:
        out["lengths"] = torch.tensor(_lengths(case), dtype=torch.int64, device="cuda")
    return out


def _split(case, packed):
    """Queries and keys as views of the packed projection."""
    b, t = packed.shape[:2]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    return packed[:, :, : h * d].view(b, t, h, d), packed[:, :, h * d: (h + hk) * d].view(b, t, hk, d)


class _State:
    def __init__(self, case, inputs):
        self.case = case
        self.torch = inputs
        if own:
            self.package = _Package()
            if "packed" in inputs:
                self.q, self.k = (self.package.device(x) for x in _split(case, inputs["packed"]))
            for name, value in inputs.items():
                setattr(self, name, self.package.device(value))


class _Package:
    """The package's modules, and tensors handed to it and back."""

    def __init__(self):
        self.tensor = importlib.import_module("tensorplay-mlu_amd.tensor")
        self.abi = importlib.import_module("tensorplay-mlu_amd._abi")
        self.ops = importlib.import_module("tensorplay-mlu_amd.ops")
        self.codes = {torch.float32: self.abi.FLOAT32, torch.float16: self.abi.FLOAT16,
                      torch.bfloat16: self.abi.BFLOAT16, torch.int64: self.abi.INT64}
        self.types = {self.abi.FLOAT32: ("<f4", None), self.abi.FLOAT16: ("<f2", None),
                      self.abi.BFLOAT16: ("<i2", torch.bfloat16)}
        self.held = None
        self.views = {}

    def device(self, t):
        """The operators' view of a torch tensor's memory."""
        ref = self.abi.Tensor()
        ref.data, ref.ctx, ref.ndim = t.data_ptr(), None, t.dim()
        for i in range(t.dim()):
            ref.sizes[i], ref.strides[i] = t.shape[i], t.stride(i)
        ref.dtype, ref.device = self.codes[t.dtype], 0
        return self.tensor.DeviceTensor(ref, owner=t)

    def hand_back(self, results):
        """torch views of the results' memory, which lives until the next
        pass.  A view is made once for each place."""
        out = []
        for d in results:
            key = (d.data_ptr, d.shape, d.dtype)
            if key not in self.views:
                self.views[key] = self._view(d)
            out.append(self.views[key])
        self.held = results
        return out

    def _view(self, d):
        typestr, dtype = self.types[d.dtype]

        class Memory:
            __cuda_array_interface__ = {"shape": d.shape, "typestr": typestr, "version": 2,
                                        "data": (d.data_ptr, False), "strides": None}

        t = torch.as_tensor(Memory(), device="cuda")
        return t if dtype is None else t.view(dtype)


def prepare(case, seed):
    state = _State(dict(case), _inputs(case, seed))
    torch.cuda.synchronize()  # the operators run on a stream of their own
    return state


# ---- one pass ---------------------------------------------------------------------


def run(state):
    return _RUN[state.case["kind"]](state)


def _rope(s):
    c, t = s.case, s.torch
    if own:
        return s.package.hand_back(s.package.ops.qk_norm_rope(s.q, s.k, s.table, s.positions, s.qw, s.kw, EPS, c["interleaved"]))
    q, k = _split(c, t["packed"])
    (qo, qr), (ko, kr) = (_plain_rope(c, x, w, t) for x, w in ((q, t["qw"]), (k, t["kw"])))
    return [qo, ko, qr, kr]


def _rope_train(s):
    c, t = s.case, s.torch
    if own:
        ops = s.package.ops
        qo, ko, qr, kr = ops.qk_norm_rope(s.q, s.k, s.table, s.positions, s.qw, s.kw, EPS, c["interleaved"])
        grads = ops.qk_norm_rope_backward(s.dq, s.dk, s.q, s.k, s.table, s.positions, qr, kr, s.qw, s.kw, c["interleaved"])
        return s.package.hand_back([qo, ko, qr, kr, *grads])
    q, k = _split(c, t["packed"])
    (qo, qr), (ko, kr) = (_plain_rope(c, x, w, t) for x, w in ((q, t["qw"]), (k, t["kw"])))
    (dq, dqw), (dk, dkw) = (_plain_rope_backward(c, dy, x, r, w, t) for dy, x, r, w in
                            ((t["dq"], q, qr, t["qw"]), (t["dk"], k, kr, t["kw"])))
    return [qo, ko, qr, kr, dq, dk, dqw, dkw]


def _pairs(case, x):
    """The two elements of every rotated pair, and the rest."""
    r = case["rotary"]
    rot, rest = x[..., :r], x[..., r:]
    if case["interleaved"]:
        return rot[..., 0::2], rot[..., 1::2], rest
    return rot[..., : r // 2], rot[..., r // 2:], rest


def _joined(case, a, b, rest):
    rot = torch.stack([a, b], -1).flatten(-2) if case["interleaved"] else torch.cat([a, b], -1)
    return torch.cat([rot, rest], -1)


def _cos_sin(case, t):
    row = t["table"][t["positions"]][:, :, None, :]
    return row[..., : case["rotary"] // 2], row[..., case["rotary"] // 2:]


def _plain_rope(case, x, w, t):
    x32 = x.float()
    r = torch.rsqrt((x32 * x32).mean(-1) + EPS)
    a, b, rest = _pairs(case, x32 * r[..., None] * w.float())
    cos, sin = _cos_sin(case, t)
    return _joined(case, a * cos - b * sin, b * cos + a * sin, rest).to(x.dtype), r


def _plain_rope_backward(case, dy, x, r, w, t):
    x32 = x.float()
    cos, sin = _cos_sin(case, t)
    a, b, rest = _pairs(case, dy.float())
    g = _joined(case, a * cos + b * sin, b * cos - a * sin, rest)
    n = x32 * r[..., None]
    u = g * w.float()
    dx = r[..., None] * (u - n * (u * n).mean(-1, keepdim=True))
    return dx.to(x.dtype), (g * n).sum((0, 1, 2)).to(x.dtype)


def _attention(s):
    c, t = s.case, s.torch
    if own:
        return s.package.hand_back(s.package.ops.sliding_window_attention(
            s.q, s.k, s.v, c["window"], c["sinks"], lengths=s.lengths))
    out = [_plain_attention(c, b, n, t) for b, n in enumerate(_lengths(c))]
    return [torch.stack([o for o, _, _ in out]), torch.stack([l for _, l, _ in out])]


def _train(s):
    c, t = s.case, s.torch
    if own:
        ops = s.package.ops
        out, lse = ops.sliding_window_attention(s.q, s.k, s.v, c["window"], c["sinks"])
        grads = ops.sliding_window_attention_backward(s.do, s.q, s.k, s.v, out, lse, c["window"], c["sinks"])
        return s.package.hand_back([out, lse, *grads])
    every = []
    for b in range(c["batch"]):
        o, lse, p = _plain_attention(c, b, c["keys"], t)
        every.append((o, lse, *_plain_attention_backward(c, b, p, t)))
    return [torch.stack(list(x)) for x in zip(*every)]


def _visible(case, length, device):
    """[queries, keys]: which keys the last ``queries`` of ``length`` tokens see."""
    p = torch.arange(length - case["queries"], length, device=device)[:, None]
    j = torch.arange(length, device=device)[None, :]
    near = j <= p
    if case["window"] >= 0:
        near &= (j > p - case["window"]) | (j < case["sinks"])
    return near


def _heads_first(x, repeat=1):
    """[tokens, heads, dim] -> float32 [heads * repeat, tokens, dim], dense."""
    x = x.float().transpose(0, 1)
    return x.repeat_interleave(repeat, 0).contiguous()


def _plain_attention(case, b, length, t):
    group, scale = case["heads"] // case["kv_heads"], case["dim"] ** -0.5
    q = _heads_first(t["q"][b])
    k, v = (_heads_first(t[n][b, :length], group) for n in ("k", "v"))
    scores = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(scale)
    scores.masked_fill_(~_visible(case, length, q.device), -math.inf)
    m = scores.amax(-1, keepdim=True)
    p = scores.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(total)
    out = torch.bmm(p, v).transpose(0, 1).to(t["q"].dtype)
    return out.contiguous(), (m + total.log())[..., 0], p


def _plain_attention_backward(case, b, p, t):
    hk, scale = case["kv_heads"], case["dim"] ** -0.5
    group = case["heads"] // hk
    q, do = _heads_first(t["q"][b]), _heads_first(t["do"][b])
    k, v = (_heads_first(t[n][b], group) for n in ("k", "v"))
    pt = p.transpose(1, 2).contiguous()
    dv = torch.bmm(pt, do)
    dp = torch.bmm(do, v.transpose(1, 2).contiguous())
    ds = dp.sub_((p * dp).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.bmm(ds, k)
    dk = torch.bmm(ds.transpose(1, 2).contiguous(), q)

    def shared(x):  # the query heads of one key head add up
        return x.view(hk, group, *x.shape[1:]).sum(1)

    return [x.transpose(0, 1).to(t["q"].dtype).contiguous() for x in (dq, shared(dk), shared(dv))]


_RUN = {"rope": _rope, "rope_train": _rope_train, "prefill": _attention, "decode": _attention, "train": _train}


# ---- what a pass cannot do without ---------------------------------------------------


def _seen(case, length):
    """(visible pairs of query and key, keys that some query sees) of one sequence."""
    w, s = case["window"], case["sinks"]
    pairs, first = 0, length - case["queries"]
    for p in range(first, length):
        pairs += p + 1 if w < 0 else min(p + 1, w) + min(s, max(0, p + 1 - w))
    low = 0 if w < 0 else max(0, first - w + 1)
    return pairs, length - low + min(s, low)


def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] in ("rope", "rope_train"):
        tokens = case["batch"] * case["tokens"]
        rows = tokens * (h + hk)
        used = min(tokens, case["far"]) * case["rotary"] * 4 + tokens * 8 + 2 * d * e
        if case["kind"] == "rope":
            return {"bytes": 2 * rows * d * e + 4 * rows + used, "flops": 7 * rows * d}
        return {"bytes": 5 * rows * d * e + 8 * rows + 2 * used + 2 * d * e, "flops": 22 * rows * d}
    pairs = keys = 0
    for n in _lengths(case):
        a, b = _seen(case, n)
        pairs, keys = pairs + a, keys + b
    queries = case["batch"] * case["queries"]
    q, kv = queries * h * d * e, keys * hk * d * e
    if case["kind"] == "train":
        # forward q, k, v, o, lse; backward q, k, v, o, lse, do, and three gradients
        return {"bytes": 2 * q + 2 * kv + 4 * queries * h + 4 * q + 4 * kv + 4 * queries * h, "flops": 14 * pairs * h * d}
    return {"bytes": 2 * q + 2 * kv + 4 * queries * h, "flops": 4 * pairs * h * d}


# ---- the definition in 64 bits -----------------------------------------------------


def exact(case, seed):
    """The results of a pass from the operators' definition in float64: the
    norm and rotation as a complex product, attention as one query head at a
    time over the keys it sees, gradients by differentiating that."""
    t = _inputs(case, seed)
    with torch.enable_grad():
        if case["kind"] in ("rope", "rope_train"):
            return _exact_rope(case, t)
        return _exact_attention(case, t)


def _exact_rope(case, t):
    r, inter = case["rotary"], case["interleaved"]
    row = t["table"].double()[t["positions"]].unsqueeze(2)
    turn = torch.complex(row[..., : r // 2], row[..., r // 2:])
    outs, stats, grads, dws = [], [], [], []
    for part, (x, w) in enumerate(zip(_split(case, t["packed"]), (t["qw"], t["kw"]))):
        x64 = x.double().requires_grad_()
        w64 = w.double().requires_grad_()
        rms = (x64.pow(2).sum(-1) / case["dim"] + EPS).sqrt()
        n = x64 / rms.unsqueeze(-1) * w64
        z = n[..., :r].unflatten(-1, (r // 2, 2) if inter else (2, r // 2))
        z = torch.complex(z[..., 0], z[..., 1]) if inter else torch.complex(z[..., 0, :], z[..., 1, :])
        z = torch.view_as_real(z * turn)
        y = torch.cat([(z if inter else z.transpose(-1, -2)).flatten(-2), n[..., r:]], -1)
        outs.append(y.detach())
        stats.append((1.0 / rms).detach())
        if case["kind"] == "rope_train":
            dx, dw = torch.autograd.grad(y, (x64, w64), t["dk" if part else "dq"].double())
            grads.append(dx)
            dws.append(dw)
    return outs + stats + grads + dws


def _exact_attention(case, t):
    train = case["kind"] == "train"
    names = ("q", "k", "v") + (("do",) if train else ())
    group, tq = case["heads"] // case["kv_heads"], case["queries"]
    shape = t["q"].shape
    out = torch.zeros(shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(shape[0], shape[2], tq, dtype=torch.float64, device="cuda")
    grads = [torch.zeros(t[n].shape, dtype=torch.float64, device="cuda") for n in ("q", "k", "v")]
    step = 2048  # queries at a time
    for b, n in enumerate(_lengths(case)):
        for h in range(case["heads"]):
            for i0 in range(0, tq, step):
                i1 = min(tq, i0 + step)
                p = n - tq + torch.arange(i0, i1, device="cuda")
                low = 0 if case["window"] < 0 else max(0, int(n - tq + i0 - case["window"] + 1))
                j = torch.arange(low, n - tq + i1, device="cuda")
                if low:  # the first tokens, then the window's
                    j = torch.cat([torch.arange(min(case["sinks"], low), device="cuda"), j])
                seen = j[None] <= p[:, None]
                if case["window"] >= 0:
                    seen &= (j[None] < case["sinks"]) | (p[:, None] - j[None] < case["window"])
                q = t["q"][b, i0:i1, h].double().requires_grad_(train)
                k, v = (t[m][b, :, h // group].index_select(0, j).double().requires_grad_(train) for m in ("k", "v"))
                s = (q @ k.T) / math.sqrt(case["dim"])
                s = torch.where(seen, s, torch.full_like(s, -math.inf))
                total = torch.logsumexp(s, 1)
                o = torch.softmax(s, 1) @ v
                out[b, i0:i1, h], lse[b, h, i0:i1] = o.detach(), total.detach()
                if train:
                    dq, dk, dv = torch.autograd.grad(o, (q, k, v), t[names[3]][b, i0:i1, h].double())
                    grads[0][b, i0:i1, h] = dq
                    grads[1][b, :, h // group].index_add_(0, j, dk)
                    grads[2][b, :, h // group].index_add_(0, j, dv)
    return [out, lse] + (grads if train else [])
