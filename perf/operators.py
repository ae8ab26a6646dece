"""Performance cases of the operators on points and gradients: layer normalization, attention to another sequence's
states, and the global norm of a list of gradients with its clipping.

A verification program runs them beside the set layers: it evaluates a network on points of an input box, follows
the gradient of a specification's margin back to the input (or to the weights, when the network is trained further on
the counterexamples it found), and bounds the step.  All tensors are torch tensors on the GPU.

A case is a dict of

    op      "norm", "norm_grad", "attend", "attend_grad" or "clip"
    type    "bf16", "f16" or "f32": the type of the inputs and of what is computed from them; row statistics, the
            logarithms of the softmax sums and the gradient norm are f32
  norm, norm_grad:
    rows, size      rows of ``size`` values
  attend, attend_grad:
    batch, queries, keys, heads, kv_heads, head
                    q is batch x queries x heads x head, k and v are batch x keys x kv_heads x head; kv_heads divides
                    heads, and heads / kv_heads consecutive heads share their keys and values
    cover           which keys count: "all", "lengths" (a length per sequence, between half of the keys and all of
                    them) or "mask" (truth values per sequence and key; one key in eight is left out)
  clip:
    tensors, most   so many tensors; the largest has ``most`` values, the others are spread below it
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
EPSILON = 1e-5


def _norm(name, op, type, rows, size):
    return dict({"op": op, "type": type, "rows": rows, "size": size}, **({"name": name} if name else {}))


def _attend(name, op, type, batch, queries, keys, heads, kv_heads, head, cover):
    c = {"op": op, "type": type, "batch": batch, "queries": queries, "keys": keys, "heads": heads, "kv_heads": kv_heads,
         "head": head, "cover": cover}
    return dict(c, name=name) if name else c


def _clip(name, type, tensors, most):
    return dict({"op": "clip", "type": type, "tensors": tensors, "most": most}, **({"name": name} if name else {}))


def listed():
    return [
        # one decoding step of a few sequences: latency
        _norm("norm_token", "norm", "bf16", 16, 1024),
        # a batch of long sequences in a wide model
        _norm("norm_wide", "norm", "bf16", 16384, 4096),
        # the backward pass over a batch of small images' patches, a width that is no power of two
        _norm("norm_grad_patches", "norm_grad", "f32", 12345, 768),
        # the backward pass of norm_wide's layer
        _norm("norm_grad_wide", "norm_grad", "bf16", 16384, 4096),
        # a decoder's pass over whole targets, encoder sequences padded to a common length
        _attend("attend_ragged", "attend", "bf16", 8, 448, 1500, 16, 16, 64, "lengths"),
        # long sequences on both sides, heads that share keys and values
        _attend("attend_long", "attend", "bf16", 2, 4096, 4096, 32, 8, 128, "all"),
        # one decoding step against cached encoder states
        _attend("attend_token", "attend", "bf16", 16, 1, 1500, 16, 16, 64, "lengths"),
        # one decoding step against a very long document, few sequences
        _attend("attend_token_long", "attend", "bf16", 2, 1, 65536, 32, 8, 128, "lengths"),
        # gradients at single precision with an odd head size, keys left out here and there
        _attend("attend_grad_odd", "attend_grad", "f32", 4, 333, 577, 12, 12, 80, "mask"),
        # the training step of attend_long
        _attend("attend_grad_long", "attend_grad", "bf16", 2, 4096, 4096, 32, 8, 128, "all"),
        # the gradients of one small block: latency
        _clip("clip_block", "f32", 16, 262144),
        # the gradients of a model of some hundred million weights
        _clip("clip_model", "bf16", 60, 1 << 24),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm; every other one as round as its size allows."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        step = 64 if n >= 256 else 8
        n = n // step * step
    return min(hi, max(lo, n))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "attend", "attend_grad", "token", "clip"])
    type = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("norm", "norm_grad"):
        while True:
            rows, size = _spread(rng, 1, 65536), _spread(rng, 64, 8192)
            if rows * size * BYTES[type] <= 16384 * 4096 * 2:
                return _norm(None, kind, type, rows, size)
    if kind == "clip":
        return _clip(None, type, rng.randint(1, 60), _spread(rng, 64, (1 << 25) // BYTES[type]))
    cover = rng.choice(["all", "lengths", "mask"])
    head = rng.choice([32, 40, 64, 64, 80, 96, 128, 128])
    group = rng.choice([1, 1, 2, 4, 8])
    if kind == "token":
        while True:
            batch, keys, kv_heads = _spread(rng, 1, 64), _spread(rng, 128, 65536), rng.choice([1, 2, 4, 8, 16])
            if batch * keys * kv_heads * head * BYTES[type] <= 2 * 65536 * 8 * 128 * 2:
                return _attend(None, "attend", type, batch, 1, keys, group * kv_heads, kv_heads, head, cover)
    most = 2 * 4096 * 4096 * 32 * 128 // (16 if type == "f32" or (type == "f16" and kind == "attend_grad") else 1)
    while True:
        batch, queries, keys = _spread(rng, 1, 16), _spread(rng, 2, 4096), _spread(rng, 16, 4096)
        kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
        if batch * queries * keys * group * kv_heads * head <= most and group * kv_heads <= 64:
            return _attend(None, kind, type, batch, queries, keys, group * kv_heads, kv_heads, head, cover)


# ---- inputs --------------------------------------------------------------------------------------------------


def _lengths(case):
    """The lengths of the sequences: the same numbers for every seed, so that the work is the same."""
    b, n = case["batch"], case["keys"]
    return [max(1, n - (n // 2) * i // b) for i in range(b)]


def _sizes(case):
    n, most = case["tensors"], case["most"]
    return [max(1, int(most * 2.0 ** (-(i % 8)) - 3 * i)) if i else most for i in range(n)]


def _counted_pairs(case):
    keys = sum(_lengths(case)) if case["cover"] == "lengths" else case["batch"] * case["keys"]
    return keys


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t = TYPES[case["type"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=None):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype or t)

    s = {"case": case}
    op = case["op"]
    if op in ("norm", "norm_grad"):
        rows, size = case["rows"], case["size"]
        # activations with a mean and an outlying channel, as they are between a model's blocks
        x = torch.randn(rows, size, generator=g, device="cuda") * 1.5 + 0.25
        x[:, size // 3] *= 8
        s["x"] = x.to(t)
        s["scale"], s["offset"] = normal(size, scale=0.2, shift=1.0), normal(size, scale=0.1)
        if op == "norm_grad":
            s["dy"] = normal(rows, size)
            _, s["mean"], s["rstd"] = _plain_norm(s["x"], s["scale"], s["offset"])
    elif op in ("attend", "attend_grad"):
        b, lq, lk, h, hkv, d = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "head"))
        s["q"] = normal(b, lq, h, d)
        s["k"], s["v"] = normal(b, lk, hkv, d), normal(b, lk, hkv, d)
        s["key_lengths"] = s["key_mask"] = None
        if case["cover"] == "lengths":
            order = torch.randperm(b, generator=g, device="cuda")
            s["key_lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")[order]
        elif case["cover"] == "mask":
            s["key_mask"] = torch.rand(b, lk, generator=g, device="cuda") >= 0.125
        if op == "attend_grad":
            s["do"] = normal(b, lq, h, d)
            s["o"], s["lse"] = _plain_attend(s)
    else:
        s["gradients"] = [normal(n, scale=0.02) for n in _sizes(case)]
        s["out"] = [torch.empty_like(x) for x in s["gradients"]]
        s["threshold"] = 1.0
    return s


# ---- the plain forms: 32 bits, rounded once at the end -------------------------------------------------------


def _plain_norm(x, scale, offset):
    f = x.float()
    mean = f.mean(-1)
    c = f - mean[:, None]
    rstd = torch.rsqrt((c * c).mean(-1) + EPSILON)
    return (c * rstd[:, None] * scale.float() + offset.float()).to(x.dtype), mean, rstd


def _plain_norm_grad(dy, x, mean, rstd, scale):
    g = dy.float()
    xhat = (x.float() - mean[:, None]) * rstd[:, None]
    w = g * scale.float()
    dx = (w - w.mean(-1, keepdim=True) - xhat * (w * xhat).mean(-1, keepdim=True)) * rstd[:, None]
    return dx.to(x.dtype), (g * xhat).sum(0).to(scale.dtype), g.sum(0).to(scale.dtype)


def _counts(s):
    """batch x keys truth values, or None where every key counts."""
    if s["key_mask"] is not None:
        return s["key_mask"]
    if s["key_lengths"] is not None:
        return torch.arange(s["k"].shape[1], device="cuda")[None, :] < s["key_lengths"][:, None]
    return None


def _by_kv_head(x, kv_heads):
    """batch x tokens x heads x head -> batch x kv_heads x (heads of the group * tokens) x head, f32."""
    b, n, h, d = x.shape
    return x.float().view(b, n, kv_heads, h // kv_heads, d).permute(0, 2, 3, 1, 4).reshape(b, kv_heads, h // kv_heads * n, d)


def _by_token(x, tokens):
    """The other way: batch x kv_heads x (group * tokens) x head -> batch x tokens x heads x head."""
    b, hkv, m, d = x.shape
    return x.view(b, hkv, m // tokens, tokens, d).permute(0, 3, 1, 2, 4).reshape(b, tokens, hkv * (m // tokens), d)


def _plain_weights(s):
    """(q, k, v by key/value head, exp(score - its row's largest), their sums, the largest scores)."""
    hkv, d = s["k"].shape[2], s["q"].shape[3]
    q, k, v = (_by_kv_head(x, hkv) for x in (s["q"], s["k"], s["v"]))
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * d ** -0.5
    counts = _counts(s)
    if counts is not None:
        scores.masked_fill_(~counts[:, None, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(scores.sub_(top))
    return q, k, v, p, p.sum(-1, keepdim=True), top


def _plain_attend(s):
    lq = s["q"].shape[1]
    q, k, v, p, total, top = _plain_weights(s)
    o = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
    lse = torch.log(total) + top
    b, h = s["q"].shape[0], s["q"].shape[2]
    return _by_token(o, lq).to(s["q"].dtype), lse.view(b, h, lq)


def _plain_attend_grad(s):
    lq, lk, hkv, d = s["q"].shape[1], s["k"].shape[1], s["k"].shape[2], s["q"].shape[3]
    q, k, v, p, total, _ = _plain_weights(s)
    p.div_(torch.where(total == 0, torch.ones_like(total), total))
    g = _by_kv_head(s["do"], hkv)
    dv = torch.matmul(p.transpose(2, 3), g)
    dp = torch.matmul(g, v.transpose(2, 3).contiguous())
    ds = p.mul_(dp - (p * dp).sum(-1, keepdim=True)).mul_(d ** -0.5)
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(2, 3), q)
    t = s["q"].dtype
    return _by_token(dq, lq).to(t), _by_token(dk, lk).to(t), _by_token(dv, lk).to(t)


def _plain_clip(gradients, threshold, out):
    norm = torch.stack([x.float().square().sum() for x in gradients]).sum().sqrt()
    factor = torch.where(norm > threshold, threshold / norm, torch.ones_like(norm))
    return [y.copy_(x.float() * factor) for x, y in zip(gradients, out)], norm


def run(state):
    s = state
    op = s["case"]["op"]
    if own:
        import nnv_amd as nnv
        if op == "norm":
            return nnv.layer_norm(s["x"], s["scale"], s["offset"], EPSILON)
        if op == "norm_grad":
            return nnv.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["scale"])
        if op == "attend":
            return nnv.cross_attention(s["q"], s["k"], s["v"], key_lengths=s["key_lengths"], key_mask=s["key_mask"])
        if op == "attend_grad":
            return nnv.cross_attention_backward(s["do"], s["q"], s["k"], s["v"], s["o"], s["lse"], key_lengths=s["key_lengths"],
                                                key_mask=s["key_mask"])
        return nnv.clip_gradients(s["gradients"], s["threshold"], out=s["out"])
    if op == "norm":
        return _plain_norm(s["x"], s["scale"], s["offset"])
    if op == "norm_grad":
        return _plain_norm_grad(s["dy"], s["x"], s["mean"], s["rstd"], s["scale"])
    if op == "attend":
        return _plain_attend(s)
    if op == "attend_grad":
        return _plain_attend_grad(s)
    return _plain_clip(s["gradients"], s["threshold"], s["out"])


def work(case):
    e, op = BYTES[case["type"]], case["op"]
    if op in ("norm", "norm_grad"):
        rows, size = case["rows"], case["size"]
        if op == "norm":
            return {"bytes": 2 * rows * size * e + 2 * size * e + 8 * rows, "flops": 8 * rows * size}
        return {"bytes": 3 * rows * size * e + 3 * size * e + 8 * rows, "flops": 14 * rows * size}
    if op in ("attend", "attend_grad"):
        b, lq, h, hkv, d = (case[k] for k in ("batch", "queries", "heads", "kv_heads", "head"))
        keys = _counted_pairs(case)                      # over all sequences
        rows, kv = b * lq * h, keys * hkv * d
        if op == "attend":
            return {"bytes": (2 * rows * d + 2 * kv) * e + 4 * rows, "flops": 4 * lq * h * d * keys}
        dkv = b * case["keys"] * hkv * d                 # the gradients of keys that do not count are written too
        return {"bytes": (4 * rows * d + 2 * kv + 2 * dkv) * e + 4 * rows, "flops": 10 * lq * h * d * keys}
    n = sum(_sizes(case))
    return {"bytes": 2 * n * e, "flops": 3 * n}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------


def _exact_sequence(s, i):
    """Attention of sequence i, one key/value head after the other: a generator of (heads of the group, the keys that
    count, q, k, v of them in 64 bits, weights, logarithms of the sums)."""
    n_keys, hkv, d = s["k"].shape[1], s["k"].shape[2], s["q"].shape[3]
    group = s["q"].shape[2] // hkv
    if s["key_mask"] is not None:
        at = s["key_mask"][i].nonzero()[:, 0]
    else:
        at = torch.arange(n_keys if s["key_lengths"] is None else int(s["key_lengths"][i]), device="cuda")
    for j in range(hkv):
        k, v = s["k"][i, at, j].double(), s["v"][i, at, j].double()
        for h in range(j * group, (j + 1) * group):
            q = s["q"][i, :, h].double()
            logits = (q @ k.T.contiguous()) / math.sqrt(d)
            lse = torch.logsumexp(logits, -1)
            yield h, j, at, q, k, v, torch.exp(logits - lse[:, None]), lse


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("norm", "norm_grad"):
        x, w = s["x"].double(), s["scale"].double()
        if op == "norm":
            var, mean = torch.var_mean(x, dim=1, unbiased=False)
            rstd = 1 / torch.sqrt(var + EPSILON)
            return (x - mean[:, None]) * rstd[:, None] * w + s["offset"].double(), mean, rstd
        # the gradient for the statistics that the forward pass handed on
        g, xhat = s["dy"].double(), (x - s["mean"].double()[:, None]) * s["rstd"].double()[:, None]
        gw, n = g * w, case["size"]
        dx = s["rstd"].double()[:, None] / n * (n * gw - gw.sum(1, keepdim=True) - xhat * (gw * xhat).sum(1, keepdim=True))
        return dx, (g * xhat).sum(0), g.sum(0)
    if op == "attend":
        o, lse = torch.zeros_like(s["q"], dtype=torch.float64), None
        b, lq, h, _ = s["q"].shape
        lse = torch.full((b, h, lq), -math.inf, dtype=torch.float64, device="cuda")
        for i in range(b):
            for h, _, at, q, k, v, p, logs in _exact_sequence(s, i):
                if len(at):
                    o[i, :, h], lse[i, h] = p @ v, logs
        return o, lse
    if op == "attend_grad":
        dq, dk, dv = (torch.zeros_like(s[x], dtype=torch.float64) for x in "qkv")
        for i in range(s["q"].shape[0]):
            for h, j, at, q, k, v, p, _ in _exact_sequence(s, i):
                if not len(at):
                    continue
                g = s["do"][i, :, h].double()
                dp = g @ v.T.contiguous()
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(q.shape[1])
                dq[i, :, h] = ds @ k
                dk[i, at, j] += ds.T.contiguous() @ q
                dv[i, at, j] += p.T.contiguous() @ g
        return dq, dk, dv
    norm = math.sqrt(sum(float((x.double() ** 2).sum()) for x in s["gradients"]))
    factor = s["threshold"] / norm if norm > s["threshold"] else 1.0
    return [x.double() * factor for x in s["gradients"]], torch.tensor(norm, dtype=torch.float64)
