"""Performance cases of the operators on points that are images and videos: group normalization with an activation over
features whose channels come last, rotary positions with several axes, and differential attention.

A program that evaluates a network with such layers on points of an input box, and follows gradients back to the input or
to the weights, runs them beside the set layers.  All tensors are torch tensors on the GPU.

A case is a dict of

    op      "group", "group_grad", "rotate", "differ" or "differ_grad"
    type    "bf16", "f16" or "f32": the type of the inputs and of what is computed from them; the statistics of the
            normalization and the logarithms of the softmax sums are f32
  group, group_grad:
    batch, height, width, channels, groups
                    x is batch x height x width x channels
    activation      "none", "relu" or "silu"
  rotate:
    batch, tokens, heads, head, kv_heads
                    two tensors, batch x tokens x heads x head and batch x tokens x kv_heads x head, as queries and keys are
    sections        pairs of values that each axis of the positions turns, as text "16,24,24"
    shared          whether the axes share one list of frequencies, or have one each
    interleaved     whether a pair are neighbours, or one value of either half
    inverse         turned back, as in the backward pass
  differ, differ_grad:
    batch, queries, keys, heads, kv_heads, head
                    q is batch x queries x 2 heads x head (the two maps of a head follow one another), k is batch x keys x
                    2 kv_heads x head, v is batch x keys x kv_heads x 2 head; heads / kv_heads consecutive heads share keys
                    and values
    cover           which keys count: "all", "lengths" (a length per sequence, between half of the keys and all of
                    them) or "mask" (truth values per sequence and key; one key in eight is left out)
    causal          whether a query sees the keys up to its own place alone, the last query's being the last key's
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
EPSILON = 1e-5
BASE = 10000.0


def _named(name, **c):
    return dict(c, name=name) if name else c


def _group(name, op, type, batch, height, width, channels, groups, activation):
    return _named(name, op=op, type=type, batch=batch, height=height, width=width, channels=channels, groups=groups, activation=activation)


def _rotate(name, type, batch, tokens, heads, kv_heads, head, sections, shared=False, interleaved=False, inverse=False):
    return _named(name, op="rotate", type=type, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, head=head, sections=sections,
                  shared=shared, interleaved=interleaved, inverse=inverse)


def _differ(name, op, type, batch, queries, keys, heads, kv_heads, head, cover, causal):
    return _named(name, op=op, type=type, batch=batch, queries=queries, keys=keys, heads=heads, kv_heads=kv_heads, head=head, cover=cover,
                  causal=causal)


def listed():
    return [
        # a late, small stage of an image network, a few points: latency
        _group("group_small", "group", "bf16", 4, 8, 8, 256, 32, "silu"),
        # an early stage of an image network over a batch; ten channels a group
        _group("group_image", "group", "bf16", 16, 64, 64, 320, 32, "silu"),
        # the training step of group_image's layer
        _group("group_grad_image", "group_grad", "bf16", 16, 64, 64, 320, 32, "silu"),
        # the gradient search at single precision on images of odd sizes
        _group("group_grad_odd", "group_grad", "f32", 5, 53, 79, 96, 8, "relu"),
        # one new token of a few sequences: latency
        _rotate("rotate_token", "bf16", 16, 1, 32, 8, 128, "16,24,24", shared=True),
        # a video of 8 x 40 x 60 places, positions of time, row and column
        _rotate("rotate_video", "bf16", 2, 19200, 24, 8, 128, "16,24,24", shared=True),
        # the backward pass over images' patches, rows and columns with frequencies of their own, a head that is partly turned
        _rotate("rotate_back_odd", "f32", 3, 1577, 12, 12, 80, "16,16", interleaved=True, inverse=True),
        # one new token of some sequences against cached keys
        _differ("differ_token", "differ", "bf16", 16, 1, 8000, 16, 4, 64, "lengths", True),
        # images' patches at half precision, sequences padded to a common length
        _differ("differ_ragged", "differ", "f16", 8, 577, 1000, 12, 12, 40, "lengths", False),
        # long sequences of wide heads that share keys and values
        _differ("differ_long", "differ", "bf16", 2, 4096, 4096, 16, 4, 128, "all", True),
        # gradients at single precision with an odd head size, keys left out here and there
        _differ("differ_grad_odd", "differ_grad", "f32", 4, 333, 577, 6, 6, 40, "mask", False),
        # a training step over long sequences
        _differ("differ_grad_long", "differ_grad", "bf16", 2, 4096, 4096, 16, 4, 64, "all", True),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm; every other one as round as its size allows."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        step = 64 if n >= 256 else 8
        n = n // step * step
    return min(hi, max(lo, n))


def draw(rng):
    kind = rng.choice(["group", "group_grad", "rotate", "rotate", "differ", "differ_grad", "token"])
    type = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("group", "group_grad"):
        activation = rng.choice(["none", "relu", "silu", "silu"])
        while True:
            batch, height, width = _spread(rng, 1, 64), _spread(rng, 1, 256), _spread(rng, 1, 256)
            groups, each = rng.choice([1, 4, 8, 16, 32, 32]), _spread(rng, 2, 64)
            if 1 << 12 <= batch * height * width * groups * each * BYTES[type] <= 16 * 64 * 64 * 320 * 2 and height * width * each > 16:
                return _group(None, kind, type, batch, height, width, groups * each, groups, activation)
    if kind == "rotate":
        while True:
            batch, tokens = _spread(rng, 1, 16), _spread(rng, 1, 32768)
            head, kv_heads, group = rng.choice([32, 40, 64, 64, 80, 96, 128, 128]), rng.choice([1, 2, 4, 8, 12]), rng.choice([1, 1, 2, 4])
            if batch * tokens * kv_heads * (group + 1) * head * BYTES[type] > 2 * 19200 * 32 * 128 * 2:
                continue
            axes, pairs = rng.choice([1, 2, 2, 3, 3]), rng.choice([head // 2, head // 2, head // 4])
            cuts = sorted(rng.sample(range(1, pairs), axes - 1))
            sections = ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [pairs]))
            return _rotate(None, type, batch, tokens, group * kv_heads, kv_heads, head, sections, rng.random() < 0.5, rng.random() < 0.5,
                           rng.random() < 0.5)
    cover, causal = rng.choice(["all", "lengths", "mask"]), rng.random() < 0.5
    head = rng.choice([32, 40, 64, 64, 80, 96, 128, 128])
    group = rng.choice([1, 1, 2, 4, 8])
    if kind == "token":
        while True:
            batch, keys, kv_heads = _spread(rng, 1, 64), _spread(rng, 128, 65536), rng.choice([1, 2, 4, 8, 16])
            if batch * keys * kv_heads * head * BYTES[type] <= 65536 * 8 * 128 * 2:
                return _differ(None, "differ", type, batch, 1, keys, group * kv_heads, kv_heads, head, cover, causal)
    most = 4096 * 4096 * 16 * 64 * (1 if kind == "differ_grad" else 2) // (16 if type == "f32" or (type == "f16" and kind == "differ_grad") else 1)
    while True:
        batch, queries, keys = _spread(rng, 1, 16), _spread(rng, 2, 4096), _spread(rng, 16, 4096)
        kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
        if batch * queries * keys * group * kv_heads * head <= most and group * kv_heads <= 32:
            return _differ(None, kind, type, batch, queries, keys, group * kv_heads, kv_heads, head, cover, causal)


# ---- inputs --------------------------------------------------------------------------------------------------


def _lengths(case):
    """The lengths of the sequences: the same numbers for every seed, so that the work is the same."""
    b, n = case["batch"], case["keys"]
    return [max(1, n - (n // 2) * i // b) for i in range(b)]


def _sections(case):
    return [int(n) for n in case["sections"].split(",")]


def _places(n, axes):
    """n positions with so many axes: the places of a grid, one after the other, as a video or an image has them."""
    side = max(1, math.ceil(n ** (1.0 / axes)))
    at = torch.arange(n, device="cuda")
    return torch.stack([at // side ** k % side if k + 1 < axes else at // side ** k for k in reversed(range(axes))], -1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t = TYPES[case["type"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=None):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype or t)

    s = {"case": case}
    op = case["op"]
    if op in ("group", "group_grad"):
        shape = [case[k] for k in ("batch", "height", "width", "channels")]
        # features with means of their own, and an outlying channel
        x = torch.randn(*shape, generator=g, device="cuda") * 1.5 + torch.randn(shape[3], generator=g, device="cuda") * 0.5
        x[..., shape[3] // 3] *= 4
        s["x"] = x.to(t)
        s["scale"], s["offset"] = normal(shape[3], scale=0.2, shift=1.0), normal(shape[3], scale=0.3)
        if op == "group_grad":
            s["dy"] = normal(*shape)
            _, s["mean"], s["rstd"] = _plain_group(s)
    elif op == "rotate":
        b, n, d = case["batch"], case["tokens"], case["head"]
        s["q"], s["k"] = normal(b, n, case["heads"], d), normal(b, n, case["kv_heads"], d)
        places = _places(n, len(_sections(case)))
        # a window of a longer video or document in each sequence
        s["positions"] = (places[None] + torch.randint(0, 4096, (b, 1, places.shape[1]), generator=g, device="cuda")).to(torch.int32)
        s["sections"] = _sections(case)
    else:
        b, lq, lk, h, hkv, d = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "head"))
        s["q"] = normal(b, lq, 2 * h, d)
        s["k"], s["v"] = normal(b, lk, 2 * hkv, d), normal(b, lk, hkv, 2 * d)
        s["weights"] = normal(h, scale=0.1, shift=0.6)
        s["key_lengths"] = s["key_mask"] = None
        if case["cover"] == "lengths":
            order = torch.randperm(b, generator=g, device="cuda")
            s["key_lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")[order]
        elif case["cover"] == "mask":
            s["key_mask"] = torch.rand(b, lk, generator=g, device="cuda") >= 0.125
        if op == "differ_grad":
            s["do"] = normal(b, lq, h, 2 * d)
            s["o"], s["lse"], s["second"] = _plain_differ(s)
    return s


# ---- the plain forms: 32 bits, rounded once at the end -------------------------------------------------------


def _grouped(x, groups):
    """batch x places x groups x (channels of a group), f32."""
    return x.float().reshape(x.shape[0], -1, groups, x.shape[-1] // groups)


def _plain_group(s):
    case, x = s["case"], s["x"]
    f = _grouped(x, case["groups"])
    mean = f.mean((1, 3))
    c = f - mean[:, None, :, None]
    rstd = torch.rsqrt((c * c).mean((1, 3)) + EPSILON)
    z = (c * rstd[:, None, :, None]).reshape(x.shape) * s["scale"].float() + s["offset"].float()
    if case["activation"] == "relu":
        z = torch.where(z < 0, torch.zeros_like(z), z)
    elif case["activation"] == "silu":
        z = z / (1 + torch.exp(-z))
    return z.to(x.dtype), mean, rstd


def _plain_group_grad(s):
    case, x = s["case"], s["x"]
    groups, w = case["groups"], s["scale"].float()
    rstd = s["rstd"][:, None, :, None]
    xhat = ((_grouped(x, groups) - s["mean"][:, None, :, None]) * rstd).reshape(x.shape)
    g = s["dy"].float()
    if case["activation"] == "relu":      # which side of zero: values next to it need more bits
        z = (x.double().reshape(x.shape[0], -1, groups, x.shape[-1] // groups) - s["mean"].double()[:, None, :, None]) * rstd.double()
        g = g * (z.reshape(x.shape) * s["scale"].double() + s["offset"].double() > 0)
    elif case["activation"] == "silu":
        z = xhat * w + s["offset"].float()
        sig = 1 / (1 + torch.exp(-z))
        g = g * (sig * (1 + z * (1 - sig)))
    by_channel = tuple(range(x.dim() - 1))
    dscale, doffset = (g * xhat).sum(by_channel), g.sum(by_channel)
    gw, xh = _grouped(g * w, groups), _grouped(xhat, groups)
    dx = (gw - gw.mean((1, 3), keepdim=True) - xh * (gw * xh).mean((1, 3), keepdim=True)) * rstd
    return dx.reshape(x.shape).to(x.dtype), dscale.to(s["scale"].dtype), doffset.to(s["scale"].dtype)


def _plain_rotate(s):
    case = s["case"]
    sections, at = s["sections"], s["positions"].double()
    pairs, head = sum(sections), case["head"]
    # angles of far positions in 64 bits
    angles, first = [], 0
    for axis, n in enumerate(sections):
        i = torch.arange(n, device="cuda", dtype=torch.float64)
        exponent = (i + first) / pairs if case["shared"] else i / n
        angles.append(at[..., axis, None] * BASE ** -exponent)
        first += n
    angle = torch.cat(angles, -1)[:, :, None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    if case["inverse"]:
        sin = -sin
    done = []
    for x in (s["q"], s["k"]):
        y = x.float().clone()
        if case["interleaved"]:
            a, b = slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)
        else:
            a, b = slice(0, pairs), slice(pairs, 2 * pairs)
        u, w = x[..., a].float(), x[..., b].float()
        y[..., a] = u * cos - w * sin
        y[..., b] = u * sin + w * cos
        done.append(y.to(x.dtype))
    return done


def _counts(s):
    """batch (or 1) x queries (or 1) x keys truth values, or None where every key counts."""
    case, lk = s["case"], s["k"].shape[1]
    lengths = s["key_lengths"]
    counts = None
    if s["key_mask"] is not None:
        counts = s["key_mask"][:, None, :]
    elif lengths is not None:
        counts = (torch.arange(lk, device="cuda")[None, :] < lengths[:, None])[:, None, :]
    if case["causal"]:
        lq = s["q"].shape[1]
        ends = torch.arange(lq, device="cuda")[None, :] + 1 - lq + (lk if lengths is None else lengths[:, None])
        seen = torch.arange(lk, device="cuda")[None, None, :] < ends[:, :, None]
        counts = seen if counts is None else counts & seen
    return counts


def _by_kv_head(x, kv_heads):
    """batch x tokens x heads x head -> batch x kv_heads x (heads of the group * tokens) x head, f32."""
    b, n, h, d = x.shape
    return x.float().view(b, n, kv_heads, h // kv_heads, d).permute(0, 2, 3, 1, 4).reshape(b, kv_heads, h // kv_heads * n, d)


def _by_token(x, tokens):
    """The other way: batch x kv_heads x (group * tokens) x head -> batch x tokens x heads x head."""
    b, hkv, m, d = x.shape
    return x.view(b, hkv, m // tokens, tokens, d).permute(0, 3, 1, 2, 4).reshape(b, tokens, hkv * (m // tokens), d)


def _plain_weights(s, which):
    """(q, k by key/value head, exp(score - its row's largest), their sums, the largest scores) of one map."""
    hkv, d = s["v"].shape[2], s["q"].shape[3]
    q, k = (_by_kv_head(s[x][:, :, which::2].contiguous(), hkv) for x in "qk")
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * d ** -0.5
    counts = _counts(s)
    if counts is not None:
        b, lq = s["q"].shape[:2]
        by_query = scores.view(b, hkv, -1, lq, scores.shape[3])
        by_query.masked_fill_(~counts[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(scores.sub_(top))
    return q, k, p, p.sum(-1, keepdim=True), top


def _over(total):
    return torch.where(total == 0, torch.ones_like(total), total)


def _plain_differ(s):
    b, lq, h2, d = s["q"].shape
    hkv = s["v"].shape[2]
    v = _by_kv_head(s["v"], hkv)
    o, lse = [], torch.empty(b, h2, lq, device="cuda")
    for which in (0, 1):
        _, _, p, total, top = _plain_weights(s, which)
        o.append(_by_token(torch.matmul(p, v) / _over(total), lq))
        lse[:, which::2] = (torch.log(total) + top).view(b, h2 // 2, lq)
    t = s["q"].dtype
    return (o[0] - s["weights"].float()[:, None] * o[1]).to(t), lse, o[1].to(t)


def _plain_differ_grad(s):
    b, lq, h2, d = s["q"].shape
    lk, hkv = s["k"].shape[1], s["v"].shape[2]
    v, g = _by_kv_head(s["v"], hkv), _by_kv_head(s["do"], hkv)
    share = s["weights"].float().view(hkv, -1, 1).expand(hkv, -1, lq).reshape(1, hkv, -1, 1)
    dp = torch.matmul(g, v.transpose(2, 3).contiguous())
    dq, dk, dv, dweights = torch.empty_like(s["q"]), torch.empty_like(s["k"]), None, None
    for which in (0, 1):
        q, k, p, total, _ = _plain_weights(s, which)
        p.div_(_over(total))
        delta = (p * dp).sum(-1, keepdim=True)
        if which:
            dweights = -delta.view(b, h2 // 2, lq).sum((0, 2))
        times = -share if which else torch.ones_like(share)
        part = torch.matmul((p * times).transpose(2, 3), g)
        dv = part if dv is None else dv + part
        ds = p.mul_(dp - delta).mul_(times * d ** -0.5)
        dq[:, :, which::2] = _by_token(torch.matmul(ds, k), lq).to(dq.dtype)
        dk[:, :, which::2] = _by_token(torch.matmul(ds.transpose(2, 3), q), lk).to(dk.dtype)
    return dq, dk, _by_token(dv, lk).to(s["v"].dtype), dweights.to(s["weights"].dtype)


def run(state):
    s = state
    case = s["case"]
    op = case["op"]
    if own:
        import nnv_amd as nnv
        if op in ("group", "group_grad"):
            activation = None if case["activation"] == "none" else case["activation"]
            if op == "group":
                return nnv.group_norm(s["x"], case["groups"], s["scale"], s["offset"], EPSILON, activation)
            return nnv.group_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["scale"], s["offset"], activation)
        if op == "rotate":
            return nnv.rotate_positions([s["q"], s["k"]], s["positions"], s["sections"], BASE, shared=case["shared"],
                                        interleaved=case["interleaved"], inverse=case["inverse"])
        kw = {"key_lengths": s["key_lengths"], "key_mask": s["key_mask"], "causal": case["causal"]}
        if op == "differ":
            return nnv.differential_attention(s["q"], s["k"], s["v"], s["weights"], **kw)[:2]
        return nnv.differential_attention_backward(s["do"], s["q"], s["k"], s["v"], s["weights"], s["o"], s["lse"], s["second"], **kw)
    if op == "group":
        return _plain_group(s)
    if op == "group_grad":
        return _plain_group_grad(s)
    if op == "rotate":
        return _plain_rotate(s)
    if op == "differ":
        return _plain_differ(s)[:2]
    return _plain_differ_grad(s)


def _pairs(case):
    """(pairs of a query and a key that it sees, over all sequences, per head; keys that count, over all sequences)"""
    b, lq, lk = case["batch"], case["queries"], case["keys"]
    lengths = _lengths(case) if case["cover"] == "lengths" else [lk] * b
    if not case["causal"]:
        return lq * sum(lengths), sum(lengths)
    return sum(max(0, n - lq + i + 1) for n in lengths for i in range(lq)), sum(lengths)


def work(case):
    e, op = BYTES[case["type"]], case["op"]
    if op in ("group", "group_grad"):
        n = case["batch"] * case["height"] * case["width"] * case["channels"]
        stats = 8 * case["batch"] * case["groups"]
        if op == "group":
            return {"bytes": 2 * n * e + 2 * case["channels"] * e + stats, "flops": 10 * n}
        return {"bytes": 3 * n * e + 4 * case["channels"] * e + stats, "flops": 24 * n}
    if op == "rotate":
        rows = case["batch"] * case["tokens"]
        n, pairs = rows * (case["heads"] + case["kv_heads"]), sum(_sections(case))
        return {"bytes": 2 * n * case["head"] * e + 4 * rows * len(_sections(case)), "flops": 6 * n * pairs + 4 * rows * pairs}
    b, lq, h, hkv, d = (case[k] for k in ("batch", "queries", "heads", "kv_heads", "head"))
    seen, keys = _pairs(case)
    rows, kv = b * lq * h, keys * hkv * 2 * d
    if op == "differ":
        return {"bytes": (2 * rows * 2 * d + 2 * kv + h) * e + 8 * rows, "flops": 12 * h * d * seen}
    dkv = b * case["keys"] * hkv * 2 * d                 # the gradients of keys that do not count are written too
    return {"bytes": (5 * rows * 2 * d + 2 * kv + 2 * dkv + 2 * h) * e + 8 * rows, "flops": 20 * h * d * seen}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------


def _exact_group(s):
    case, x = s["case"], s["x"]
    b, c, groups = x.shape[0], x.shape[-1], case["groups"]
    each = c // groups
    y, mean, rstd = torch.empty(x.shape, dtype=torch.float64, device="cuda"), [], []
    for j in range(groups):
        at = slice(j * each, (j + 1) * each)
        part = x[..., at].double().reshape(b, -1)
        var, m = torch.var_mean(part, dim=1, unbiased=False)
        r = 1 / torch.sqrt(var + EPSILON)
        z = ((part - m[:, None]) * r[:, None]).view(x[..., at].shape) * s["scale"][at].double() + s["offset"][at].double()
        y[..., at] = {"none": lambda u: u, "relu": lambda u: u.clamp(min=0), "silu": lambda u: u * torch.sigmoid(u)}[case["activation"]](z)
        mean.append(m)
        rstd.append(r)
    return y, torch.stack(mean, 1), torch.stack(rstd, 1)


def _exact_group_grad(s):
    case, x = s["case"], s["x"]
    b, c, groups = x.shape[0], x.shape[-1], case["groups"]
    each = c // groups
    dx, dscale, doffset = torch.empty(x.shape, dtype=torch.float64, device="cuda"), [], []
    for j in range(groups):
        at = slice(j * each, (j + 1) * each)
        # the gradient for the statistics that the forward pass handed on
        m, r = (s[k][:, j].double()[:, None, None] for k in ("mean", "rstd"))
        part, w = x[..., at].double().reshape(b, -1, each), s["scale"][at].double()
        xhat = (part - m) * r
        z, g = xhat * w + s["offset"][at].double(), s["dy"][..., at].double().reshape(b, -1, each)
        if case["activation"] == "relu":
            g = g * (z > 0)
        elif case["activation"] == "silu":
            sig = torch.sigmoid(z)
            g = g * sig + g * z * sig * (1 - sig)
        dscale.append((g * xhat).sum((0, 1)))
        doffset.append(g.sum((0, 1)))
        gw, n = g * w, part.shape[1] * each
        back = r / n * (n * gw - gw.sum((1, 2), keepdim=True) - xhat * (gw * xhat).sum((1, 2), keepdim=True))
        dx[..., at] = back.view(x[..., at].shape)
    return dx, torch.cat(dscale), torch.cat(doffset)


def _exact_rotate(s):
    case = s["case"]
    total, done = sum(s["sections"]), [s["q"].double(), s["k"].double()]
    pair = 0
    for axis, n in enumerate(s["sections"]):
        for i in range(n):
            frequency = math.exp(-math.log(BASE) * ((pair / total) if case["shared"] else (i / n)))
            angle = s["positions"][..., axis].double() * (-frequency if case["inverse"] else frequency)
            turn = torch.polar(torch.ones_like(angle), angle)[..., None]
            one, two = (2 * pair, 2 * pair + 1) if case["interleaved"] else (pair, pair + total)
            for y in done:
                turned = torch.complex(y[..., one].clone(), y[..., two].clone()) * turn
                y[..., one], y[..., two] = turned.real, turned.imag
            pair += 1
    return done


def _exact_sequence(s, i, j):
    """The keys of sequence i and key/value head j that some query may see, and of each head of the group: (head, v, do-independent
    maps [(q, k, weights, logarithms of the sums)])."""
    lk, lq, d = s["k"].shape[1], s["q"].shape[1], s["q"].shape[3]
    hkv = s["v"].shape[2]
    group = s["q"].shape[2] // 2 // hkv
    n = lk if s["key_lengths"] is None else int(s["key_lengths"][i])
    counted = torch.arange(lk, device="cuda") < n
    if s["key_mask"] is not None:
        counted &= s["key_mask"][i]
    seen = counted[None, :].repeat(lq, 1)
    if s["case"]["causal"]:
        seen &= torch.ones(lq, lk, dtype=torch.bool, device="cuda").tril(n - lq)
    for h in range(j * group, (j + 1) * group):
        maps = []
        for m in (0, 1):
            q, k = s["q"][i, :, 2 * h + m].double(), s["k"][i, :, 2 * j + m].double()
            logits = ((q @ k.T.contiguous()) / math.sqrt(d)).masked_fill(~seen, -math.inf)
            logs = torch.logsumexp(logits, -1)
            weights = torch.exp(logits - torch.where(torch.isinf(logs), torch.zeros_like(logs), logs)[:, None])
            maps.append((q, k, weights, logs))
        yield h, maps


def _exact_differ(s):
    b, lq, h2, d = s["q"].shape
    o = torch.zeros(b, lq, h2 // 2, 2 * d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(b, h2, lq, dtype=torch.float64, device="cuda")
    for i in range(b):
        for j in range(s["v"].shape[2]):
            v = s["v"][i, :, j].double()
            for h, ((_, _, p, logs), (_, _, r, more)) in _exact_sequence(s, i, j):
                o[i, :, h] = (p - float(s["weights"][h]) * r) @ v
                lse[i, 2 * h], lse[i, 2 * h + 1] = logs, more
    return o, lse


def _exact_differ_grad(s):
    dq, dk, dv, dw = (torch.zeros(s[x].shape, dtype=torch.float64, device="cuda") for x in ("q", "k", "v", "weights"))
    for i in range(s["q"].shape[0]):
        for j in range(s["v"].shape[2]):
            v = s["v"][i, :, j].double()
            for h, maps in _exact_sequence(s, i, j):
                g, share = s["do"][i, :, h].double(), float(s["weights"][h])
                dp = g @ v.T.contiguous()
                dv[i, :, j] += (maps[0][2] - share * maps[1][2]).T.contiguous() @ g
                dw[h] -= (maps[1][2] * dp).sum()
                for m, (q, k, p, _) in enumerate(maps):
                    ds = p * (dp - (p * dp).sum(1, keepdim=True)) * ((-share if m else 1.0) / math.sqrt(q.shape[1]))
                    dq[i, :, 2 * h + m] = ds @ k
                    dk[i, :, 2 * j + m] += ds.T.contiguous() @ q
    return dq, dk, dv, dw


def exact(case, seed):
    s = prepare(case, seed)
    return {"group": _exact_group, "group_grad": _exact_group_grad, "rotate": _exact_rotate, "differ": _exact_differ,
            "differ_grad": _exact_differ_grad}[case["op"]](s)
