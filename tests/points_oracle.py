"""Plain 64-bit forms of the operators on points, and how far a right kernel may be from them.

The bounds follow the arithmetic: u(T) is half a unit in the last place of type T relative to the value (2^-24 for f32,
2^-11 for f16, 2^-8 for bf16); a sum of n terms in f32 is off by at most (n + a few) u(f32) times the sum of the terms' sizes;
each result is rounded once to its type; and the attention kernels may round the softmax's weights, and the gradients of the
scores, to 16 bits before the product that uses them when the tensors have 16 bits."""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}  # what an underflow loses at most
U32 = U[torch.float32]


def assert_within(got, exact, bound, what):
    """|got - exact| <= u |exact| + bound, element by element, u of got's type; NaN and inf in the same places."""
    assert got.shape == exact.shape, "%s: %s instead of %s" % (what, tuple(got.shape), tuple(exact.shape))
    g = got.double()
    fine = torch.isfinite(exact)
    assert torch.equal(fine, torch.isfinite(g)), "%s: not finite in other places" % what
    assert torch.equal(g[~fine], exact[~fine]) or torch.isnan(exact[~fine]).all() and torch.isnan(g[~fine]).all(), what
    allowed = (U[got.dtype] * exact.abs() + bound + TINY[got.dtype])[fine]
    err = (g - exact)[fine].abs()
    if err.numel():
        worst = (err / allowed).max().item()
        assert worst <= 1.0, "%s: an error is %.3g times what rounding explains" % (what, worst)


# ---- layer normalization ------------------------------------------------------------------------------

ROW_ADDS = 64   # additions in a row on one lane (at most 16 values), over lanes (6) and waves (8), and what is done to them


def norm(x, scale, offset, eps):
    x = x.double()
    mean = x.mean(-1)
    c = x - mean[..., None]
    rstd = 1 / torch.sqrt((c * c).mean(-1) + eps)
    xh = c * rstd[..., None]
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if scale is None else scale.double()
    b = torch.zeros_like(w) if offset is None else offset.double()
    return xh * w + b, mean, rstd


def norm_bounds(x, scale, offset, eps, adds=ROW_ADDS):
    """(for y, for the mean, for rstd) beyond their own rounding."""
    y, mean, rstd = norm(x, scale, offset, eps)
    x = x.double()
    size = x.abs().mean(-1)                       # the mean's error is adds u of this
    spread = (x - mean[..., None]).abs()
    w = 1.0 if scale is None else scale.double().abs()
    b = 0.0 if offset is None else offset.double().abs()
    d_mean = adds * U32 * size
    # the variance around a mean that is off: its own sum, and the square of the offset, which is below it
    d_rstd = rstd * (adds * U32 + rstd * d_mean * (rstd * d_mean + 0))
    d_y = w * (rstd * d_mean + (spread * d_rstd[..., None]).max(-1).values)[..., None] + 8 * U32 * (spread * rstd[..., None] * w + b)
    return d_y, d_mean, d_rstd


def norm_grad(dy, x, mean, rstd, scale):
    dy, x, mean, rstd = dy.double(), x.double(), mean.double(), rstd.double()
    xh = (x - mean[..., None]) * rstd[..., None]
    g = dy if scale is None else dy * scale.double()
    dx = rstd[..., None] * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    lead = tuple(range(x.dim() - 1))
    return dx, (dy * xh).sum(lead), dy.sum(lead)


def norm_grad_bounds(dy, x, mean, rstd, scale, adds=ROW_ADDS):
    dy, x, mean, rstd = dy.double(), x.double(), mean.double(), rstd.double()
    # the difference x - mean is rounded once, and so is the product
    xh = (x - mean[..., None]).abs() * rstd[..., None]
    g = (dy if scale is None else dy * scale.double()).abs()
    d_dx = adds * U32 * rstd[..., None] * (g + g.mean(-1, keepdim=True) + xh * (g * xh).mean(-1, keepdim=True))
    rows = max(1, x.numel() // x.shape[-1])
    lead = tuple(range(x.dim() - 1))
    n = (min(rows, 256) + 64) * U32
    return d_dx, n * (dy.abs() * xh).sum(lead), n * dy.abs().sum(lead)


# ---- attention ------------------------------------------------------------------------------------------


def counting(q, k, key_lengths, key_mask):
    """batch x keys truth values: which keys count."""
    b, n = k.shape[0], k.shape[1]
    c = torch.ones(b, n, dtype=torch.bool, device=q.device)
    if key_lengths is not None:
        c &= torch.arange(n, device=q.device)[None] < key_lengths[:, None]
    if key_mask is not None:
        c &= key_mask.bool()
    return c


def _spread_heads(q, k, v, key_lengths, key_mask):
    """f64 (q, k, v) as batch x heads x tokens x head, keys that do not count zero, and which count."""
    c = counting(q, k, key_lengths, key_mask)
    group = q.shape[2] // k.shape[2]

    def keys(x):
        x = torch.where(c[:, :, None, None], x.double(), torch.zeros((), dtype=torch.float64, device=x.device))
        return x.repeat_interleave(group, dim=2).permute(0, 2, 1, 3).contiguous()

    return q.double().permute(0, 2, 1, 3).contiguous(), keys(k), keys(v), c


def _product(a, b):
    return torch.matmul(a, b.transpose(-1, -2).contiguous())


def attend(q, k, v, key_lengths=None, key_mask=None, scale=None):
    """(o, lse) in f64."""
    scale = q.shape[3] ** -0.5 if scale is None else scale
    q, k, v, c = _spread_heads(q, k, v, key_lengths, key_mask)
    s = (_product(q, k) * scale).masked_fill(~c[:, None, None, :], -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(lse[..., None] == -math.inf, torch.zeros_like(s), torch.exp(s - lse[..., None]))
    return torch.matmul(p, v).permute(0, 2, 1, 3), lse


def _attend_sizes(q, k, v, key_lengths, key_mask, scale):
    """What the bounds are made of: (weights, how far a weight may be off relative to itself, sizes of q, k, v by head)."""
    scale_ = q.shape[3] ** -0.5 if scale is None else scale
    _, lse = attend(q, k, v, key_lengths, key_mask, scale)
    qa, ka, va, c = _spread_heads(q, k, v, key_lengths, key_mask)
    s = (_product(qa, ka) * scale_).masked_fill(~c[:, None, None, :], -math.inf)
    p = torch.where(lse[..., None] == -math.inf, torch.zeros_like(s), torch.exp(s - lse[..., None]))
    qa, ka, va = qa.abs(), ka.abs(), va.abs()
    off = (q.shape[3] + 16) * U32 * _product(qa, ka) * abs(scale_)          # of a score
    off = off.amax(-1, keepdim=True) if off.shape[-1] else off.sum(-1, keepdim=True)
    finite = torch.where(torch.isfinite(lse), lse, torch.zeros_like(lse))[..., None]
    return p, off + 8 * U32 * (finite.abs() + 1), qa, ka, va


def attend_bounds(q, k, v, key_lengths=None, key_mask=None, scale=None):
    """(for o, for lse): the weights are off by twice their exponent's error (their own and the sum's), and rounded."""
    p, off, _, _, va = _attend_sizes(q, k, v, key_lengths, key_mask, scale)
    n = (k.shape[1] + 32) * U32
    weights = 0.0 if q.dtype == torch.float32 else U[q.dtype]
    d_o = (2 * off + n + weights) * torch.matmul(p, va)
    small = 0.0 if q.dtype != torch.float16 else TINY[q.dtype] * va.sum(-2, keepdim=True)   # weights below f16's range
    return (d_o + small).permute(0, 2, 1, 3), (2 * off + n)[..., 0]


def attend_grad(do, q, k, v, key_lengths=None, key_mask=None, scale=None):
    """(dq, dk, dv) in f64, from the inputs alone."""
    group = q.shape[2] // k.shape[2]
    scale = q.shape[3] ** -0.5 if scale is None else scale
    o, lse = attend(q, k, v, key_lengths, key_mask, scale)
    q, k, v, c = _spread_heads(q, k, v, key_lengths, key_mask)
    empty = lse[..., None] == -math.inf
    p = torch.where(empty, torch.zeros((), dtype=torch.float64, device=q.device), torch.exp(_product(q, k) * scale - torch.where(empty, 0.0, lse[..., None])))
    p = torch.where(c[:, None, None, :], p, 0.0)
    g = do.double().permute(0, 2, 1, 3).contiguous()
    g, q = torch.where(empty, 0.0, g), torch.where(empty, 0.0, q)
    dp = _product(g, v)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale

    def over_group(x):
        b, h, n, d = x.shape
        return x.view(b, h // group, group, n, d).sum(2).permute(0, 2, 1, 3)

    t = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    return torch.matmul(ds, k).permute(0, 2, 1, 3), over_group(torch.matmul(t(ds), q)), over_group(torch.matmul(t(p), g))


def attend_grad_bounds(do, q, k, v, key_lengths=None, key_mask=None, scale=None):
    group = q.shape[2] // k.shape[2]
    scale_ = abs(q.shape[3] ** -0.5 if scale is None else scale)
    u = U[q.dtype]
    short = 0.0 if q.dtype == torch.float32 else u
    p, off, qa, ka, va = _attend_sizes(q, k, v, key_lengths, key_mask, scale)
    o = attend(q, k, v, key_lengths, key_mask, scale)[0].permute(0, 2, 1, 3).abs()
    d_o = attend_bounds(q, k, v, key_lengths, key_mask, scale)[0].permute(0, 2, 1, 3) + u * o
    g = do.double().permute(0, 2, 1, 3).contiguous().abs()
    head = q.shape[3] + 16
    n = (max(k.shape[1], group * q.shape[1]) + 64) * U32
    weight = 3 * off + n + short                                   # of a weight, relative to it
    dp = _product(g, va)                                           # a bound of dP's size, and of D's
    d_dp = head * U32 * dp + (g * (head * U32 * o + d_o)).sum(-1, keepdim=True)
    size = p * (dp + (g * o).sum(-1, keepdim=True))                # a bound of dS's size
    d_ds = size * (weight + short + 4 * U32) + p * d_dp

    def over_group(x):
        b, h, m, d = x.shape
        return x.view(b, h // group, group, m, d).sum(2).permute(0, 2, 1, 3)

    t = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    dq = scale_ * torch.matmul(d_ds + n * size, ka)
    dk = scale_ * torch.matmul(t(d_ds + n * size), qa)
    dv = torch.matmul(t(p * (weight + n)), g)
    return dq.permute(0, 2, 1, 3), over_group(dk), over_group(dv)


# ---- clipping -------------------------------------------------------------------------------------------


def clip(gradients, threshold):
    n = math.sqrt(sum(float((x.double() ** 2).sum()) for x in gradients))
    f = threshold / n if n > threshold else 1.0
    return [x.double() * f for x in gradients], n
