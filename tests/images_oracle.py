"""Plain 64-bit forms of the operators on points that are images or videos, and how far a right kernel may be from them: the rules are those
of tests/points_oracle.py."""
import math

import torch

from tests.points_oracle import TINY, U, U32

# ---- group normalization ------------------------------------------------------------------------

GROUP_ADDS = 400    # f32 additions one behind the other in the backward pass: 128 places of a thread, up to 256 threads' sums, what is done to them


def _by_group(x, groups):
    """batch x places x groups x (channels of a group), f64"""
    return x.double().reshape(x.shape[0], -1, groups, x.shape[-1] // groups)


def _params(x, scale, offset):
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if scale is None else scale.double()
    b = torch.zeros_like(w) if offset is None else offset.double()
    return w, b


def _z(x, mean, rstd, scale, offset):
    w, b = _params(x, scale, offset)
    f = _by_group(x, mean.shape[1])
    xh = ((f - mean.double()[:, None, :, None]) * rstd.double()[:, None, :, None]).reshape(x.shape)
    return xh, xh * w + b, w, b


def group(x, groups, scale, offset, eps, activation):
    f = _by_group(x, groups)
    mean = f.mean((1, 3))
    c = f - mean[:, None, :, None]
    rstd = 1 / torch.sqrt((c * c).mean((1, 3)) + eps)
    z = _z(x, mean, rstd, scale, offset)[1]
    y = {None: lambda u: u, "relu": lambda u: torch.where(u < 0, 0.0, u), "silu": lambda u: u * torch.sigmoid(u)}[activation](z)
    return y, mean, rstd


def _to_places(x, by_group):
    """batch x groups -> x's shape"""
    return by_group[:, None, :, None].expand(_by_group(x, by_group.shape[1]).shape).reshape(x.shape)


def group_bounds(x, groups, scale, offset, eps, activation):
    """(for y, for the mean, for rstd) beyond their own rounding: the sums are f64, mean and rstd rounded to f32."""
    y, mean, rstd = group(x, groups, scale, offset, eps, activation)
    xh, z, w, b = _z(x, mean, rstd, scale, offset)
    # n terms in f64, of which the variance is a difference: below 2^-53 n times the mean square
    n = x[0].numel() / groups * 2.0 ** -53
    square = (_by_group(x, groups) ** 2).mean((1, 3))
    d_mean = n * square.sqrt()
    d_rstd = rstd ** 3 * n * square
    # x - mean with the mean rounded, the difference, rstd w, their product and the sum with b
    d_z = w.abs() * _to_places(x, rstd * (U32 * mean.abs() + d_mean)) + (xh * w).abs() * _to_places(x, d_rstd / rstd) + 6 * U32 * ((xh * w).abs() + b.abs())
    if activation == "silu":    # a slope of at most 1.1; an exponent of z / ln 2 that is rounded, and what is formed of it
        d_z = 1.1 * d_z + (2 * z.abs() + 8) * U32 * y.abs() + 2.0 ** -120
    return d_z, d_mean, d_rstd


def _slope(z, activation):
    if activation == "relu":
        return (z > 0).double()
    if activation == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def group_grad(dy, x, mean, rstd, scale, offset, activation):
    xh, z, w, _ = _z(x, mean, rstd, scale, offset)
    h = dy.double() * _slope(z, activation)
    lead = tuple(range(x.dim() - 1))
    groups = mean.shape[1]
    gw, gx = _by_group(h * w, groups), _by_group(xh, groups)
    dx = rstd.double()[:, None, :, None] * (gw - gw.mean((1, 3), keepdim=True) - gx * (gw * gx).mean((1, 3), keepdim=True))
    return dx.reshape(x.shape), (h * xh).sum(lead), h.sum(lead)


def group_grad_bounds(dy, x, mean, rstd, scale, offset, activation, adds=GROUP_ADDS):
    xh, z, w, b = _z(x, mean, rstd, scale, offset)
    g, slope = dy.double().abs(), _slope(z, activation).abs()
    d_xh = 3 * U32 * xh.abs()
    d_h = torch.zeros_like(z)
    if activation == "silu":    # the slope's own slope is at most a half; its terms are rounded
        d_h = g * (0.5 * (w.abs() * d_xh + 2 * U32 * ((xh * w).abs() + b.abs())) + (2 * z.abs() + 8) * (1 + z.abs()) * U32)
    h = g * slope
    n = adds * U32
    lead, groups = tuple(range(x.dim() - 1)), mean.shape[1]

    def over_group(t):
        return _to_places(x, _by_group(t, groups).mean((1, 3)))

    m0, d_m0 = over_group(h * w.abs()), over_group((d_h + n * h) * w.abs())
    m1, d_m1 = over_group(h * w.abs() * xh.abs()), over_group(((d_h + n * h) * xh.abs() + h * d_xh) * w.abs())
    r = _to_places(x, rstd.double())
    d_dx = r * (d_h * w.abs() + d_m0 + xh.abs() * d_m1 + d_xh * m1 + 6 * U32 * (h * w.abs() + m0 + xh.abs() * m1))
    d_dscale = (d_h * xh.abs() + h * d_xh + n * h * xh.abs()).sum(lead)
    return d_dx, d_dscale, (d_h + n * h).sum(lead)


# ---- rotary positions ---------------------------------------------------------------------------


def rotate(x, positions, sections, base=10000.0, shared=False, interleaved=False, inverse=False):
    """As complex numbers, pair by pair."""
    y, total, pair = x.double().clone(), sum(sections), 0
    at = positions.double()
    at = at if at.dim() == 3 else at[None].expand(x.shape[0], -1, -1)
    for axis, n in enumerate(sections):
        for i in range(n):
            angle = at[..., axis] * base ** -(pair / total if shared else i / n)
            turn = torch.polar(torch.ones_like(angle), -angle if inverse else angle)[..., None]
            a, b = (2 * pair, 2 * pair + 1) if interleaved else (pair, pair + total)
            t = torch.complex(y[..., a].clone(), y[..., b].clone()) * turn
            y[..., a], y[..., b] = t.real, t.imag
            pair += 1
    return y


def rotate_bounds(x, positions, sections, base=10000.0, shared=False, interleaved=False):
    """cos and sin in f32 (two units each, a turn's fraction rounded to f32: half a turn's 2^-25 times 2 pi), two products and a sum; angles in f64
    of positions and frequencies."""
    total = sum(sections)
    size = torch.zeros_like(x, dtype=torch.float64)
    f = x.double()
    a = slice(0, 2 * total, 2) if interleaved else slice(0, total)
    b = slice(1, 2 * total, 2) if interleaved else slice(total, 2 * total)
    size[..., a] = size[..., b] = f[..., a].abs() + f[..., b].abs()
    far = float(positions.double().abs().max()) if positions.numel() else 0.0
    return size * ((math.pi + 2 + 2) * U32 + 8 * far * 2.0 ** -53)


# ---- differential attention ---------------------------------------------------------------------


def seen(q, k, key_lengths=None, key_mask=None, causal=False):
    """batch x queries x keys truth values: which keys a query sees."""
    b, lq, lk = q.shape[0], q.shape[1], k.shape[1]
    n = torch.full((b,), lk, device=q.device) if key_lengths is None else key_lengths.long().clamp(0, lk)
    c = torch.arange(lk, device=q.device)[None, None] < n[:, None, None]
    if key_mask is not None:
        c = c & key_mask.bool()[:, None]
    if causal:
        c = c & (torch.arange(lk, device=q.device)[None, None] < (n[:, None] - lq + torch.arange(lq, device=q.device) + 1)[:, :, None])
    return c.expand(b, lq, lk)


def _split_maps(q, k, v, c):
    """f64 [(q, k) of each map], v, as batch x heads x tokens x values; keys that no query sees, and queries that see none, are zero."""
    group = q.shape[2] // k.shape[2]
    counts, takes = c.any(1), c.any(2)

    def heads(x, keep, repeat=1):
        x = torch.where(keep[:, :, None, None], x.double(), torch.zeros((), dtype=torch.float64, device=x.device))
        return x.repeat_interleave(repeat, dim=2).permute(0, 2, 1, 3).contiguous()

    return [(heads(q[:, :, m::2], takes), heads(k[:, :, m::2], counts, group)) for m in (0, 1)], heads(v, counts, group)


def _matmul(a, b):
    return torch.matmul(a, b.transpose(-1, -2).contiguous())


def _softmax(q, k, c, scale):
    """(weights, logarithms of the sums) of a map"""
    s = (_matmul(q, k) * scale).masked_fill(~c[:, None], -math.inf)
    lse = torch.logsumexp(s, -1) if s.shape[-1] else torch.full(s.shape[:-1], -math.inf, dtype=s.dtype, device=s.device)
    none = lse == -math.inf
    return torch.exp(s - torch.where(none, 0.0, lse)[..., None]), lse


def _tokens(x):
    return x.permute(0, 2, 1, 3)


def differ(q, k, v, weights, key_lengths=None, key_mask=None, causal=False, scale=None):
    """(o, lse, second) in f64."""
    scale = q.shape[3] ** -0.5 if scale is None else scale
    c = seen(q, k, key_lengths, key_mask, causal)
    maps, v = _split_maps(q, k, v, c)
    (p0, l0), (p1, l1) = (_softmax(*m, c, scale) for m in maps)
    second = torch.matmul(p1, v)
    o = torch.matmul(p0, v) - weights.double()[None, :, None, None] * second
    return _tokens(o), torch.stack([l0, l1], 2).flatten(1, 2), _tokens(second)


def _differ_sizes(q, k, v, c, scale):
    """Per map: (weights, how far one may be off relative to itself, sizes of q and k), and v's sizes, by head."""
    maps, v = _split_maps(q, k, v, c)
    found = []
    for qm, km in maps:
        p, lse = _softmax(qm, km, c, scale)
        off = (q.shape[3] + 16) * U32 * _matmul(qm.abs(), km.abs()) * abs(scale)
        off = off.amax(-1, keepdim=True) if off.shape[-1] else off.sum(-1, keepdim=True)
        finite = torch.where(torch.isfinite(lse), lse, torch.zeros_like(lse))[..., None]
        found.append((p, off + 8 * U32 * (finite.abs() + 1), qm.abs(), km.abs()))
    return found, v


def differ_bounds(q, k, v, weights, key_lengths=None, key_mask=None, causal=False, scale=None):
    """(for o, for lse, for second): as attend_bounds of either map, and the difference."""
    scale = q.shape[3] ** -0.5 if scale is None else scale
    c = seen(q, k, key_lengths, key_mask, causal)
    found, v = _differ_sizes(q, k, v, c, scale)
    n, short = (k.shape[1] + 32) * U32, 0.0 if q.dtype == torch.float32 else U[q.dtype]
    w = weights.double().abs()[None, :, None, None]
    small = 0.0 if q.dtype != torch.float16 else TINY[q.dtype] * v.abs().sum(-2, keepdim=True)
    d_maps, sizes, d_lse = [], [], []
    for p, off, _, _ in found:
        d_maps.append((2 * off + n + short) * torch.matmul(p, v.abs()) + small)
        sizes.append(torch.matmul(p, v).abs())
        d_lse.append((2 * off + n)[..., 0])
    d_o = d_maps[0] + w * d_maps[1] + 4 * U32 * (sizes[0] + w * sizes[1])
    return _tokens(d_o), torch.stack(d_lse, 2).flatten(1, 2), _tokens(d_maps[1])


def _by_map(x0, x1):
    """batch x heads x tokens x values of two maps -> batch x tokens x 2 heads x values"""
    return torch.stack([_tokens(x0), _tokens(x1)], 3).flatten(2, 3)


def _over_group(x, group):
    b, h, n, d = x.shape
    return x.view(b, h // group, group, n, d).sum(2)


def differ_grad(do, q, k, v, weights, key_lengths=None, key_mask=None, causal=False, scale=None):
    """(dq, dk, dv, dweights) in f64, from the inputs alone."""
    scale, group = q.shape[3] ** -0.5 if scale is None else scale, q.shape[2] // k.shape[2]
    c = seen(q, k, key_lengths, key_mask, causal)
    maps, vh = _split_maps(q, k, v, c)
    w = weights.double()[None, :, None, None]
    g = torch.where(c.any(2)[:, None, :, None], do.double().permute(0, 2, 1, 3), 0.0).contiguous()
    dp = _matmul(g, vh)
    t = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    dq, dk, both, dw = [], [], 0.0, None
    for m, (qm, km) in enumerate(maps):
        by = -w if m else 1.0
        p, _ = _softmax(qm, km, c, scale)
        delta = (p * dp).sum(-1, keepdim=True)
        ds = by * p * (dp - delta) * scale
        dq.append(torch.matmul(ds, km))
        dk.append(_over_group(torch.matmul(t(ds), qm), group))
        both = both + by * p
        dw = -delta.sum((0, 2, 3))
    return _by_map(*dq), _by_map(*dk), _tokens(_over_group(torch.matmul(t(both), g), group)), dw


def differ_grad_bounds(do, q, k, v, weights, key_lengths=None, key_mask=None, causal=False, scale=None):
    """As attend_grad_bounds of either map; D of the first one is formed from the rounded o and that of the second from the rounded second."""
    scale_, group = abs(q.shape[3] ** -0.5 if scale is None else scale), q.shape[2] // k.shape[2]
    c = seen(q, k, key_lengths, key_mask, causal)
    found, vh = _differ_sizes(q, k, v, c, scale_ if scale is None else scale)
    u = U[q.dtype]
    short = 0.0 if q.dtype == torch.float32 else u
    o, _, second = differ(q, k, v, weights, key_lengths, key_mask, causal, scale)
    bo, _, bs = differ_bounds(q, k, v, weights, key_lengths, key_mask, causal, scale)
    o, second, bo, bs = (x.permute(0, 2, 1, 3).abs() for x in (o, second, bo, bs))
    w = weights.double().abs()[None, :, None, None]
    g = torch.where(c.any(2)[:, None, :, None], do.double().permute(0, 2, 1, 3).abs(), 0.0).contiguous()
    wide = (2 * q.shape[3] + 16) * U32
    n = (max(k.shape[1], group * q.shape[1]) + 64) * U32
    dp = _matmul(g, vh.abs())
    d_d1 = (g * (wide * second + bs + u * second)).sum(-1, keepdim=True)
    d_d0 = (g * (wide * o + bo + u * o)).sum(-1, keepdim=True) + w * (d_d1 + 4 * U32 * (g * second).sum(-1, keepdim=True))
    t = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    dq, dk, dv = [], [], 0.0
    for m, (p, off, qm, km) in enumerate(found):
        by, d_d = (w, d_d1) if m else (1.0, d_d0)
        own = torch.matmul(p, vh).abs()
        weight = 3 * off + n + short
        size = by * p * (dp + (g * own).sum(-1, keepdim=True))
        d_ds = size * (weight + short + 6 * U32) + by * p * (wide * dp + d_d)
        dq.append(scale_ * torch.matmul(d_ds + n * size, km))
        dk.append(_over_group(scale_ * torch.matmul(t(d_ds + n * size), qm), group))
        dv = dv + by * p * (weight + n + 2 * U32)
    dv = _tokens(_over_group(torch.matmul(t(dv), g), group))
    return _by_map(*dq), _by_map(*dk), dv, (d_d1 + 2.0 ** -24 * (g * second).sum(-1, keepdim=True)).sum((0, 2, 3))
