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
