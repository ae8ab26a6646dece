"""Operators on points that are images or videos: group normalization with an activation over features whose channels come last,
rotary positions with several axes (rows and columns, time), and differential attention.

They stand beside the operators of ``nnv_amd.points`` and follow the same rules: torch tensors on one GPU (f32, bf16 or f16), queued on torch's
current stream of that device, no waiting, workspaces from torch's allocator, no part of torch's graph (tensors that require a
gradient are refused where torch records one).  Sums and statistics are f32 or more, and each result is rounded once; what attention rounds on
the way in 16 bits is said at ``differential_attention``.
"""
from __future__ import annotations

import ctypes as C
import functools
import operator
import struct
from numbers import Integral

import torch

from ._lib import check
from .points import _INT64, _LARGEST, _dense_values, _enter, _mask_args, _ptr, _type

# ---- group normalization ------------------------------------------------------------------------

_ACTIVATIONS = {None: 0, "relu": 1, "silu": 2}
_GROUP = struct.Struct("=7qdQ2qQQQQQQ2qQQQ")   # struct nnvhip_group_norm_args


def _places(x):
    """x (batch x ... x channels) with its places evenly spaced and its channels dense: (tensor, places, strides of batch and place);
    copied where they are not."""
    batch, channels = x.shape[0], x.shape[-1]
    if x.is_contiguous():
        places = x.numel() // (batch * channels) if batch else 1
        return x, places, places * channels, channels
    if x.stride(-1) == 1 or channels == 1:
        try:
            rows = x.view(batch, -1, channels) if x.numel() else None
        except RuntimeError:
            rows = None
        if rows is not None:
            return rows, rows.shape[1], rows.stride(0), rows.stride(1)
    return _places(x.contiguous())


def _group_params(what, x, groups, scale, offset, activation):
    t = _type(what, x)
    if x.dim() < 2:
        raise ValueError("%s: x is batch x ... x channels" % what)
    channels = x.shape[-1]
    if not ((isinstance(groups, int) or isinstance(groups, Integral)) and groups >= 1 and channels >= 1 and channels % groups == 0):
        raise ValueError("%s: the channels (%d) must come in equal groups, not %s" % (what, channels, groups))
    if 0 in x.shape[1:]:
        raise ValueError("%s: at least one place is expected, not the shape %s" % (what, tuple(x.shape)))
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError("%s: the activation is None, 'relu' or 'silu', not %r" % (what, activation))
    w = t
    for p in (scale, offset):
        if p is not None:
            if p.shape != (channels,):
                raise ValueError("%s: scale and offset have one value per channel (%d), not the shape %s" % (what, channels, tuple(p.shape)))
            w = _type(what, p)
            if w not in (t, 0):
                raise ValueError("%s: scale and offset have the type of the values, or float32" % what)
    if scale is not None and offset is not None and scale.dtype != offset.dtype:
        raise ValueError("%s: scale and offset must have the same type" % what)
    return t, w, act


@functools.lru_cache(maxsize=256)
def _group_workspace(lib, backward, t, batch, places, channels, groups):
    n = _INT64()
    d = _GROUP.pack(t, t, 0, batch, places, channels, groups, 0.0, *[0] * 14)
    check((lib.nnvhip_group_norm_backward_workspace if backward else lib.nnvhip_group_norm_workspace)(d, C.byref(n)))
    return n.value


def _dense(p):
    return p if p is None or p.is_contiguous() else p.contiguous()


def group_norm(x, groups, scale=None, offset=None, epsilon=1e-5, activation=None, ctx=None):
    """y = act((x - mean) / sqrt(var + epsilon) * scale + offset), mean and var over all places and the channels of a group.

    x: batch x ... x channels; the channels come last, in ``groups`` equal groups of consecutive ones.  activation: None, "relu" or
    "silu" (z / (1 + exp(-z))).  scale and offset: vectors of x's type or f32, or None.
    Returns (y, mean, rstd): y in x's shape and type, the statistics f32, batch x groups; group_norm_backward takes them."""
    what = "group_norm"
    ctx, lib, stream = _enter(what, ctx, x, scale, offset)
    t, w, act = _group_params(what, x, groups, scale, offset, activation)
    if not epsilon >= 0:
        raise ValueError("group_norm: epsilon must not be negative")
    batch, channels = x.shape[0], x.shape[-1]
    scale, offset = _dense(scale), _dense(offset)
    rows, places, xb, xp = _places(x)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    mean = x.new_empty((batch, groups), dtype=torch.float32)
    rstd = torch.empty_like(mean)
    need = _group_workspace(lib, False, t, batch, places, channels, groups)
    work = x.new_empty((need,), dtype=torch.uint8) if need else None
    d = _GROUP.pack(t, w, act, batch, places, channels, groups, epsilon, rows.data_ptr(), xb, xp, _ptr(scale) or 0, _ptr(offset) or 0,
                    y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), 0, 0, 0, 0, 0, 0)
    check(lib.nnvhip_group_norm(ctx.handle, d, _ptr(work), need, stream))
    return y, mean, rstd


def group_norm_backward(dy, x, mean, rstd, scale=None, offset=None, activation=None, ctx=None):
    """The gradients of group_norm: (dx, dscale, doffset) from that of its result and its statistics (which say how many groups there are).

    dx has x's type, dscale and doffset the type of scale or offset (x's if both are None).  The gradient of "relu" is zero at zero."""
    what = "group_norm_backward"
    ctx, lib, stream = _enter(what, ctx, x, dy, mean, rstd, scale, offset)
    batch = x.shape[0] if x.dim() else 0
    for s in (mean, rstd):
        if s.dim() != 2 or s.shape != mean.shape or s.shape[0] != batch or s.dtype != torch.float32:
            raise ValueError("%s: mean and rstd must be what group_norm returned" % what)
    groups = mean.shape[1]
    t, w, act = _group_params(what, x, groups, scale, offset, activation)
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError("%s: dy must have the shape and type of x" % what)
    channels = x.shape[-1]
    scale, offset, mean, rstd = _dense(scale), _dense(offset), _dense(mean), _dense(rstd)
    rows, places, xb, xp = _places(x)
    grows, _, gb, gp = _places(dy)
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    like = scale if scale is not None else offset if offset is not None else x
    dscale = like.new_empty((channels,))
    doffset = torch.empty_like(dscale)
    need = _group_workspace(lib, True, t, batch, places, channels, groups)
    work = x.new_empty((need,), dtype=torch.uint8) if need else None
    d = _GROUP.pack(t, w, act, batch, places, channels, groups, 0.0, rows.data_ptr(), xb, xp, _ptr(scale) or 0, _ptr(offset) or 0, 0,
                    mean.data_ptr(), rstd.data_ptr(), grows.data_ptr(), gb, gp, dx.data_ptr(), dscale.data_ptr(), doffset.data_ptr())
    check(lib.nnvhip_group_norm_backward(ctx.handle, d, _ptr(work), need, stream))
    return dx, dscale, doffset


# ---- rotary positions ---------------------------------------------------------------------------

_ROTATE_TENSORS, _ROTATE_PAIRS = 4, 256
_ROTATE = struct.Struct("=10qQ3qQQ4q4Q4Q12q")   # struct nnvhip_rotate_args
_POSITIONS = {torch.int32: 0, torch.int64: 1, torch.float32: 2}


@functools.lru_cache(maxsize=64)
def _frequencies(sections, base, shared):
    """(frequencies, axes) of the pairs, as arrays that the library reads."""
    pairs = sum(sections)
    values, axes = [], []
    for axis, n in enumerate(sections):
        for i in range(n):
            values.append(base ** -((len(values) / pairs) if shared else (i / n)))
            axes.append(axis)
    return (C.c_double * pairs)(*values), (C.c_uint8 * pairs)(*axes)


_SECTIONS = "rotate_positions: sections are numbers of pairs, one per axis, %d together at most" % _ROTATE_PAIRS


@functools.lru_cache(maxsize=64)
def _turns(sections, base, shared):
    """(pairs, axes, addresses of _frequencies, which they belong to) of a call's arguments, or the error.  sections: ints (a cache takes 2.0 for 2)."""
    if not sections or min(sections) < 0 or not 1 <= sum(sections) <= _ROTATE_PAIRS or len(sections) > 255:
        raise ValueError(_SECTIONS)
    if not 0 < base < float("inf"):
        raise ValueError("rotate_positions: the base must be positive and finite")
    held = _frequencies(sections, base, shared)
    return sum(sections), len(sections), C.addressof(held[0]), C.addressof(held[1]), held


def rotate_positions(x, positions, sections, base=10000.0, shared=False, interleaved=False, inverse=False, ctx=None):
    """x with its heads' values turned by their tokens' positions: rotary positions with several axes.

    x: batch x tokens x heads x head, any strides, or a list of such tensors (queries and keys) whose heads may differ in number.
    positions: tokens x axes, or batch x tokens x axes (i32, i64 or f32).  sections[a] pairs of a head's values are turned by axis a, one axis after
    the other; what is behind 2 * sum(sections) values stays.  A pair is (i, i + sum(sections)), or neighbours (2 i, 2 i + 1) if interleaved.  Its angle is
    position * base^-e with e = (its place in its section) / (pairs of the section), or, if shared, (its place among all pairs) / (all pairs).
    inverse: turned back, which is the backward pass.

    Returns new tensors, a list if x is one."""
    what = "rotate_positions"
    several = not isinstance(x, torch.Tensor)
    tensors = list(x) if several else [x]
    if not tensors:
        raise ValueError("%s: at least one tensor is expected" % what)
    ctx, lib, stream = _enter(what, ctx, tensors[0], *tensors[1:], positions)
    first = tensors[0]
    t = _type(what, first)
    try:
        sections = tuple(map(operator.index, sections))
    except TypeError:
        raise ValueError(_SECTIONS) from None
    pairs, axes, frequency, axis, held = _turns(sections, float(base), bool(shared))   # held: what the addresses are of
    if first.dim() != 4:
        raise ValueError("%s: tensors are batch x tokens x heads x head, alike but for the number of heads" % what)
    batch, tokens, _, head = first.shape
    for y in tensors[1:]:
        if y.dim() != 4 or y.dtype != first.dtype or y.shape[:2] != first.shape[:2] or y.shape[3] != head:
            raise ValueError("%s: tensors are batch x tokens x heads x head, alike but for the number of heads" % what)
    if head < 2 * pairs:
        raise ValueError("%s: heads of %d values do not hold %d pairs" % (what, head, pairs))
    kind, shape, stride = _POSITIONS.get(positions.dtype), positions.shape, positions.stride()
    if len(shape) == 2:
        stride = (0, *stride)
    if kind is None or len(shape) not in (2, 3) or shape[-2:] != (tokens, axes) or (len(shape) == 3 and shape[0] != batch):
        raise ValueError("%s: positions are (batch x) tokens x axes whole numbers or float32, not %s %s" % (what, positions.dtype, tuple(shape)))
    fixed = (t, batch, tokens, head)
    turned = (pairs, axes, bool(interleaved), bool(inverse), kind, positions.data_ptr(), *stride, frequency, axis)
    done = []
    for k in range(0, len(tensors), _ROTATE_TENSORS):
        part = [y if y.stride(3) == 1 or head == 1 else y.contiguous() for y in tensors[k:k + _ROTATE_TENSORS]]
        out = [torch.empty_like(y, memory_format=torch.contiguous_format) for y in part]
        none = (0,) * (_ROTATE_TENSORS - len(part))
        heads, strides = [], []
        for y in part:
            heads.append(y.shape[2])
            strides += y.stride()[:3]
        d = _ROTATE.pack(*fixed, len(part), *turned, *heads, *none, *[y.data_ptr() for y in part], *none, *[y.data_ptr() for y in out], *none,
                         *strides, *none, *none, *none)
        check(lib.nnvhip_rotate_positions(ctx.handle, d, stream))
        done += out
    del held
    return done if several else done[0]


# ---- differential attention ---------------------------------------------------------------------

_DIFFER = struct.Struct("=9qd3Q9qQQQ2qQQQQ3q4Q")   # struct nnvhip_differ_args


def _differ_sizes(what, q, k, v, weights, key_lengths, key_mask, scale):
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("%s: q, k and v are batch x tokens x heads x head" % what)
    batch, queries, heads, head = q.shape
    keys, kv_heads = v.shape[1], v.shape[2]
    if k.shape != (batch, keys, 2 * kv_heads, head) or v.shape != (batch, keys, kv_heads, 2 * head):
        raise ValueError("%s: q %s, k %s and v %s do not fit together" % (what, tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("%s: q, k and v must have one type" % what)
    if not 1 <= head <= 128:
        raise ValueError("%s: heads of 1 to 128 values (and as many again in v) are supported" % what)
    if scale is not None and not abs(scale) <= _LARGEST:
        raise ValueError("%s: the scale must be a finite number of f32" % what)
    if heads % 2 or heads < 2 or kv_heads < 1 or heads // 2 % kv_heads:
        raise ValueError("%s: q has two maps a head, of as many heads as a multiple of the key/value heads" % what)
    t = _type(what, q)
    if weights.shape != (heads // 2,):
        raise ValueError("%s: weights has one value per head (%d), not the shape %s" % (what, heads // 2, tuple(weights.shape)))
    w = _type(what, weights)
    if w not in (t, 0):
        raise ValueError("%s: weights has the type of the values, or float32" % what)
    if key_lengths is not None and (key_lengths.shape != (batch,) or key_lengths.dtype not in (torch.int32, torch.int64)):
        raise ValueError("%s: key_lengths is one whole number per sequence" % what)
    if key_mask is not None and (key_mask.shape != (batch, keys) or key_mask.dtype not in (torch.bool, torch.uint8)):
        raise ValueError("%s: key_mask is one truth value per sequence and key" % what)
    return t, w, batch, queries, keys, heads // 2, kv_heads, head


@functools.lru_cache(maxsize=256)
def _differ_workspace(lib, backward, causal, *sizes):
    n = _INT64()
    d = _DIFFER.pack(*sizes, causal, 0.0, *[0] * 28)
    check((lib.nnvhip_differential_attention_backward_workspace if backward else lib.nnvhip_differential_attention_workspace)(d, C.byref(n)))
    return n.value


def differential_attention(q, k, v, weights, key_lengths=None, key_mask=None, causal=False, scale=None, for_backward=False, ctx=None):
    """softmax(scale * q0 k0^T) v - weights * softmax(scale * q1 k1^T) v: the difference of two attention maps, with a weight per head.

    q: batch x queries x 2 heads x head, the two maps' queries of a head one after the other (2 h and 2 h + 1); k: batch x keys x
    2 kv_heads x head, as well; v: batch x keys x kv_heads x 2 head; any strides; consecutive heads / kv_heads heads share keys and values; head is 128 at
    most.  weights: a vector of ``heads`` values of q's type or f32.  key_lengths and key_mask say which keys count, as in
    cross_attention: what the others hold is of no effect.  causal: query i of a sequence of n keys sees the keys in front of n - queries + i + 1 alone (the
    last query's place is the last key's); v should then be finite in the keys that count: zero weights of keys that are seen later are multiplied with it.  scale:
    1 / sqrt(head) if None.

    Returns (o, lse, second): o, batch x queries x heads x 2 head, of q's type; the logarithms of both maps' softmax sums, batch x 2 heads x queries, f32; and, if
    for_backward, the second map's softmax times v, in o's shape and type, else None.  A query that sees no key has the result 0 and the logarithm -inf.

    In 16 bits the maps' weights, and in the backward pass their difference and the gradients of the scores, go into their products in two pieces that hold all but 2^-16 of them (2^-22
    in f16), so that a result is off by its own rounding alone.  But rows that see more
    than 256 keys take D, the sum of do times each map's result, for dq from the o and second that were rounded: dq is mostly up to 1.1 times as far off as its rounding (0.0018 for 0.0017 in bf16), up
    to 1.4 times where a mask leaves few of the keys, and 2.5 times with heads of a few values."""
    what = "differential_attention"
    ctx, lib, stream = _enter(what, ctx, q, k, v, weights, key_lengths, key_mask)
    sizes = _differ_sizes(what, q, k, v, weights, key_lengths, key_mask, scale)
    t, w, batch, queries, keys, heads, kv_heads, head = sizes
    q, k, v, weights = _dense_values(q), _dense_values(k), _dense_values(v), _dense(weights)
    lengths, mask_stride = _mask_args(key_lengths, key_mask, keys)
    o = q.new_empty((batch, queries, heads, 2 * head))
    second = torch.empty_like(o) if for_backward else None
    lse = q.new_empty((batch, 2 * heads, queries), dtype=torch.float32)
    d = _DIFFER.pack(*sizes, bool(causal), head ** -0.5 if scale is None else scale, q.data_ptr(), k.data_ptr(), v.data_ptr(), *q.stride()[:3],
                     *k.stride()[:3], *v.stride()[:3], weights.data_ptr(), _ptr(lengths) or 0, _ptr(key_mask) or 0, *mask_stride, o.data_ptr(),
                     lse.data_ptr(), _ptr(second) or 0, 0, 0, 0, 0, 0, 0, 0, 0)
    need = _differ_workspace(lib, False, bool(causal), *sizes)
    work = q.new_empty((need,), dtype=torch.uint8) if need else None
    check(lib.nnvhip_differential_attention(ctx.handle, d, _ptr(work), need, stream))
    return o, lse, second


def differential_attention_backward(do, q, k, v, weights, o, lse, second, key_lengths=None, key_mask=None, causal=False, scale=None, ctx=None):
    """The gradients (dq, dk, dv, dweights) of differential_attention, from that of o and from what the forward call (with for_backward)
    returned; the other arguments are that call's.  Rows that see no key and keys that do not count get zero.  A value of q or do that is not finite reaches the
    gradients of all keys that count, and causal one of k those of queries that do not see it (zero weights are multiplied with them).  dweights has the type of weights."""
    what = "differential_attention_backward"
    ctx, lib, stream = _enter(what, ctx, q, k, v, weights, key_lengths, key_mask, do, o, lse, second)
    sizes = _differ_sizes(what, q, k, v, weights, key_lengths, key_mask, scale)
    t, w, batch, queries, keys, heads, kv_heads, head = sizes
    for x in (do, o, second):
        if x is None or x.shape != (batch, queries, heads, 2 * head) or x.dtype != q.dtype:
            raise ValueError("%s: do, o and second must have the shape and type of what differential_attention returned (for_backward)" % what)
    if lse.shape != (batch, 2 * heads, queries) or lse.dtype != torch.float32:
        raise ValueError("%s: lse must be what differential_attention returned" % what)
    q, k, v, do, weights = _dense_values(q), _dense_values(k), _dense_values(v), _dense_values(do), _dense(weights)
    o, lse, second = o.contiguous(), lse.contiguous(), second.contiguous()
    lengths, mask_stride = _mask_args(key_lengths, key_mask, keys)
    dq, dk, dv = (torch.empty_like(x, memory_format=torch.contiguous_format) for x in (q, k, v))
    dweights = torch.empty_like(weights)
    d = _DIFFER.pack(*sizes, bool(causal), head ** -0.5 if scale is None else scale, q.data_ptr(), k.data_ptr(), v.data_ptr(), *q.stride()[:3],
                     *k.stride()[:3], *v.stride()[:3], weights.data_ptr(), _ptr(lengths) or 0, _ptr(key_mask) or 0, *mask_stride, o.data_ptr(),
                     lse.data_ptr(), second.data_ptr(), do.data_ptr(), *do.stride()[:3], dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                     dweights.data_ptr())
    need = _differ_workspace(lib, True, bool(causal), *sizes)
    work = q.new_empty((need,), dtype=torch.uint8) if need else None
    check(lib.nnvhip_differential_attention_backward(ctx.handle, d, _ptr(work), need, stream))
    return dq, dk, dv, dweights


# ---- layers -------------------------------------------------------------------------------------


class GroupNormalizationLayer:
    """A group normalization over NumGroups groups of the channels (the last dimension) and all places, with an Activation behind it (None, "relu"
    or "silu"); properties as of the reference's normalization layers (nn/layers/BatchNormalizationLayer.m:33-83).  Scale and Offset are
    device tensors or None."""

    def __init__(self, NumGroups, **kw):
        self.Name = kw.get("Name", "GroupNormalizationLayer")
        self.NumGroups = int(NumGroups)
        self.Scale = kw.get("Scale")
        self.Offset = kw.get("Offset")
        self.Epsilon = float(kw.get("Epsilon", 0.00001))
        self.Activation = kw.get("Activation")
        known = [p for p in (self.Scale, self.Offset) if p is not None]
        self.NumChannels = kw.get("NumChannels") or (known[0].shape[0] if known else None)

    def evaluate(self, x):
        return self.forward(x)[0]

    def forward(self, x):
        """(y, what backward takes)."""
        if self.NumChannels is not None and x.shape[-1] != self.NumChannels:
            raise ValueError("Inconsistent number of channels between the input and the group normalization")
        y, mean, rstd = group_norm(x, self.NumGroups, self.Scale, self.Offset, self.Epsilon, self.Activation)
        return y, (x, mean, rstd)

    def backward(self, dy, saved):
        """(dx, [dScale, dOffset])."""
        x, mean, rstd = saved
        dx, dscale, doffset = group_norm_backward(dy, x, mean, rstd, self.Scale, self.Offset, self.Activation)
        return dx, [dscale, doffset]


class DifferentialAttentionLayer:
    """Differential attention of NumHeads heads (two maps each) to keys and values of NumKeyValueHeads (NumHeads if not given); Weights: the second map's
    weight in each head.  Inputs are batch x tokens x channels, the channels of all heads (and maps) side by side; with Sections, queries and keys are turned by the
    positions that go with them (rotate_positions, Rotary: its other arguments)."""

    def __init__(self, NumHeads, Weights, NumKeyValueHeads=None, Causal=False, Scale=None, Sections=None, Rotary=None, Name="DifferentialAttentionLayer"):
        self.Name = Name
        self.NumHeads = int(NumHeads)
        self.NumKeyValueHeads = int(NumKeyValueHeads or NumHeads)
        self.Weights = Weights
        self.Causal = bool(Causal)
        self.Scale = Scale
        self.Sections = None if Sections is None else tuple(Sections)
        self.Rotary = dict(Rotary or {})

    def _heads(self, x, heads):
        if x.dim() != 3 or x.shape[2] % heads:
            raise ValueError("The channels of the input must be a multiple of the number of heads and maps")
        return x.unflatten(2, (heads, x.shape[2] // heads))

    def _turn(self, q, k, q_positions, k_positions, inverse=False):
        if self.Sections is None:
            return q, k
        if q_positions is k_positions:
            return rotate_positions([q, k], q_positions, self.Sections, inverse=inverse, **self.Rotary)
        return tuple(rotate_positions(x, at, self.Sections, inverse=inverse, **self.Rotary) for x, at in ((q, q_positions), (k, k_positions)))

    def evaluate(self, q, k, v, q_positions=None, k_positions=None, key_lengths=None, key_mask=None):
        return self._forward(q, k, v, q_positions, k_positions, key_lengths, key_mask, False)[0]

    def forward(self, q, k, v, q_positions=None, k_positions=None, key_lengths=None, key_mask=None):
        """(o, what backward takes)."""
        return self._forward(q, k, v, q_positions, k_positions, key_lengths, key_mask, True)

    def _forward(self, q, k, v, q_positions, k_positions, key_lengths, key_mask, for_backward):
        if self.Sections is not None and (q_positions is None or k_positions is None):
            raise ValueError("Queries and keys that are turned need positions")
        q, k, v = self._heads(q, 2 * self.NumHeads), self._heads(k, 2 * self.NumKeyValueHeads), self._heads(v, self.NumKeyValueHeads)
        q, k = self._turn(q, k, q_positions, k_positions)
        masks = {"key_lengths": key_lengths, "key_mask": key_mask, "causal": self.Causal, "scale": self.Scale}
        o, lse, second = differential_attention(q, k, v, self.Weights, for_backward=for_backward, **masks)
        return o.flatten(2), (q, k, v, o, lse, second, q_positions, k_positions, masks)

    def backward(self, do, saved):
        """(dq, dk, dv, dWeights)."""
        q, k, v, o, lse, second, q_positions, k_positions, masks = saved
        dq, dk, dv, dweights = differential_attention_backward(self._heads(do, self.NumHeads), q, k, v, self.Weights, o, lse, second, **masks)
        dq, dk = self._turn(dq, dk, q_positions, k_positions, inverse=True)
        return dq.flatten(2), dk.flatten(2), dv.flatten(2), dweights
