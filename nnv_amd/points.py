"""Operators on points and gradients: layer normalization, attention to another sequence's states, and the global norm of
a list of gradients with its clipping.

Sets are what this package reaches; these are what a program runs beside them: a network with such layers is evaluated on
points of the input box, the gradient of a specification's margin is followed back to the input (see
``nnv_amd.falsify``) or to the weights, and the step is bounded.  The reference's layers evaluate points as well (e.g.
nn/layers/BatchNormalizationLayer.m:118-229); it has no gradients, and no counterpart of the two layers here in its reach path.

All arguments and results are torch tensors on one GPU, that of the context if one is given: f32, bf16 or f16.  A call is queued on torch's current
stream of that device, like torch's own operations, and returns without waiting; what it needs besides its results comes from torch's
allocator.  They are no part of torch's graph: where torch records gradients, tensors that
require one are refused.  The layers' sums and statistics are f32 (the gradient norm's squares f64), and each
result is rounded once; attention in 16 bits rounds the softmax's weights, and in bf16 the gradients of its scores, in front of the products that take
them, and its backward pass takes the o that was rounded.
"""
from __future__ import annotations

import ctypes as C
import functools
import operator
import struct

import torch

from ._lib import check, context_on, default_context

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_INT64 = C.c_int64


_requires_grad, _dtype = operator.attrgetter("requires_grad"), operator.attrgetter("dtype")
_records_gradients = torch.is_grad_enabled
_stream_of = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _not_recorded(what):
    return ValueError("%s: a tensor requires a gradient, which is not recorded here: call it under torch.no_grad() (the backward functions "
                      "form the gradients)" % what)


def _enter(what, ctx, first, *others):
    """(context, its library, stream) for tensors (others: or None) that have to be on that context's GPU; ctx None: the one of theirs."""
    try:
        index, recording = first.get_device(), _records_gradients()
        asked = recording and first.requires_grad
        for t in others:
            if t is not None:
                if t.get_device() != index:
                    raise ValueError("%s: the tensors must be on one GPU" % what)
                if recording and t.requires_grad:
                    asked = True
    except AttributeError:
        raise TypeError("%s: expected torch tensors, got %s" % (what, ", ".join(type(t).__name__ for t in (first, *others)))) from None
    if asked:
        raise _not_recorded(what)
    if index < 0:
        raise ValueError("%s: the tensors must be on the GPU" % what)
    ctx = ctx or context_on(index)
    if index != ctx.device:
        raise ValueError("%s: the tensors are on GPU %d, the context is GPU %d's" % (what, index, ctx.device))
    return ctx, ctx.lib, _stream_of(index)


def _type(what, t):
    k = _TYPES.get(t.dtype)
    if k is None:
        raise ValueError("%s: the values must be float32, bfloat16 or float16, not %s" % (what, t.dtype))
    return k


# ---- layer normalization ----------------------------------------------------------------------


def _as_rows(x, size):
    """(tensor, rows, stride of its rows): x as rows of its last dimension, copied only where they are not evenly spaced."""
    if x.is_contiguous():
        return x, x.numel() // size, size
    if x.stride(-1) == 1 or size == 1:
        try:
            rows = x.view(-1, size)
            return rows, rows.shape[0], rows.stride(0)
        except RuntimeError:
            pass
    x = x.contiguous()
    return x, x.numel() // size, size


def _norm_params(what, x, scale, offset):
    t = _type(what, x)
    size = x.shape[-1] if x.dim() else 0
    if size < 1:
        raise ValueError("%s: rows of at least one value are expected" % what)
    w = t
    for p in (scale, offset):
        if p is not None:
            if p.shape != (size,):
                raise ValueError("%s: scale and offset have one value per channel (%d), not the shape %s" % (what, size, tuple(p.shape)))
            w = _type(what, p)
            if w not in (t, 0):
                raise ValueError("%s: scale and offset have the type of the values, or float32" % what)
    if scale is not None and offset is not None and scale.dtype != offset.dtype:
        raise ValueError("%s: scale and offset must have the same type" % what)
    return t, w


def _ptr(t):
    return None if t is None else t.data_ptr()


def layer_norm(x, scale=None, offset=None, epsilon=1e-5, ctx=None):
    """y = (x - mean) / sqrt(var + epsilon) * scale + offset over the last dimension of x.

    Returns (y, mean, rstd): y in x's shape and type, the statistics f32, one per row, in x's leading shape;
    layer_norm_backward takes them.  scale and offset: vectors of x's type or f32, or None."""
    ctx, lib, stream = _enter("layer_norm", ctx, x, scale, offset)
    t, w = _norm_params("layer_norm", x, scale, offset)
    if not epsilon >= 0:
        raise ValueError("layer_norm: epsilon must not be negative")
    shape = x.shape
    lead, size = shape[:-1], shape[-1]
    if scale is not None and not scale.is_contiguous():
        scale = scale.contiguous()
    if offset is not None and not offset.is_contiguous():
        offset = offset.contiguous()
    rows_of, rows, stride = _as_rows(x, size)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    mean = x.new_empty(lead, dtype=torch.float32)
    rstd = torch.empty_like(mean)
    check(lib.nnvhip_layer_norm(ctx.handle, t, w, rows, size, rows_of.data_ptr(), stride, _ptr(scale), _ptr(offset), epsilon,
                                y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), stream))
    return y, mean, rstd


@functools.lru_cache(maxsize=256)
def _norm_workspace(lib, t, rows, size):
    n = _INT64()
    check(lib.nnvhip_layer_norm_backward_workspace(t, rows, size, C.byref(n)))
    return n.value


def layer_norm_backward(dy, x, mean, rstd, scale=None, ctx=None):
    """The gradients of layer_norm: (dx, dscale, doffset) from that of its result and its statistics.

    dx has x's type, dscale and doffset the type of scale (x's if scale is None)."""
    what = "layer_norm_backward"
    ctx, lib, stream = _enter(what, ctx, x, dy, mean, rstd, scale)
    t, w = _norm_params(what, x, scale, None)
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError("%s: dy must have the shape and type of x" % what)
    lead, size = x.shape[:-1], x.shape[-1]
    for s in (mean, rstd):
        if s.shape != lead or s.dtype != torch.float32:
            raise ValueError("%s: mean and rstd must be what layer_norm returned" % what)
    scale = scale if scale is None else scale.contiguous()
    mean, rstd = mean.contiguous(), rstd.contiguous()
    xr, rows, xs = _as_rows(x, size)
    gr, _, gs = _as_rows(dy, size)
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    dscale = (x if scale is None else scale).new_empty((size,))
    doffset = torch.empty_like(dscale)
    need = _norm_workspace(lib, t, rows, size)
    work = x.new_empty((need,), dtype=torch.uint8) if need else None
    check(lib.nnvhip_layer_norm_backward(ctx.handle, t, w, rows, size, gr.data_ptr(), gs, xr.data_ptr(), xs, mean.data_ptr(),
                                         rstd.data_ptr(), _ptr(scale), dx.data_ptr(), dscale.data_ptr(), doffset.data_ptr(),
                                         _ptr(work), need, stream))
    return dx, dscale, doffset


# ---- attention to another sequence's states ---------------------------------------------------------

# struct nnvhip_attention
_ATTENTION = struct.Struct("=7qd3Q9qQQ2qQQQ3q3Q")


def _dense_values(t):
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


_LARGEST = 3.4028234663852886e38   # of f32


def _attention_sizes(what, q, k, v, key_lengths, key_mask, scale):
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("%s: q, k and v are batch x tokens x heads x head" % what)
    if k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError("%s: q %s, k %s and v %s do not fit together" % (what, tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("%s: q, k and v must have one type" % what)
    batch, queries, heads, head = q.shape
    keys, kv_heads = k.shape[1], k.shape[2]
    if not 1 <= head <= 128:
        raise ValueError("%s: heads of 1 to 128 values are supported" % what)
    if scale is not None and not abs(scale) <= _LARGEST:
        raise ValueError("%s: the scale must be a finite number of f32" % what)
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError("%s: the number of heads must be a multiple of the number of key/value heads" % what)
    if key_lengths is not None and (key_lengths.shape != (batch,) or key_lengths.dtype not in (torch.int32, torch.int64)):
        raise ValueError("%s: key_lengths is one whole number per sequence" % what)
    if key_mask is not None and (key_mask.shape != (batch, keys) or key_mask.dtype not in (torch.bool, torch.uint8)):
        raise ValueError("%s: key_mask is one truth value per sequence and key" % what)
    return _type(what, q), batch, queries, keys, heads, kv_heads, head


@functools.lru_cache(maxsize=256)
def _attention_workspace(lib, backward, *sizes):
    n = _INT64()
    d = _ATTENTION.pack(*sizes, 0.0, *[0] * 25)
    fn = lib.nnvhip_cross_attention_backward_workspace if backward else lib.nnvhip_cross_attention_workspace
    check(fn(d, C.byref(n)))
    return n.value


def _mask_args(key_lengths, key_mask, keys):
    if key_lengths is not None and (key_lengths.dtype != torch.int32 or not key_lengths.is_contiguous()):
        if key_lengths.dtype != torch.int32:   # beyond what 32 bits hold: as beyond the keys
            key_lengths = key_lengths.clamp(0, keys)
        key_lengths = key_lengths.to(torch.int32).contiguous()
    return key_lengths, (key_mask.stride() if key_mask is not None else (0, 0))


def cross_attention(q, k, v, key_lengths=None, key_mask=None, scale=None, ctx=None):
    """softmax(scale * q k^T) v for queries of one sequence and keys and values of another.

    q: batch x queries x heads x head, k and v: batch x keys x kv_heads x head, any strides; consecutive heads / kv_heads
    heads share keys and values; head is 128 at most.  key_lengths (one number per sequence; beyond [0, keys]
    it is taken as that bound) and key_mask (truth values, batch x keys) say which keys count; what the others hold is of no effect.  scale: 1 / sqrt(head) if None.

    Returns (o, lse): o in q's shape and type and the logarithm of the softmax's sums, batch x heads x queries, f32.
    Where no key counts o is zero and lse -inf."""
    what = "cross_attention"
    ctx, lib, stream = _enter(what, ctx, q, k, v, key_lengths, key_mask)
    sizes = _attention_sizes(what, q, k, v, key_lengths, key_mask, scale)
    q, k, v = _dense_values(q), _dense_values(k), _dense_values(v)
    lengths, mask_stride = _mask_args(key_lengths, key_mask, sizes[3])
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = q.new_empty((sizes[1], sizes[4], sizes[2]), dtype=torch.float32)
    d = _ATTENTION.pack(*sizes, sizes[6] ** -0.5 if scale is None else scale, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                        *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], _ptr(lengths) or 0, _ptr(key_mask) or 0,
                        *mask_stride, o.data_ptr(), lse.data_ptr(), 0, 0, 0, 0, 0, 0, 0)
    need = _attention_workspace(lib, False, *sizes)
    work = q.new_empty((need,), dtype=torch.uint8) if need else None
    check(lib.nnvhip_cross_attention(ctx.handle, d, _ptr(work), need, stream))
    return o, lse


def cross_attention_backward(do, q, k, v, o, lse, key_lengths=None, key_mask=None, scale=None, ctx=None):
    """The gradients (dq, dk, dv) of cross_attention, from that of o and from what the forward call returned; the other
    arguments are that call's.  Rows without keys and keys that do not count get zero."""
    what = "cross_attention_backward"
    ctx, lib, stream = _enter(what, ctx, q, k, v, key_lengths, key_mask, do, o, lse)
    sizes = _attention_sizes(what, q, k, v, key_lengths, key_mask, scale)
    if do.shape != q.shape or do.dtype != q.dtype or o.shape != q.shape or o.dtype != q.dtype:
        raise ValueError("%s: do and o must have the shape and type of q" % what)
    if lse.shape != (sizes[1], sizes[4], sizes[2]) or lse.dtype != torch.float32:
        raise ValueError("%s: lse must be what cross_attention returned" % what)
    q, k, v, do = _dense_values(q), _dense_values(k), _dense_values(v), _dense_values(do)
    o, lse = o.contiguous(), lse.contiguous()
    lengths, mask_stride = _mask_args(key_lengths, key_mask, sizes[3])
    dq, dk, dv = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))
    d = _ATTENTION.pack(*sizes, sizes[6] ** -0.5 if scale is None else scale, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                        *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], _ptr(lengths) or 0, _ptr(key_mask) or 0,
                        *mask_stride, o.data_ptr(), lse.data_ptr(), do.data_ptr(), *do.stride()[:3], dq.data_ptr(),
                        dk.data_ptr(), dv.data_ptr())
    need = _attention_workspace(lib, True, *sizes)
    work = q.new_empty((need,), dtype=torch.uint8) if need else None
    check(lib.nnvhip_cross_attention_backward(ctx.handle, d, _ptr(work), need, stream))
    return dq, dk, dv


# ---- the norm of all gradients, and clipping ---------------------------------------------------------


@functools.lru_cache(maxsize=64)
def _clip_plan(lib, count):
    """(bytes of the workspace, what packs the four arrays of a call, where the second one begins)."""
    n = _INT64()
    check(lib.nnvhip_clip_gradients_workspace(count, C.byref(n)))
    return n.value, struct.Struct("=%di%dx%dq%dQ%dQ" % (count, count % 2 * 4, count, count, count)).pack, (count + count % 2) * 4


def _all_tensors(values):   # (a set of few members takes a fifth of the time of a loop)
    return set(map(type, values)) == {torch.Tensor} or all(isinstance(v, torch.Tensor) for v in values)


def clip_gradients(gradients, threshold, out=None, ctx=None):
    """The tensors of a list scaled so that the norm over all of them is at most threshold:
    out[k] = gradients[k] * (norm > threshold ? threshold / norm : 1), norm = sqrt(sum of all squares).

    Returns (the scaled tensors, norm as an f32 tensor of no dimensions); the norm stays on the GPU.  out: tensors of the same shapes
    and types to write to, e.g. the gradients themselves, none of which may share memory with another; new ones if None.  A norm beyond f32 is told as infinite, and
    clipped as what it is; one that is infinite, by an infinite gradient, gives zeros and NaNs, and one that is no number leaves the
    gradients as they are."""
    what = "clip_gradients"
    gradients = list(gradients)
    if not threshold > 0:
        raise ValueError("%s: the threshold must be positive" % what)
    if not gradients:
        ctx = ctx or default_context()
        return [], torch.zeros((), dtype=torch.float32, device=torch.device("cuda", ctx.device))
    ctx, lib, stream = _enter(what, ctx, gradients[0])
    device = gradients[0].device
    fresh = out is None
    tensor, index, strided = torch.Tensor, device.index, []
    if not _all_tensors(gradients):
        raise TypeError("%s: expected torch tensors" % what)
    result = [torch.empty(g.shape, dtype=g.dtype, device=device) for g in gradients] if fresh else list(out)
    count = len(gradients)
    if len(result) != count:
        raise ValueError("%s: %d gradients and %d tensors to write to" % (what, count, len(result)))
    dtypes = list(map(_dtype, gradients))
    if set(map(tensor.get_device, gradients)) != {index}:
        raise ValueError("%s: the tensors must be on one GPU" % what)
    if not fresh:
        if not _all_tensors(result) or set(map(tensor.get_device, result)) != {index} or list(map(_dtype, result)) != dtypes or \
                not all(map(tensor.is_same_size, result, gradients)):
            raise ValueError("%s: out must have the shapes, types and device of the gradients" % what)
    if _records_gradients() and (any(map(_requires_grad, gradients)) or not fresh and any(map(_requires_grad, result))):
        raise _not_recorded(what)
    types = list(map(_TYPES.get, dtypes))
    if None in types:
        _type(what, gradients[types.index(None)])
    dense, to = gradients, result
    if not all(map(tensor.is_contiguous, gradients)):
        dense = [g.contiguous() for g in gradients]
    if not all(map(tensor.is_contiguous, result)):   # through dense tensors, copied back below
        to = [y if y.is_contiguous() else torch.empty(y.shape, dtype=y.dtype, device=device) for y in result]
        strided = [(y, t) for y, t in zip(result, to) if y is not t]
    sizes, source, target = map(tensor.numel, dense), map(tensor.data_ptr, dense), map(tensor.data_ptr, to)
    norm = torch.empty((), dtype=torch.float32, device=device)
    need, pack, second = _clip_plan(lib, count)
    work = torch.empty(need, dtype=torch.uint8, device=device)
    at = C.addressof(C.c_char.from_buffer(held := bytearray(pack(*types, *sizes, *source, *target))))
    longs = at + second
    check(lib.nnvhip_clip_gradients(ctx.handle, count, at, longs, longs + 8 * count, longs + 16 * count, threshold, norm.data_ptr(),
                                    work.data_ptr(), need, stream))
    del held
    for y, t in strided:
        y.copy_(t)
    return result, norm


# ---- layers -------------------------------------------------------------------------------------


class LayerNormalizationLayer:
    """A layer normalization over the channels (the last dimension), with the properties of the reference's normalization layers
    (name/value constructor, nn/layers/BatchNormalizationLayer.m:33-83).  Scale and Offset are device tensors or None."""

    def __init__(self, **kw):
        self.Name = kw.get("Name", "LayerNormalizationLayer")
        self.Scale = kw.get("Scale")
        self.Offset = kw.get("Offset")
        self.Epsilon = float(kw.get("Epsilon", 0.00001))
        known = [p for p in (self.Scale, self.Offset) if p is not None]
        self.NumChannels = kw.get("NumChannels") or (known[0].shape[0] if known else None)

    def _check(self, x):
        if self.NumChannels is not None and x.shape[-1] != self.NumChannels:
            raise ValueError("Inconsistent number of channels between the input and the layer normalization")

    def evaluate(self, x):
        return self.forward(x)[0]

    def forward(self, x):
        """(y, what backward takes)."""
        self._check(x)
        y, mean, rstd = layer_norm(x, self.Scale, self.Offset, self.Epsilon)
        return y, (x, mean, rstd)

    def backward(self, dy, saved):
        """(dx, [dScale, dOffset])."""
        x, mean, rstd = saved
        dx, dscale, doffset = layer_norm_backward(dy, x, mean, rstd, self.Scale)
        return dx, [dscale, doffset]


class CrossAttentionLayer:
    """Attention of NumHeads heads to another sequence's keys and values (NumKeyValueHeads of them, NumHeads if not given);
    inputs are batch x tokens x channels, the channels of all heads side by side."""

    def __init__(self, NumHeads, NumKeyValueHeads=None, Scale=None, Name="CrossAttentionLayer"):
        self.Name = Name
        self.NumHeads = int(NumHeads)
        self.NumKeyValueHeads = int(NumKeyValueHeads or NumHeads)
        self.Scale = Scale

    def _heads(self, x, heads):
        if x.dim() != 3 or x.shape[2] % heads:
            raise ValueError("The channels of the input must be a multiple of the number of heads")
        return x.unflatten(2, (heads, x.shape[2] // heads))

    def evaluate(self, q, k, v, key_lengths=None, key_mask=None):
        return self.forward(q, k, v, key_lengths, key_mask)[0]

    def forward(self, q, k, v, key_lengths=None, key_mask=None):
        """(o, what backward takes)."""
        q = self._heads(q, self.NumHeads)
        k, v = (self._heads(x, self.NumKeyValueHeads) for x in (k, v))
        o, lse = cross_attention(q, k, v, key_lengths, key_mask, self.Scale)
        return o.flatten(2), (q, k, v, o, lse, key_lengths, key_mask)

    def backward(self, do, saved):
        """(dq, dk, dv)."""
        q, k, v, o, lse, key_lengths, key_mask = saved
        return tuple(g.flatten(2) for g in cross_attention_backward(self._heads(do, self.NumHeads), q, k, v, o, lse, key_lengths,
                                                                    key_mask, self.Scale))
