"""The operators on points that are images or videos (nnv_amd.images) on the GPU against plain 64-bit forms, at the sizes, strides and
values where they can go wrong."""
import math

import numpy as np
import pytest
import torch

from tests import images_oracle as io
from tests import points_oracle as po

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES, IDS = [F32, BF16, F16], ["f32", "bf16", "f16"]
ACTIVATIONS = [None, "relu", "silu"]


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=F32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)


# ---- group normalization ------------------------------------------------------------------------


def check_group(x, groups, w, b, activation, seed=1, backward=True, tag=""):
    import nnv_amd as nnv
    y, mean, rstd = nnv.group_norm(x, groups, w, b, 1e-5, activation)
    assert y.dtype == x.dtype and y.shape == x.shape and mean.shape == rstd.shape == (x.shape[0], groups)
    for name, got, e, bd in zip(("y", "mean", "rstd"), (y, mean, rstd), io.group(x, groups, w, b, 1e-5, activation),
                                io.group_bounds(x, groups, w, b, 1e-5, activation)):
        po.assert_within(got, e, bd, tag + " " + name)
    if not backward:
        return
    dy = rand(gen(seed), *x.shape, dtype=x.dtype)
    grads = nnv.group_norm_backward(dy, x, mean, rstd, w, b, activation)
    pt = w.dtype if w is not None else b.dtype if b is not None else x.dtype
    assert [t.dtype for t in grads] == [x.dtype, pt, pt]
    for name, got, e, bd in zip(("dx", "dscale", "doffset"), grads, io.group_grad(dy, x, mean, rstd, w, b, activation),
                                io.group_grad_bounds(dy, x, mean, rstd, w, b, activation)):
        po.assert_within(got, e, bd, tag + " " + name)


# batch, places, channels, groups: one place, one channel a group, packs that end inside a group, chunks of several groups and
# groups of several chunks, parts of the places that do not come out even
GROUP_SIZES = [(1, (1,), 8, 2), (2, (1, 1), 64, 64), (3, (5,), 1, 1), (2, (7, 3), 6, 3), (1, (64, 64), 10, 1), (4, (8, 8), 256, 32), (2, (33, 17), 70, 7),
               (1, (9,), 1030, 515), (2, (13,), 1024, 1), (2, (11, 5), 2056, 2), (1, (301,), 5000, 4), (3, (50, 41), 96, 8), (1, (128, 130), 40, 8),
               (65, (10,), 24, 4), (2, (3, 5, 7), 132, 11), (1, (70001,), 3, 1)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("size", GROUP_SIZES, ids=lambda s: "%dx%sx%d/%d" % (s[0], "x".join(map(str, s[1])), s[2], s[3]))
def test_group_norm_forward_and_backward(size, dtype):
    batch, places, channels, groups = size
    g = gen(channels + batch)
    x = rand(g, batch, *places, channels, dtype=dtype, scale=1.5, shift=2.0)
    for k, activation in enumerate(ACTIVATIONS):
        for pt in {dtype, F32}:
            w, b = rand(g, channels, dtype=pt, shift=1.0), rand(g, channels, dtype=pt)
            check_group(x, groups, w, b, activation, seed=k, tag="%s %s" % (activation, pt))
    check_group(x, groups, None, None, "silu")
    check_group(x, groups, None, rand(g, channels, dtype=dtype), "relu")


def test_group_norm_of_views():
    """Places that lie apart, channels of a wider tensor, images whose channels come first in memory, an odd start; one sequence for all."""
    g = gen(7)
    wide = rand(g, 3, 6, 10, 72, dtype=BF16)
    w, b = rand(g, 40, shift=1.0), rand(g, 40)
    for view in (wide[..., 5:45], wide[:, :, ::2, 32:], wide[:, 1:, :, :40], wide[::2, ..., 1:41], wide[:1, ..., 8:48].expand(4, -1, -1, -1),
                 wide.permute(0, 3, 1, 2)[:, :40].permute(0, 2, 3, 1), rand(g, 3, 40, 5, 9, dtype=BF16).permute(0, 2, 3, 1),
                 rand(g, 6, 10, 40, 3, dtype=BF16).permute(3, 0, 1, 2)):
        check_group(view, 8, w, b, "silu")
    import nnv_amd as nnv
    x, dy = wide[..., :40], rand(g, 3, 40, 6, 10, dtype=BF16).permute(0, 2, 3, 1)
    _, mean, rstd = nnv.group_norm(x, 5, w[:40], b[:40])
    strided = torch.stack([mean, rstd], -1)
    got = nnv.group_norm_backward(dy, x, strided[..., 0], strided[..., 1], torch.stack([w, b], -1)[:, 0], b)
    for name, a, e in zip(("dx", "dscale", "doffset"), got, nnv.group_norm_backward(dy.contiguous(), x.contiguous(), mean, rstd, w, b)):
        assert torch.equal(a, e), name


def test_group_norm_of_no_sequences():
    import nnv_amd as nnv
    x = torch.empty(0, 4, 5, 24, device="cuda", dtype=F16)
    w = torch.ones(24, device="cuda")
    y, mean, rstd = nnv.group_norm(x, 4, w, w)
    assert y.shape == x.shape and mean.shape == (0, 4)
    dx, dw, db = nnv.group_norm_backward(x, x, mean, rstd, w, w, "silu")
    assert dx.shape == x.shape and float(dw.abs().sum() + db.abs().sum()) == 0


def test_group_norm_of_constant_infinite_missing_and_far_values():
    import nnv_amd as nnv
    x = torch.full((3, 40, 16), 7.25, device="cuda")
    x[1, 3, 5] = math.inf
    x[2, 39, 15] = math.nan
    b = torch.arange(16.0, device="cuda") - 8
    y, mean, rstd = nnv.group_norm(x, 4, None, b, 1e-5)
    assert torch.equal(y[0], b.expand(40, 16)) and (mean[0] == 7.25).all()      # no spread: the offset alone, exactly
    assert torch.isnan(y[1, :, 4:8]).all() and torch.isnan(y[2, :, 12:]).all()   # a group without a mean, and none but it
    assert torch.equal(y[1, :, :4], y[0, :, :4]) and torch.equal(y[1, :, 8:], y[0, :, 8:]) and torch.equal(y[2, :, :12], y[0, :, :12])
    y = nnv.group_norm(x, 4, None, b, 1e-5, "relu")[0]
    assert torch.isnan(y[1, :, 4:8]).all() and torch.equal(y[0], b.clamp(min=0).expand(40, 16))
    # large values next to a small spread, and activations far out on both sides
    far = 1e4 + torch.arange(640.0, device="cuda").view(1, 40, 16) / 64
    check_group(far, 2, None, None, None)
    w = torch.linspace(-200, 200, 16, device="cuda")
    check_group(rand(gen(3), 2, 40, 16), 2, w, b, "silu")


def test_the_side_of_zero_is_decided_exactly():
    """A gradient passes where z > 0: offsets that put z within a few roundings of zero on either side."""
    import nnv_amd as nnv
    g = gen(9)
    x = rand(g, 2, 300, 32)
    _, mean, rstd = nnv.group_norm(x, 4)
    w = rand(g, 32, shift=2.0)
    at = (x[0, 17].double() - mean[0].double().repeat_interleave(8)) * rstd[0].double().repeat_interleave(8) * w.double()
    dy = rand(g, 2, 300, 32)
    for steps in (-2, -1, 0, 1, 2):
        b = (-at).float()
        b = b + steps * b.abs() * 2.0 ** -24
        dx, dw, db = nnv.group_norm_backward(dy, x, mean, rstd, w, b, "relu")
        for name, got, e, bd in zip(("dx", "dscale", "doffset"), (dx, dw, db), io.group_grad(dy, x, mean, rstd, w, b, "relu"),
                                    io.group_grad_bounds(dy, x, mean, rstd, w, b, "relu")):
            po.assert_within(got, e, bd, "%d %s" % (steps, name))


@pytest.mark.parametrize("activation", ACTIVATIONS)
def test_group_norm_gradient_against_differences(activation):
    import nnv_amd as nnv
    g = gen(11)
    x, w, b, dy = rand(g, 2, 37, 24), rand(g, 24), rand(g, 24), rand(g, 2, 37, 24)
    _, mean, rstd = nnv.group_norm(x, 3, w, b)
    grads = nnv.group_norm_backward(dy, x, mean, rstd, w, b, activation)
    bounds = io.group_grad_bounds(dy, x, mean, rstd, w, b, activation)
    h = 1e-7   # (a step of relu's z across zero changes the difference by h at most, of a few of some thousand values)
    for k, t in enumerate((x, w, b)):
        d = torch.randn(t.shape, generator=g, device="cuda", dtype=torch.float64)

        def loss(s):
            at = [u.double() + (s * d if i == k else 0) for i, u in enumerate((x, w, b))]
            return float((io.group(at[0], 3, at[1], at[2], 1e-5, activation)[0] * dy.double()).sum())

        slope = (loss(h) - loss(-h)) / (2 * h)
        size = float((grads[k].double().abs() * d.abs()).sum())
        # the kernel's rounding, that of the statistics it was handed, and the differences' own: 2^-53 of sums of some 1e3, over h
        allowed = float(((bounds[k] + po.U32 * grads[k].double().abs()) * d.abs()).sum()) + 1e-5 * size + 1e-5
        assert abs(float((grads[k].double() * d).sum()) - slope) <= allowed


def test_group_norm_gives_the_same_bits_again():
    import nnv_amd as nnv
    g = gen(12)
    x, dy, w, b = rand(g, 7, 61, 43, 64, dtype=BF16), rand(g, 7, 61, 43, 64, dtype=BF16), rand(g, 64), rand(g, 64)
    one = nnv.group_norm(x, 8, w, b, activation="silu")
    for a, e in zip(one, nnv.group_norm(x, 8, w, b, activation="silu")):
        assert torch.equal(a, e)
    for a, e in zip(*(nnv.group_norm_backward(dy, x, one[1], one[2], w, b, "silu") for _ in range(2))):
        assert torch.equal(a, e)


# ---- rotary positions ---------------------------------------------------------------------------

# head, sections: full and partly turned heads, packs that hold the end of the pairs, sections of no pairs, odd heads
HEADS = [(128, (16, 24, 24)), (64, (32,)), (80, (16, 16)), (40, (7, 13)), (32, (3, 0, 5)), (96, (48, 0)), (6, (1, 1)), (7, (3,)), (2, (1,)), (17, (2, 1, 1, 2)), (512, (100, 156))]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("head,sections", HEADS, ids=lambda s: str(s).replace(" ", ""))
def test_rotary_positions(head, sections, dtype):
    import nnv_amd as nnv
    g = gen(head)
    for batch, tokens, heads in ((2, 5, (3, 1)), (1, 1, (8,)), (3, 67, (2, 2, 5, 1, 4)), (1, 1300, (1, 2))):
        xs = [rand(g, batch, tokens, h, head, dtype=dtype) for h in heads]
        at = torch.randint(0, 5000, (batch, tokens, len(sections)), generator=g, device="cuda", dtype=torch.int32)
        for shared, interleaved, inverse in ((False, False, False), (True, True, False), (True, False, True), (False, True, True)):
            got = nnv.rotate_positions(xs, at, sections, shared=shared, interleaved=interleaved, inverse=inverse)
            assert len(got) == len(xs)
            for x, y in zip(xs, got):
                assert y.dtype == dtype and y.is_contiguous()
                po.assert_within(y, io.rotate(x, at, sections, 10000.0, shared, interleaved, inverse),
                                 io.rotate_bounds(x, at, sections, 10000.0, shared, interleaved), "%d x %d" % (batch, tokens))
                assert torch.equal(y[..., 2 * sum(sections):], x[..., 2 * sum(sections):])


def test_rotary_positions_of_every_type_far_away_and_shared():
    import nnv_amd as nnv
    g = gen(5)
    x = rand(g, 2, 9, 4, 32)
    for at in (torch.randint(-2**31, 2**31 - 1, (9, 2), generator=g, device="cuda").int(), torch.randint(-2**40, 2**40, (2, 9, 2), generator=g, device="cuda"),
               torch.rand(9, 2, generator=g, device="cuda") * 1e6 - 5e5, torch.zeros(9, 2, device="cuda", dtype=torch.int64)):
        y = nnv.rotate_positions(x, at, [6, 9], base=500.0)
        assert torch.is_tensor(y)
        po.assert_within(y, io.rotate(x, at, [6, 9], 500.0), io.rotate_bounds(x, at, [6, 9], 500.0), str(at.dtype))
        if not at.any():
            assert torch.equal(y, x)
    # views: heads before tokens, every other token, a part of a wider projection, positions with strides of their own
    wide, at = rand(g, 2, 4, 18, 3 * 40, dtype=F16), torch.randint(0, 900, (3, 18, 2), generator=g, device="cuda")
    for view, where in ((wide[..., 40:80].transpose(1, 2), at[:2]), (wide[:, :, ::2, 7:47].transpose(1, 2), at[0, ::2]),
                        (wide.transpose(1, 2)[:, :, :1, 1:41].expand(-1, -1, 5, -1), at[1]), (wide.permute(0, 2, 3, 1)[:, :, ::3], at.flip(2)[1:])):
        sections = [view.shape[3] // 4, view.shape[3] // 4]
        po.assert_within(nnv.rotate_positions(view, where, sections), io.rotate(view, where, sections), io.rotate_bounds(view, where, sections), "view")
    for empty in (x[:0], x[:, :0], x[:, :, :0]):
        assert nnv.rotate_positions(empty, torch.zeros(empty.shape[1], 1, device="cuda"), [4]).shape == empty.shape


def test_rotating_back_is_the_gradient():
    """<rotate(x), y> = <x, rotate back(y)>, and lengths stay."""
    import nnv_amd as nnv
    g = gen(6)
    x, y = rand(g, 2, 33, 3, 64), rand(g, 2, 33, 3, 64)
    at = torch.randint(0, 10000, (33, 3), generator=g, device="cuda")
    for kw in (dict(shared=True), dict(interleaved=True)):
        r, back = nnv.rotate_positions(x, at, [8, 12, 12], **kw), nnv.rotate_positions(y, at, [8, 12, 12], inverse=True, **kw)
        one, two = float((r.double() * y.double()).sum()), float((x.double() * back.double()).sum())
        # each value is off by the bound of both turns and a rounding
        off = float(((io.rotate_bounds(x, at, [8, 12, 12], **kw) + po.U32 * r.abs()) * y.abs()).sum() +
                    ((io.rotate_bounds(y, at, [8, 12, 12], **kw) + po.U32 * back.abs()) * x.abs()).sum())
        assert abs(one - two) <= off


# ---- streams and graphs -------------------------------------------------------------------------


def test_images_on_another_stream_and_in_a_graph():
    import nnv_amd as nnv
    g = gen(21)
    x, dy, w, b = rand(g, 4, 20, 30, 64, dtype=BF16), rand(g, 4, 20, 30, 64, dtype=BF16), rand(g, 64), rand(g, 64)
    at = torch.randint(0, 100, (600, 2), generator=g, device="cuda", dtype=torch.int32)

    def step():
        y, mean, rstd = nnv.group_norm(x, 8, w, b, activation="silu")
        q = nnv.rotate_positions(y.view(4, 600, 2, 32), at, [8, 8])
        back = nnv.rotate_positions(q, at, [8, 8], inverse=True)
        return [y, mean, rstd, q, back, *nnv.group_norm_backward(dy, x, mean, rstd, w, b, "silu")]

    eager = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for a, e in zip(other, eager):
        assert torch.equal(a, e)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        x.copy_(rand(gen(100 + k), 4, 20, 30, 64, dtype=BF16))
        graph.replay()
        fresh = step()
        torch.cuda.synchronize()
        for a, e in zip(held, fresh):
            assert torch.equal(a, e)


# ---- differential attention ---------------------------------------------------------------------


def make_differ(g, b, lq, lk, h, hkv, d, dtype, weight_dtype=None):
    return (rand(g, b, lq, 2 * h, d, dtype=dtype), rand(g, b, lk, 2 * hkv, d, dtype=dtype), rand(g, b, lk, hkv, 2 * d, dtype=dtype),
            rand(g, h, dtype=weight_dtype or dtype, scale=0.3, shift=0.5))


def check_differ(q, k, v, w, backward=True, tag="", **kw):
    import nnv_amd as nnv
    o, lse, second = nnv.differential_attention(q, k, v, w, for_backward=backward, **kw)
    assert o.dtype == q.dtype and (second is None) == (not backward)
    exact, bounds = io.differ(q, k, v, w, **kw), io.differ_bounds(q, k, v, w, **kw)
    for name, got, e, bd in zip(("o", "lse", "second"), (o, lse, second), exact, bounds):
        if got is not None:
            po.assert_within(got, e, bd, tag + " " + name)
    if not backward:
        return o, lse
    do = rand(gen(q.shape[1]), *o.shape, dtype=q.dtype)
    grads = nnv.differential_attention_backward(do, q, k, v, w, o, lse, second, **kw)
    for name, t, got, e, bd in zip(("dq", "dk", "dv", "dweights"), (q, k, v, w), grads, io.differ_grad(do, q, k, v, w, **kw),
                                   io.differ_grad_bounds(do, q, k, v, w, **kw)):
        assert got.dtype == t.dtype and got.shape == t.shape
        po.assert_within(got, e, bd, tag + " " + name)
    return o, lse


# batch, queries, keys, heads, key/value heads, head: single tokens, one key, tiles that do not come out even, rows of several heads in a tile, every template
DIFFER_SIZES = [(1, 1, 1, 1, 1, 8), (2, 1, 33, 4, 4, 64), (3, 1, 700, 8, 2, 128), (1, 1, 5000, 16, 1, 32), (2, 3, 17, 3, 1, 16), (1, 64, 64, 2, 2, 64), (2, 65, 63, 2, 1, 40),
                (1, 130, 257, 4, 2, 80), (1, 33, 129, 6, 3, 96), (2, 100, 300, 2, 2, 128), (1, 70, 90, 2, 1, 112), (1, 40, 50, 2, 2, 7), (1, 31, 65, 3, 3, 33), (1, 20, 45, 2, 1, 50),
                (1, 17, 40, 2, 2, 90), (1, 19, 21, 2, 2, 126), (1, 300, 290, 1, 1, 64), (2, 5, 4000, 4, 4, 48), (1, 16, 64, 20, 4, 24), (1, 513, 40, 2, 1, 72)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("size", DIFFER_SIZES, ids=lambda s: "x".join(map(str, s)))
def test_differential_attention(size, dtype):
    b, lq, lk, h, hkv, d = size
    g = gen(sum(size))
    q, k, v, w = make_differ(g, *size, dtype)
    check_differ(q, k, v, w, tag="all")
    check_differ(q, k, v, w, causal=True, tag="causal")
    lengths = torch.randint(0, lk + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    lengths[0] = lk - lk // 3
    mask = torch.rand(b, lk, generator=g, device="cuda") < 0.8
    check_differ(q, k, v, w.float(), key_lengths=lengths, causal=True, tag="lengths, causal")
    check_differ(q, k, v, w, key_lengths=lengths, key_mask=mask, tag="lengths, mask")
    check_differ(q, k, v, w, key_mask=mask, causal=True, scale=-0.3, tag="mask, causal")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_differential_attention_without_keys_and_past_the_last(dtype):
    """Rows that see no key, and what lies in keys that do not count: zeros, -inf, and no trace of it."""
    import nnv_amd as nnv
    for d, lq in ((64, 70), (128, 70), (40, 1), (48, 5), (33, 20)):
        g = gen(d)
        q, k, v, w = make_differ(g, 4, lq, 150, 4, 2, d, dtype)
        lengths = torch.tensor([0, 150, 40, 67], device="cuda")
        mask = torch.ones(4, 150, device="cuda", dtype=torch.bool)
        mask[1] = False
        mask[3, 5:60] = False
        clean_k, clean_v = k.clone(), v.clone()
        for i, n in enumerate((0, 0, 40, 67)):
            k[i, n:], v[i, n:] = math.nan, math.inf
        k[3, 5:60], v[3, 5:60] = -math.inf, math.nan
        for causal in (False, True):
            kw = dict(key_lengths=lengths, key_mask=mask, causal=causal)
            o, lse, second = nnv.differential_attention(q, k, v, w, for_backward=True, **kw)
            for name, got, e, bd in zip(("o", "lse", "second"), (o, lse, second), io.differ(q, clean_k, clean_v, w, **kw), io.differ_bounds(q, clean_k, clean_v, w, **kw)):
                po.assert_within(got, e, bd, name)
            assert (o[:2] == 0).all() and (lse[:2] == -math.inf).all()
            do = rand(g, *o.shape, dtype=dtype)
            # what rows without keys hold reaches no gradient either
            q2, do2 = q.clone(), do.clone()
            q2[:2], do2[:2] = math.nan, math.inf
            if causal and lq > 40:
                q2[2, :lq - 40], do2[2, :lq - 40] = math.inf, math.nan
            for name, got, e, bd in zip(("dq", "dk", "dv", "dweights"), nnv.differential_attention_backward(do2, q2, k, v, w, o, lse, second, **kw),
                                        io.differ_grad(do, q, clean_k, clean_v, w, **kw), io.differ_grad_bounds(do, q, clean_k, clean_v, w, **kw)):
                po.assert_within(got, e, bd, "%s %s" % (causal, name))


def test_differential_attention_of_nothing():
    import nnv_amd as nnv
    for b, lq, lk in ((0, 5, 7), (2, 0, 7), (2, 5, 0)):
        q, k, v, w = make_differ(gen(1), b, lq, lk, 4, 2, 32, BF16)
        o, lse, second = nnv.differential_attention(q, k, v, w, for_backward=True)
        assert o.shape == (b, lq, 4, 64) and float(o.abs().sum()) == 0 and bool((lse == -math.inf).all())
        grads = nnv.differential_attention_backward(torch.ones_like(o), q, k, v, w, o, lse, second)
        assert [t.shape for t in grads] == [q.shape, k.shape, v.shape, w.shape] and all(float(t.abs().sum()) == 0 for t in grads)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_differential_attention_of_views(dtype):
    """Strides of a joint projection, heads before tokens, odd starts, one sequence's keys for all, masks and lengths with strides."""
    import nnv_amd as nnv
    g = gen(31)
    joint = rand(g, 3, 77, 8 * 64 + 4 * 64 + 2 * 128 + 5, dtype=dtype)
    w = rand(g, 8, shift=0.5)[::2]
    for odd in (0, 5):
        q = joint[..., odd:odd + 512].unflatten(2, (8, 64))
        k = joint[..., odd + 512:odd + 768].unflatten(2, (4, 64))
        v = joint[..., odd + 768:odd + 1024].unflatten(2, (2, 128))
        check_differ(q, k, v, w, causal=True, tag="joint %d" % odd)
        check_differ(q[:, ::7], k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1), w, tag="shared %d" % odd)
    q, k, v, _ = make_differ(g, 2, 50, 60, 4, 2, 32, dtype)
    mask = torch.rand(60, 2, 3, generator=g, device="cuda") < 0.7
    lengths = torch.tensor([[59, 0], [13, 0]], device="cuda")[:, 0]
    check_differ(q.transpose(1, 2).contiguous().transpose(1, 2), k.flip(3).transpose(2, 3).contiguous().transpose(2, 3), v, w, key_mask=mask[:, :, 1].t(),
                 key_lengths=lengths, tag="transposed")
    # lengths beyond 32 bits, and below zero
    beyond = torch.tensor([1 << 40, -(1 << 35)], device="cuda")
    for a, e in zip(nnv.differential_attention(q, k, v, w, key_lengths=beyond)[:2],
                    nnv.differential_attention(q, k, v, w, key_lengths=torch.tensor([60, 0], device="cuda"))[:2]):
        assert torch.equal(a, e)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_differential_attention_with_equal_maps_and_weight_zero(dtype):
    """A weight of zero is the first map alone, one of one on equal maps leaves nothing."""
    import nnv_amd as nnv
    g = gen(41)
    for lq in (1, 90):
        q, k, v, w = make_differ(g, 2, lq, 300, 4, 2, 64, dtype)
        one = nnv.differential_attention(q, k, v, torch.zeros_like(w))[0]
        e, bd = io.differ(q, k, v, torch.zeros_like(w)), io.differ_bounds(q, k, v, torch.zeros_like(w))
        po.assert_within(one, e[0], bd[0], "one map")
        q[:, :, 1::2], k[:, :, 1::2] = q[:, :, ::2], k[:, :, ::2]
        assert float(nnv.differential_attention(q, k, v, torch.ones_like(w))[0].abs().max()) == 0


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_differential_attention_of_far_scores(dtype):
    """Scores of some hundreds, weights that nothing is left of, a largest score late in the sequence."""
    g = gen(43)
    for lq, lk, d in ((1, 3000, 64), (140, 700, 128), (70, 300, 40)):
        q, k, v, w = make_differ(g, 1, lq, lk, 2, 1, d, dtype)
        k[:, lk - 3] = q[:, 0, :2] * 4
        check_differ(q * 8, k, v, w, tag="%d" % lq)
        check_differ(q, k, v, w, scale=1e-30, tag="flat %d" % lq)
        check_differ(q, k, v, w, scale=0.0, tag="zero %d" % lq)


def test_differential_attention_gradient_against_differences():
    import nnv_amd as nnv
    g = gen(51)
    q, k, v, w = make_differ(g, 2, 19, 37, 4, 2, 24, F32)
    kw = dict(causal=True, key_mask=torch.rand(2, 37, generator=g, device="cuda") < 0.8)
    o, lse, second = nnv.differential_attention(q, k, v, w, for_backward=True, **kw)
    do = rand(g, *o.shape)
    grads = nnv.differential_attention_backward(do, q, k, v, w, o, lse, second, **kw)
    bounds = io.differ_grad_bounds(do, q, k, v, w, **kw)
    h = 1e-5
    for i, t in enumerate((q, k, v, w)):
        d = torch.randn(t.shape, generator=g, device="cuda", dtype=torch.float64)
        loss = lambda s: float((io.differ(*[u.double() + (s * d if i == j else 0) for j, u in enumerate((q, k, v, w))], **kw)[0] * do.double()).sum())  # noqa: E731
        slope = (loss(h) - loss(-h)) / (2 * h)
        size = float((grads[i].double().abs() * d.abs()).sum())
        allowed = float(((bounds[i] + po.U32 * grads[i].double().abs()) * d.abs()).sum()) + 1e-5 * size + 1e-7
        assert abs(float((grads[i].double() * d).sum()) - slope) <= allowed


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("size", [(2, 1, 9000, 8, 2, 64), (2, 600, 700, 4, 2, 64), (1, 300, 500, 4, 2, 128), (1, 64, 5000, 2, 1, 96)], ids=lambda s: "x".join(map(str, s)))
def test_differential_attention_gives_the_same_bits_again_anywhere(size, dtype):
    """Twice, on another stream, and replayed from a graph among eager calls."""
    import nnv_amd as nnv
    g = gen(61)
    q, k, v, w = make_differ(g, *size, dtype)
    do = rand(g, size[0], size[1], size[3], 2 * size[5], dtype=dtype)
    lengths = torch.tensor([size[2] - 30] * size[0], device="cuda", dtype=torch.int32)

    def step():
        o, lse, second = nnv.differential_attention(q, k, v, w, key_lengths=lengths, causal=True, for_backward=True)
        return [o, lse, second, *nnv.differential_attention_backward(do, q, k, v, w, o, lse, second, key_lengths=lengths, causal=True)]

    eager = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = step()
    torch.cuda.current_stream().wait_stream(s)
    for a, b, e in zip(step(), other, eager):
        assert torch.equal(a, e) and torch.equal(b, e)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n in range(3):
        q.copy_(rand(gen(200 + n), *q.shape, dtype=dtype))
        lengths.fill_(size[2] - 100 * n)
        graph.replay()
        fresh = step()
        torch.cuda.synchronize()
        for a, e in zip(held, fresh):
            assert torch.equal(a, e)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_differential_attention_gradients_of_every_size(dtype):
    """Rows whose gradients are 2^-12 to 2^9 of the others', the largest ones last; weights of either sign beyond one."""
    import nnv_amd as nnv
    for d, lq, lk in ((64, 200, 333), (128, 70, 140), (40, 300, 90)):
        g = gen(71)
        q, k, v, w = make_differ(g, 2, lq, lk, 4, 2, d, dtype)
        w[0], w[1] = -3.0, 17.0
        kw = dict(causal=lk > lq)
        o, lse, second = nnv.differential_attention(q, k, v, w, for_backward=True, **kw)
        by = 2.0 ** (torch.arange(lq, device="cuda") * 21 // lq - 12)
        do = (rand(g, *o.shape) * by[None, :, None, None]).to(dtype)
        grads = nnv.differential_attention_backward(do, q, k, v, w, o, lse, second, **kw)
        for name, got, e, bd in zip(("dq", "dk", "dv", "dweights"), grads, io.differ_grad(do, q, k, v, w, **kw), io.differ_grad_bounds(do, q, k, v, w, **kw)):
            po.assert_within(got, e, bd, "%d %s" % (d, name))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_a_missing_value_shows_where_it_counts(dtype):
    """A query with a missing value: its row has none of o, lse and dq, the other rows keep theirs, and the gradients of the keys that it sees have none."""
    import nnv_amd as nnv
    for d, lq, lk in ((64, 90, 150), (40, 1, 70), (128, 40, 33)):
        g = gen(81)
        q, k, v, w = make_differ(g, 2, lq, lk, 4, 2, d, dtype)
        mask = torch.rand(2, lk, generator=g, device="cuda") < 0.8
        clean, row = q.clone(), lq // 2
        q[1, row] = math.nan
        o, lse, second = nnv.differential_attention(q, k, v, w, key_mask=mask, for_backward=True)
        exact, bounds = io.differ(clean, k, v, w, key_mask=mask), io.differ_bounds(clean, k, v, w, key_mask=mask)
        others = torch.ones(2, lq, dtype=torch.bool, device="cuda")
        others[1, row] = False
        for name, got, e, bd in zip(("o", "lse", "second"), (o, lse, second), exact, bounds):
            if name == "lse":
                got, e, bd = (x.transpose(1, 2) for x in (got, e, bd))
            assert got[1, row].isnan().all()
            po.assert_within(got[others], e[others], bd[others], name)
        do = rand(g, *o.shape, dtype=dtype)
        dq, dk, dv, dw = nnv.differential_attention_backward(do, q, k, v, w, o, lse, second, key_mask=mask)
        e, bd = io.differ_grad(do, clean, k, v, w, key_mask=mask)[0], io.differ_grad_bounds(do, clean, k, v, w, key_mask=mask)[0]
        assert dq[1, row].isnan().all() and dw.isnan().all()
        po.assert_within(dq[others], e[others], bd[others], "dq")
        for x in (dk, dv):
            assert x[1][mask[1]].isnan().all() and (x[1][~mask[1]] == 0).all() and x[0].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_differential_attention_of_many_sequences_by_length(dtype):
    """More sequences than a wave has lanes; keys that are the queries themselves."""
    g = gen(91)
    for lq in (1, 20):
        q, k, v, w = make_differ(g, 70, lq, 45, 2, 1, 32, dtype)
        lengths = torch.randint(0, 46, (70,), generator=g, device="cuda", dtype=torch.int32)
        check_differ(q, k, v, w, key_lengths=lengths, causal=True, tag="%d" % lq)
    q = rand(g, 3, 50, 4, 64, dtype=dtype)
    check_differ(q, q, rand(g, 3, 50, 2, 128, dtype=dtype), w, causal=True, tag="self")


def far(g, shape, strides, dtype):
    """A tensor of random values that lie far apart."""
    last = sum((n - 1) * s for n, s in zip(shape, strides)) + 1
    x = torch.empty(last, dtype=dtype, device="cuda").as_strided(shape, strides)
    return x.copy_(rand(g, *shape, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_offsets_past_32_bits(dtype):
    """Tokens, places and sequences more than 2^31 elements apart, and results longer than that."""
    import nnv_amd as nnv
    g, most = gen(95), 1 << 31
    for lq in (1, 70):
        for b, token in ((1, 1 << 22), (2, 1 << 9)):
            lk, batch = 600, most + (1 << 14)
            q, w = rand(g, b, lq, 8, 64, dtype=dtype), rand(g, 4, dtype=dtype)
            k = far(g, (b, lk, 2, 64), (batch, token, 64, 1), dtype)
            v = far(g, (b, lk, 1, 128), (batch, token, 128, 1), dtype)
            do = rand(g, b, lq, 4, 128, dtype=dtype)
            found = []
            for kk, vv in ((k, v), (k.contiguous(), v.contiguous())):
                o, lse, second = nnv.differential_attention(q, kk, vv, w, causal=True, for_backward=True)
                found.append([o, lse, second, *nnv.differential_attention_backward(do, q, kk, vv, w, o, lse, second, causal=True)])
            for a, e in zip(*found):
                assert torch.equal(a, e)
            del k, v, kk, vv
    q = far(g, (1, 550, 8, 64), (0, 1 << 22, 64, 1), dtype)
    k, v = rand(g, 1, 90, 2, 64, dtype=dtype), rand(g, 1, 90, 1, 128, dtype=dtype)
    found = []
    for qq in (q, q.contiguous()):
        o, lse, second = nnv.differential_attention(qq, k, v, w, for_backward=True)
        do = far(gen(96), o.shape, (0, 1 << 22, 128, 1), dtype)
        found.append([o, *nnv.differential_attention_backward(do, qq, k, v, w, o, lse, second)])
        del do
    for a, e in zip(*found):
        assert torch.equal(a, e)
    del q, qq
    # q, o and dq of more than 2^31 elements: the last sequences
    q = torch.zeros(4100, 128, 64, 64, dtype=dtype, device="cuda")
    q[-2:] = rand(g, 2, 128, 64, 64, dtype=dtype)
    k, v, w = rand(g, 4100, 3, 4, 64, dtype=dtype), rand(g, 4100, 3, 2, 128, dtype=dtype), rand(g, 32, dtype=dtype)
    o, lse, second = nnv.differential_attention(q, k, v, w, for_backward=True)
    dq, dk, dv, _ = nnv.differential_attention_backward(o, q, k, v, w, o, lse, second)
    one = nnv.differential_attention(q[-2:], k[-2:], v[-2:], w, for_backward=True)
    for a, e in zip((o, lse, second), one):
        assert torch.equal(a[-2:], e)
    for a, e in zip((dq, dk, dv), nnv.differential_attention_backward(one[0], q[-2:], k[-2:], v[-2:], w, *one)):
        assert torch.allclose(a[-2:].float(), e.float(), rtol=2e-2, atol=1e-5)
    del q, o, second, dq
    x = far(g, (1, 700, 64), (0, 1 << 22, 1), dtype)
    dy = rand(g, 1, 700, 64, dtype=dtype)
    y, mean, rstd = nnv.group_norm(x, 8)
    for a, e in zip((y, mean, rstd, *nnv.group_norm_backward(dy, x, mean, rstd)),
                    (lambda z: (*z, *nnv.group_norm_backward(dy, x.contiguous(), *z[1:])))(nnv.group_norm(x.contiguous(), 8))):
        assert torch.equal(a, e)
    x = far(g, (1, 700, 2, 64), (0, 1 << 22, 64, 1), dtype)
    at = torch.arange(700, device="cuda", dtype=torch.int32)[:, None]
    assert torch.equal(nnv.rotate_positions(x, at, [32]), nnv.rotate_positions(x.contiguous(), at, [32]))
    x = rand(g, 1, 20, 32, 128, dtype=dtype).repeat(1, 26300, 1, 1)   # 2^31 and 6 millions
    at = torch.arange(20, device="cuda", dtype=torch.int32)[:, None].repeat(26300, 1)
    y = nnv.rotate_positions(x, at, [64])
    assert torch.equal(y[:, -20:], y[:, :20]) and torch.equal(y[:, :20], nnv.rotate_positions(x[:, :20], at[:20], [64]))
    del y
    y, mean, rstd = nnv.group_norm(x.view(2, -1, 128), 4)
    assert torch.equal(y[0], y[1])
    dx, dscale, _ = nnv.group_norm_backward(x.view(2, -1, 128), x.view(2, -1, 128), mean, rstd)
    assert torch.equal(dx[0], dx[1]) and torch.equal(mean[0], mean[1])


def test_images_in_calls_at_once_and_graphs_of_one_pool():
    """Three streams with calls of their own at once, two graphs that share memory replayed in turn, gradients that are one number, the same tensor several times."""
    import nnv_amd as nnv
    g = gen(97)
    q, k, v, w = make_differ(g, 2, 200, 300, 4, 1, 64, BF16)
    do = torch.ones(1, 1, 1, 1, dtype=BF16, device="cuda").expand(2, 200, 4, 128)
    x, scale = rand(g, 2, 40, 50, 64, dtype=BF16), rand(g, 64, dtype=BF16)

    def step():
        o, lse, second = nnv.differential_attention(q, k, v, w, causal=True, for_backward=True)
        y, mean, rstd = nnv.group_norm(x, 8, scale, activation="silu")
        return [o, lse, second, *nnv.differential_attention_backward(do, q, k, v, w, o, lse, second, causal=True), y, *nnv.group_norm_backward(y, x, mean, rstd, scale, None, "silu")]

    eager = step()
    whole = nnv.differential_attention_backward(do.contiguous(), q, k, v, w, *eager[:3], causal=True)
    assert all(torch.equal(a, e) for a, e in zip(eager[3:7], whole))
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    found = [None] * 3
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                found[i] = step()
    torch.cuda.synchronize()
    for f in found:
        assert all(torch.equal(a, e) for a, e in zip(f, eager))
    graphs, held = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph, pool=graphs[0].pool() if i else None):
            held.append(step())
    for n in range(3):
        q.copy_(rand(gen(300 + n), *q.shape, dtype=BF16))
        for i in (1, 0, 1):
            graphs[i].replay()
            fresh = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, e) for a, e in zip(held[i], fresh))
    at = torch.arange(200, device="cuda")[:, None].expand(200, 2)
    turned = nnv.rotate_positions([q] * 6, at, np.array([16, 16]))
    assert all(torch.equal(t, nnv.rotate_positions(q, at.contiguous(), (16, 16))) for t in turned)
    assert torch.equal(nnv.group_norm(x, np.int64(8))[0], nnv.group_norm(x, 8)[0])
