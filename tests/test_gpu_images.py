"""The operators on points that are images or videos (nnv_amd.images) on the GPU against plain 64-bit forms, at the sizes, strides and
values where they can go wrong."""
import math

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
