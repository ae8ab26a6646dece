"""What the operators on points that are images or videos owe to the last bit of their results' type: nothing but the result is rounded to 16 bits where a
second piece can hold what a first one leaves, in whatever order the keys lie; infinities that count stay infinite; masks and tiles that go on for long."""
import math

import pytest
import torch

from tests import images_oracle as io
from tests import points_oracle as po

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES, IDS = [F32, BF16, F16], ["f32", "bf16", "f16"]


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=F32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)


def make_differ(g, b, lq, lk, h, hkv, d, dtype):
    return (rand(g, b, lq, 2 * h, d, dtype=dtype), rand(g, b, lk, 2 * hkv, d, dtype=dtype), rand(g, b, lk, hkv, 2 * d, dtype=dtype),
            rand(g, h, scale=0.1, shift=0.6))


def check_differ(q, k, v, w, clean=None, tag="", **kw):
    """Forward and backward against the 64-bit forms (of `clean` keys and values, where those that do not count hold something else)."""
    import nnv_amd as nnv
    ck, cv = clean or (k, v)
    o, lse, second = nnv.differential_attention(q, k, v, w, for_backward=True, **kw)
    for name, got, e, bd in zip(("o", "lse", "second"), (o, lse, second), io.differ(q, ck, cv, w, **kw), io.differ_bounds(q, ck, cv, w, **kw)):
        po.assert_within(got, e, bd, tag + " " + name)
    do = rand(gen(q.shape[1]), *o.shape, dtype=q.dtype)
    grads = nnv.differential_attention_backward(do, q, k, v, w, o, lse, second, **kw)
    for name, got, e, bd in zip(("dq", "dk", "dv", "dweights"), grads, io.differ_grad(do, q, ck, cv, w, **kw), io.differ_grad_bounds(do, q, ck, cv, w, **kw)):
        po.assert_within(got, e, bd, tag + " " + name)


def off(got, exact):
    """How far a tensor is from what it should be, relative to that, as root mean squares."""
    return float((got.double() - exact).norm() / exact.norm())


def assert_rounded_once(got, exact, name):
    """No further off than a rounding at the end: two pieces hold 2^-16 (bf16) or 2^-22 (f16) of a number, sums and exponents in f32 some 1e-6, whose squares are nothing
    beside that of a rounding (0.0017, 0.00021); 2 % are left for them."""
    own = off(exact.to(got.dtype), exact)
    assert off(got, exact) <= 1.02 * own, "%s: %.3g off, its rounding is %.3g" % (name, off(got, exact), own)


def lopsided(g, b, lq, lk, h, hkv, d, dtype, heavy):
    """Keys that nearly all weight is on, or nearly none, by their place among 32 that follow one another."""
    q, k, v, w = make_differ(g, b, lq, lk, h, hkv, d, dtype)
    place = torch.arange(lk, device="cuda") % 32 // 16
    q[..., 0], k[..., 0] = d ** 0.5, ((place == heavy).float() * 6 - 3)[None, :, None].to(dtype)
    return q, k, v, w


# queries, keys, head: single tokens, rows that fill a tile of few, many rows; heads of every template in 16 bits
SIZES = [(1, 3000, 64), (3, 500, 128), (90, 1000, 64), (70, 600, 128), (150, 400, 40), (100, 300, 80), (65, 333, 96), (40, 257, 24)]


@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_results_are_rounded_once_in_whatever_order_the_keys_lie(size, dtype):
    import nnv_amd as nnv
    lq, lk, d = size
    for heavy in (0, 1, 2):      # 2: no such keys
        for weight in (0.6, 1.0, -2.5):
            g = gen(lq + lk + heavy)
            q, k, v, w = lopsided(g, 2, lq, lk, 4, 2, d, dtype, heavy)
            w = w - 0.6 + weight
            o, _, second = nnv.differential_attention(q, k, v, w, for_backward=True)
            exact = io.differ(q, k, v, w)
            assert_rounded_once(second, exact[2], "second, %d" % heavy)
            assert_rounded_once(o, exact[0], "o, %d, %g" % (heavy, weight))


def exact_gradients(do, q, k, v, w, o, second, **kw):
    """(dq, dk, dv, dweights) in f64, of more than 256 keys dq with D from the o and second of the call, as the operator has it; and what dweights may be off by: sums in f32."""
    scale, group = q.shape[3] ** -0.5, q.shape[2] // k.shape[2]
    _, dk, dv, dw = io.differ_grad(do, q, k, v, w, **kw)
    c = io.seen(q, k, kw.get("key_lengths"), kw.get("key_mask"), kw.get("causal", False))
    maps, vh = io._split_maps(q, k, v, c)
    g = torch.where(c.any(2)[:, None, :, None], do.double().permute(0, 2, 1, 3), 0.0).contiguous()
    dp, share = io._matmul(g, vh), w.double()[None, :, None, None]
    rows = lambda x: (g * x.double().permute(0, 2, 1, 3)).sum(-1, keepdim=True)  # noqa: E731
    deltas = [rows(o) + share * rows(second), rows(second)] if k.shape[1] > 256 else [(io._softmax(*m, c, scale)[0] * dp).sum(-1, keepdim=True) for m in maps]
    dq = [torch.matmul((-share if m else 1.0) * io._softmax(qm, km, c, scale)[0] * (dp - deltas[m]) * scale, km) for m, (qm, km) in enumerate(maps)]
    size = (io._softmax(*maps[1], c, scale)[0] * io._matmul(g.abs(), vh.abs())).sum((0, 2, 3))
    return io._by_map(*dq), dk, dv, dw, (k.shape[1] + 2 * q.shape[3] + 100) * po.U32 * size


def gradients(dtype, size, heavy, **kw):
    import nnv_amd as nnv
    lq, lk, d = size
    g = gen(lq + lk + heavy)
    q, k, v, w = lopsided(g, 2, lq, lk, 4, 2, d, dtype, heavy)
    q[:, :, 1::2, 1], k[:, :, 1::2, 1] = q[:, :, 1::2, 0], -k[:, :, 1::2, 0]      # (the second map's heavy keys are the others)
    q[:, :, 1::2, 0] = 0
    o, lse, second = nnv.differential_attention(q, k, v, w, for_backward=True, **kw)
    do = rand(g, *o.shape, dtype=dtype)
    return nnv.differential_attention_backward(do, q, k, v, w, o, lse, second, **kw), exact_gradients(do, q, k, v, w, o, second, **kw)


GRAD_SIZES = [(90, 1000, 64), (300, 333, 64), (70, 600, 128), (150, 400, 40), (100, 300, 80), (65, 333, 96), (40, 257, 24), (8, 500, 96)]


@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("size", GRAD_SIZES, ids=lambda s: "x".join(map(str, s)))
def test_gradients_of_queries_and_keys_are_rounded_once(size, dtype):
    for heavy in (0, 1, 2):
        for causal in (False, True):
            got, exact = gradients(dtype, size, heavy, causal=causal)
            for i, name in enumerate(("dq", "dk")):
                assert_rounded_once(got[i], exact[i], "%s %d %s" % (name, heavy, causal))
            assert ((got[3].double() - exact[3]).abs() <= exact[4]).all()


@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("size", GRAD_SIZES + [(700, 5, 64)], ids=lambda s: "x".join(map(str, s)))
def test_gradients_of_values_are_rounded_once(size, dtype):
    for heavy in (0, 1, 2):
        for causal in (False, True):
            got, exact = gradients(dtype, size, heavy, causal=causal)
            assert_rounded_once(got[2], exact[2], "dv %d %s" % (heavy, causal))


@pytest.mark.parametrize("size", [(90, 200, 64), (70, 150, 128), (60, 333, 40)], ids=lambda s: "x".join(map(str, s)))
def test_f16_keeps_the_bits_of_small_gradients_beside_large_ones(size):
    """The second map's keys in f16, whose gradients are 2^-24 of the first one's: each map's are lifted for themselves.  (As test_gradients_..._rounded_once: no further off
    than their own rounding.)"""
    import nnv_amd as nnv
    lq, lk, d = size
    g = gen(5)
    q, k, v, w = make_differ(g, 2, lq, lk, 4, 2, d, F16)
    w = w * 2.0 ** -24
    o, lse, second = nnv.differential_attention(q, k, v, w, for_backward=True)
    do = (rand(g, *o.shape) * 8192).to(F16)
    got = nnv.differential_attention_backward(do, q, k, v, w, o, lse, second)
    exact = exact_gradients(do, q, k, v, w, o, second)
    for i, name in enumerate(("dq", "dk")):
        for m in (0, 1):
            assert bool(exact[i][:, :, m::2].abs().max() < 2.0 ** 15)
            assert_rounded_once(got[i][:, :, m::2], exact[i][:, :, m::2], "%s of map %d" % (name, m))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_an_infinite_value_that_counts_stays_infinite(dtype):
    """Of a weight in two pieces neither makes an infinite value a NaN: second is infinite there, and so is o where the weight's sign adds the maps up."""
    import nnv_amd as nnv
    for lq, lk, d in ((1, 300, 64), (1, 70, 128), (16, 200, 40), (90, 200, 64), (70, 150, 128), (40, 333, 48)):
        for flat in (False, True):      # flat: every weight is a power of two, and its second piece would be zero
            g = gen(lq + d)
            q, k, v, w = make_differ(g, 2, lq, lk, 4, 2, d, dtype)
            q = (q * (0.0 if flat else 0.3)).to(dtype)
            w = -w
            for at, value in ((3, math.inf), (20, -math.inf), (lk - 1, math.inf)):
                v[1, at, 0, at % (2 * d)] = value
            o, _, second = nnv.differential_attention(q, k, v, w, for_backward=True)
            exact, bounds = io.differ(q, k, v, w), io.differ_bounds(q, k, v, w)
            assert bool(exact[2].isinf().any()) and not bool(exact[2].isnan().any())
            for name, got, e, bd in (("o", o, exact[0], bounds[0]), ("second", second, exact[2], bounds[2])):
                po.assert_within(got, e, bd, "%d %d %s %s" % (lq, d, flat, name))
            # and an infinite gradient of the result is infinite in dv of every key
            v = rand(g, *v.shape, dtype=dtype)
            o, lse, second = nnv.differential_attention(q, k, v, w, for_backward=True)
            do = rand(g, *o.shape, dtype=dtype)
            do[1, lq // 2, 1, 5], do[1, 0, 3, 7] = math.inf, -math.inf
            got, exact = (f(do, q, k, v, w, *s)[2] for f, s in ((nnv.differential_attention_backward, (o, lse, second)), (io.differ_grad, ())))
            assert bool((exact[1, :, 0, 5] == math.inf).all()) and bool((exact[1, :, 1, 7] == -math.inf).all())
            po.assert_within(got, exact, io.differ_grad_bounds(do, q, k, v, w)[2], "%d %d %s dv" % (lq, d, flat))


# heads that are no multiple of 8, which the kernels with products in f32 take
@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("size", [(90, 400, 60), (70, 200, 33), (9, 900, 126), (300, 40, 50)], ids=lambda s: "x".join(map(str, s)))
def test_gradients_of_odd_heads_are_rounded_once(size, dtype):
    for heavy in (0, 2):
        for causal in (False, True):
            got, exact = gradients(dtype, size, heavy, causal=causal)
            for i, name in enumerate(("dq", "dk", "dv")):
                assert_rounded_once(got[i], exact[i], "%s %d %s" % (name, heavy, causal))
            assert ((got[3].double() - exact[3]).abs() <= exact[4]).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_a_row_that_sees_one_key_has_no_gradient_for_it(dtype):
    """Its weight is one whatever the score: what dk is beside zero comes of sums in f32, not of the o and second that were rounded to 16 bits."""
    import nnv_amd as nnv
    for lq, lk, d in ((40, 50, 64), (70, 90, 128), (100, 30, 40), (40, 50, 60), (33, 70, 7), (1, 20, 64)):
        g = gen(d)
        q, k, v, w = make_differ(g, 2, lq, lk, 4, 2, d, dtype)
        lengths = torch.ones(2, dtype=torch.int32, device="cuda")
        o, lse, second = nnv.differential_attention(q, k, v, w, key_lengths=lengths, for_backward=True)
        do = rand(g, *o.shape, dtype=dtype)
        dk = nnv.differential_attention_backward(do, q, k, v, w, o, lse, second, key_lengths=lengths)[1]
        assert (dk[:, 1:] == 0).all()
        # a weight is off by what its score (twice: in lse as well) and its exponent are, D by the sums of do v; both times do v
        size = q.shape[3] ** -0.5
        heads = lambda x, n: x.double().abs().repeat_interleave(n, 2)  # noqa: E731   (key/value heads to heads)
        k0, v0, qa = heads(k[:, 0].view(2, 1, 2, 2 * d), 2).view(2, 1, 8, d), heads(v[:, :1], 2), q.double().abs()
        score = (qa * k0).sum(-1) * size
        dp = (do.double().abs() * v0).sum(-1).repeat_interleave(2, 2)
        off = (2 * (d + 16) * score + 8 * score + 4 * d + 64) * po.U32
        by = torch.stack([torch.ones(4, device="cuda"), w.abs() + 0], 1).flatten().double() + w.abs().double().max()   # (the first map's D is formed from o and second)
        bound = ((size * by * off * dp)[..., None] * qa).sum(1).view(2, 2, 2, 2, d).sum(2).reshape(2, 4, d)
        assert (dk[:, 0].double().abs() <= bound + po.TINY[dtype]).all(), (lq, lk, d)


@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("size", [(64, 16, 64), (200, 30, 40), (1, 130, 128), (300, 256, 64), (250, 256, 96), (300, 250, 60), (40, 3, 33), (150, 200, 128)],
                         ids=lambda s: "x".join(map(str, s)))
def test_gradients_of_queries_with_few_keys_are_rounded_once(size, dtype):
    """D is that of the weights, not of the o and second that were rounded to 16 bits."""
    import nnv_amd as nnv
    lq, lk, d = size
    for causal in (False, True):
        g = gen(sum(size))
        q, k, v, w = lopsided(g, 2, lq, lk, 4, 2, d, dtype, 2)
        lengths = torch.tensor([lk, lk // 2 + 1], dtype=torch.int32, device="cuda")
        mask = torch.rand(2, lk, generator=g, device="cuda") < 0.9
        for kw in ({}, {"key_lengths": lengths}, {"key_mask": mask}):
            o, lse, second = nnv.differential_attention(q, k, v, w, for_backward=True, causal=causal, **kw)
            do = rand(g, *o.shape, dtype=dtype)
            exact = io.differ_grad(do, q, k, v, w, causal=causal, **kw)
            for name, got, e in zip(("dq", "dk", "dv"), nnv.differential_attention_backward(do, q, k, v, w, o, lse, second, causal=causal, **kw), exact):
                assert_rounded_once(got, e, "%s %s" % (name, causal))


@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS[1:])
def test_early_rows_of_a_causal_call_are_rounded_once(dtype):
    """Those whose block sees 256 keys: blocks of 256 rows for heads of 64, of 128 above."""
    import nnv_amd as nnv
    for n, d, first in ((700, 64, 256), (600, 128, 256)):
        g = gen(n)
        q, k, v, w = make_differ(g, 2, n, n, 2, 2, d, dtype)
        o, lse, second = nnv.differential_attention(q, k, v, w, for_backward=True, causal=True)
        do = rand(g, *o.shape, dtype=dtype)
        dq = nnv.differential_attention_backward(do, q, k, v, w, o, lse, second, causal=True)[0]
        exact = io.differ_grad(do, q, k, v, w, causal=True)[0]
        assert_rounded_once(dq[:, :first], exact[:, :first], "%d" % d)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_backward_of_no_queries_through_c_reads_no_weights(dtype):
    """The C call takes NULL for what it has no rows of: the keys' gradients are zero."""
    from nnv_amd import _lib, images
    from nnv_amd._lib import context_on
    ctx = context_on(0)
    t = TYPES.index(dtype)
    k, v = torch.ones(2, 40, 4, 64, dtype=dtype, device="cuda"), torch.ones(2, 40, 2, 128, dtype=dtype, device="cuda")
    dk, dv, dw = torch.full_like(k, 7), torch.full_like(v, 7), torch.full((4,), 7.0, dtype=dtype, device="cuda")
    d = images._DIFFER.pack(t, t, 2, 0, 40, 4, 2, 64, 0, 0.125, 0, k.data_ptr(), v.data_ptr(), 0, 8 * 64, 64, *k.stride()[:3], *v.stride()[:3], 0, 0, 0, 0, 0, 0, 0, 0, 0,
                            0, 4 * 128, 128, 0, dk.data_ptr(), dv.data_ptr(), dw.data_ptr())
    need = images._differ_workspace(ctx.lib, True, False, t, t, 2, 0, 40, 4, 2, 64)
    work = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
    _lib.check(ctx.lib.nnvhip_differential_attention_backward(ctx.handle, d, work.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert (dk == 0).all() and (dv == 0).all() and (dw == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("places", [1, 40, 300, 70001], ids=str)
def test_group_norm_of_a_mean_far_from_zero(places, dtype):
    """Groups of equal values have no spread whatever the values are, and of a small spread the variance keeps its bits: sums in f64 of differences from a value of the group, which lose
    less than 2^-53 n of a variance of n values."""
    import nnv_amd as nnv
    for channels, groups in ((16, 4), (40, 8), (6, 3), (1030, 2)):
        if places * channels > 1 << 22:
            continue
        b = torch.arange(float(channels), device="cuda") - 8
        for value in (1000.1, 10000.3, -60000.7, 7.1e-3):
            x = torch.full((2, places, channels), value, device="cuda").to(dtype)
            y, mean, rstd = nnv.group_norm(x, groups, None, b, 1e-5)
            assert (mean == x[0, 0, 0].float()).all() and torch.equal(y.float(), b.to(dtype).float().expand(2, places, channels))
            assert ((rstd.double() * 1e-5 ** 0.5 - 1).abs() <= 2 * po.U32).all()      # (its own rounding, and that of epsilon)
        # f32 values next to one another around a far mean; one that lies far from the others, in front and behind
        if dtype == F32 and places > 1:
            g = gen(places)
            far = torch.tensor([1000.0, -30000.0], device="cuda")[:, None, None] + torch.randint(0, 9, (2, places, channels), generator=g, device="cuda") / 512
            out = far.clone()
            out[0, 0, 0], out[1, -1, -1] = 3e7, -1e30
            for x in (far, out):
                _, mean, rstd = nnv.group_norm(x, groups, None, None, 1e-5)
                _, e_mean, e_rstd = io.group(x, groups, None, None, 1e-5, None)
                n = places * channels // groups
                assert ((mean.double() - e_mean).abs() <= 1.01 * po.U32 * e_mean.abs()).all()
                assert ((rstd.double() / e_rstd - 1).abs() <= (1.5 + n * 2.0 ** -27) * po.U32 * 1.0).all()


def test_group_norm_whose_first_value_is_infinite():
    """Its mean is infinite, as that of any group with such a value, and the other groups know nothing of it."""
    import nnv_amd as nnv
    for places in (40, 5000):
        x = rand(gen(places), 2, places, 16, shift=100.0)
        clean = x.clone()
        x[0, 0, 4], x[1, 0, 8] = math.inf, math.nan
        y, mean, _ = nnv.group_norm(x, 4)
        e, e_mean, _ = nnv.group_norm(clean, 4)
        assert mean[0, 1] == math.inf and mean[1, 2].isnan() and y[0, :, 4:8].isnan().all() and y[1, :, 8:12].isnan().all()
        for n, hit in ((0, 1), (1, 2)):
            others = [j for j in range(4) if j != hit]
            assert torch.equal(mean[n, others], e_mean[n, others]) and all(torch.equal(y[n, :, 4 * j:4 * j + 4], e[n, :, 4 * j:4 * j + 4]) for j in others)


def test_group_norm_takes_epsilon_in_64_bits():
    """Of equal values rstd is 1 / sqrt(epsilon), also of one that f32 does not hold."""
    import nnv_amd as nnv
    for places in (40, 70001):
        for epsilon in (1e-5, 1.0 / 3, 1e-42, 1e-60):
            rstd = nnv.group_norm(torch.full((1, places, 8), 3.5, device="cuda"), 2, epsilon=epsilon)[2]
            assert ((rstd.double() * math.sqrt(epsilon) - 1).abs() <= 1.01 * po.U32).all()


def test_rotary_positions_keep_the_bits_of_the_angle():
    """Next to multiples of a quarter turn a sine or cosine is as small as what is left of the angle there, and has its bits: a few units in the last place, and of the angle 2^-53 of the whole one."""
    import nnv_amd as nnv
    at = torch.tensor([3, 11, 14, 22, 33, 44, 355, 710, 1065, 52174, 208341, 312689, 0, 1, 2, 100], device="cuda")
    for interleaved in (False, True):
        for inverse in (False, True):
            x = torch.zeros(1, len(at), 1, 2, device="cuda")
            x[..., 0] = 1.0
            y = nnv.rotate_positions(x, at[:, None], [1], interleaved=interleaved, inverse=inverse)[0, :, 0].double()
            angle = at.double() * (-1 if inverse else 1)
            exact = torch.stack([torch.cos(angle), torch.sin(angle)], 1)
            assert ((y - exact).abs() <= 8 * po.U32 * exact.abs() + (8 * at.double() * 2.0 ** -53)[:, None]).all()


def test_rotary_positions_in_f32_are_as_far_off_as_rounded_cosines():
    """No further than products and sums in f32 with cosines and sines that were rounded once, but for a tenth."""
    import nnv_amd as nnv
    g = gen(3)
    x = rand(g, 2, 3000, 4, 64)
    at = torch.randint(0, 5000, (3000, 2), generator=g, device="cuda")
    y, exact = nnv.rotate_positions(x, at, [16, 16]), io.rotate(x, at, [16, 16])
    angle = torch.cat([at[:, a, None].double() * 10000.0 ** -(torch.arange(16, device="cuda", dtype=torch.float64) / 16) for a in (0, 1)], 1)[None, :, None]
    c, s, u, w = torch.cos(angle).float(), torch.sin(angle).float(), x[..., :32], x[..., 32:]
    plain = torch.cat([u * c - w * s, u * s + w * c], -1)
    assert off(y, exact) <= 1.1 * off(plain, exact)


# Causal calls whose blocks take two tiles of keys, an early and a late one (six tiles or more: of 256 keys in 16 bits, 128 for heads above 64, of 64 in f32), an even and an odd number of them
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("size", [(800, 1400, 64, 6), (800, 1600, 40, 7), (400, 700, 128, 6), (450, 850, 96, 7), (250, 420, 64, 0), (200, 380, 33, 0)], ids=lambda s: "x".join(map(str, s[:3])))
def test_gradients_of_keys_in_paired_tiles(size, dtype):
    lq, lk, d, tiles = size
    assert dtype == F32 or tiles == 0 or -(-lk // (256 if d <= 64 else 128)) == tiles
    assert dtype != F32 or tiles or -(-lk // 64) in (6, 7)
    g = gen(lk)
    q, k, v, w = make_differ(g, 2, lq, lk, 2, 1, d, dtype)
    check_differ(q, k, v, w, causal=True, tag="all")
    lengths = torch.tensor([lk - 70, lq // 2 + 3], dtype=torch.int32, device="cuda")      # (the second one shorter than the queries: its first rows see no key)
    mask = torch.rand(2, lk, generator=g, device="cuda") < 0.9
    clean = (k.clone(), v.clone())
    for i, n in enumerate(lengths.tolist()):
        k[i, n:], v[i, n:] = math.nan, math.inf
    check_differ(q, k, v, w, clean, causal=True, key_lengths=lengths, tag="lengths")
    check_differ(q, k, v, w, clean, causal=True, key_lengths=lengths, key_mask=mask, tag="lengths, mask")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("size", [(16, 40, 4500, 16, 16, 64), (64, 1, 20000, 8, 4, 32), (32, 2, 9000, 8, 8, 128)], ids=lambda s: "x".join(map(str, s)))
def test_masks_of_many_tiles(size, dtype):
    """More tiles in a row than a mask is read for at a time (32, of 64 keys, or of 32 that eight or two groups of waves take in turn), with no period, and what is left out far behind holds anything."""
    import nnv_amd as nnv
    from nnv_amd import _lib, images
    b, lq, lk, h, hkv, d = size
    lib = _lib.load()
    t = TYPES.index(dtype)
    need = images._differ_workspace(lib, False, False, t, 0, *size)
    splits = max(1, need // (b * h * 2 * lq * (2 * d + 1) * 4))
    assert lk // (64 if lq > 16 else 32 * {32: 8, 128: 2}[d]) // splits > 32
    g = gen(lk)
    q, k, v, w = make_differ(g, *size, dtype)
    mask = torch.rand(b, lk, generator=g, device="cuda") < 0.7
    mask[:, lk // 2:] &= torch.rand(b, lk - lk // 2, generator=g, device="cuda") < 0.5
    clean = (k.clone(), v.clone())
    k[~mask], v[~mask] = math.nan, math.inf
    for causal in (False, True):
        o, lse, second = nnv.differential_attention(q, k, v, w, key_mask=mask, causal=causal, for_backward=True)
        kw = {"key_mask": mask, "causal": causal}
        for i in range(0, b, 8):      # (some sequences at a time: the 64-bit forms are large)
            part = [x[i:i + 8] for x in (q, *clean)] + [w]
            at = {"key_mask": mask[i:i + 8], "causal": causal}
            for name, got, e, bd in zip(("o", "lse", "second"), (o, lse, second), io.differ(*part, **at), io.differ_bounds(*part, **at)):
                po.assert_within(got[i:i + 8], e, bd, "%s %s" % (name, causal))
        if lq > 16:
            do = rand(g, *o.shape, dtype=dtype)
            grads = nnv.differential_attention_backward(do, q, k, v, w, o, lse, second, **kw)
            exact, bounds = (f(do[:2], q[:2], clean[0][:2], clean[1][:2], w, key_mask=mask[:2], causal=causal) for f in (io.differ_grad, io.differ_grad_bounds))
            for name, got, e, bd in zip(("dq", "dk", "dv"), grads, exact, bounds):
                po.assert_within(got[:2], e, bd, "%s %s" % (name, causal))
