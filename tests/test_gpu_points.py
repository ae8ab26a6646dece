"""The operators on points and gradients (nnv_amd.points) on the GPU against plain 64-bit forms, at the sizes, masks, strides
and values where they can go wrong."""
import math

import pytest
import torch

from tests import points_oracle as po

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
IDS = ["f32", "bf16", "f16"]


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=F32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)


# ---- layer normalization ------------------------------------------------------------------------------

# every number of lanes a row is given to, sizes next to its steps, and rows longer than a block's registers hold
SIZES = [1, 3, 7, 8, 31, 64, 65, 128, 255, 256, 257, 511, 513, 768, 1000, 1024, 1025, 2048, 2049, 4095, 4096, 4097, 8191, 8192, 8193, 20001]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("size", SIZES)
def test_norm_forward_and_backward(size, dtype):
    import nnv_amd as nnv
    for rows in (1, 2, 5, 67):
        g = gen(size * 100 + rows)
        x = rand(g, rows, size, dtype=dtype, scale=1.5, shift=3.0)
        for pt in {dtype, F32}:
            w, b, dy = rand(g, size, dtype=pt, shift=1.0), rand(g, size, dtype=pt), rand(g, rows, size, dtype=dtype)
            y, mean, rstd = nnv.layer_norm(x, w, b, 1e-5)
            ey, em, er = po.norm(x, w, b, 1e-5)
            by, bm, br = po.norm_bounds(x, w, b, 1e-5, po.ROW_ADDS + size // 512)
            tag = "%d x %d" % (rows, size)
            po.assert_within(mean, em, bm, tag + " mean")
            po.assert_within(rstd, er, br, tag + " rstd")
            po.assert_within(y, ey, by, tag + " y")
            dx, dw, db = nnv.layer_norm_backward(dy, x, mean, rstd, w)
            assert dx.dtype == dtype and dw.dtype == pt and db.dtype == pt and y.dtype == dtype
            exact, bound = po.norm_grad(dy, x, mean, rstd, w), po.norm_grad_bounds(dy, x, mean, rstd, w, po.ROW_ADDS + size // 512)
            for name, got, e, bd in zip(("dx", "dscale", "doffset"), (dx, dw, db), exact, bound):
                po.assert_within(got, e, bd, tag + " " + name)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows,size", [(3000, 64), (1003, 384), (4099, 1024), (700, 4096), (300, 8192), (70, 9000)])
def test_norm_gradient_over_many_rows(rows, size, dtype):
    """Several blocks, several turns each, partial sums in memory; twice the same bits."""
    import nnv_amd as nnv
    g = gen(rows)
    x, dy, w = rand(g, rows, size, dtype=dtype), rand(g, rows, size, dtype=dtype), rand(g, size, dtype=F32)
    _, mean, rstd = nnv.layer_norm(x, w, None)
    one, two = (nnv.layer_norm_backward(dy, x, mean, rstd, w) for _ in range(2))
    exact, bound = po.norm_grad(dy, x, mean, rstd, w), po.norm_grad_bounds(dy, x, mean, rstd, w, po.ROW_ADDS + size // 512)
    for name, a, b, e, bd in zip(("dx", "dscale", "doffset"), one, two, exact, bound):
        assert torch.equal(a, b), name
        po.assert_within(a, e, bd, "%d x %d %s" % (rows, size, name))


def test_norm_without_parameters_and_in_any_shape():
    import nnv_amd as nnv
    g = gen(4)
    x = rand(g, 3, 5, 2, 40, dtype=BF16)
    y, mean, rstd = nnv.layer_norm(x)
    assert y.shape == x.shape and mean.shape == rstd.shape == (3, 5, 2)
    po.assert_within(y, po.norm(x, None, None, 1e-5)[0], po.norm_bounds(x, None, None, 1e-5)[0], "y")
    dy = rand(g, 3, 5, 2, 40, dtype=BF16)
    for name, got, e, b in zip(("dx", "dscale", "doffset"), nnv.layer_norm_backward(dy, x, mean, rstd), po.norm_grad(dy, x, mean, rstd, None),
                               po.norm_grad_bounds(dy, x, mean, rstd, None)):
        po.assert_within(got, e, b, name)
    # no rows at all, and rows of a wider tensor, of a transposed one, and starting at an odd element
    y, mean, _ = nnv.layer_norm(x[:0])
    assert y.shape == (0, 5, 2, 40) and mean.shape == (0, 5, 2)
    assert all(t.abs().sum() == 0 for t in nnv.layer_norm_backward(x[:0], x[:0], mean, mean)[1:])
    wide = rand(g, 37, 100, dtype=BF16)
    for view in (wide[:, 13:76], wide.t(), wide.view(-1)[1:-99].view(36, 100), wide[::3, :64], wide[:, 5:6]):
        po.assert_within(nnv.layer_norm(view)[0], po.norm(view, None, None, 1e-5)[0], po.norm_bounds(view, None, None, 1e-5)[0], "view")


def test_norm_of_constant_infinite_and_missing_values():
    import nnv_amd as nnv
    x = torch.full((4, 300), 7.25, device="cuda")
    x[1, 5] = math.inf
    x[2, 299] = math.nan
    b = torch.arange(300.0, device="cuda")
    y, mean, rstd = nnv.layer_norm(x, None, b, 1e-5)
    assert torch.equal(y[0], b) and torch.equal(y[3], b) and mean[0] == 7.25    # no spread: the offset alone, exactly
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all()                   # and a row without a mean reaches no other
    # large values next to a small spread: the variance is taken around the mean
    x = 1e4 + torch.arange(512.0, device="cuda")[None] / 64
    po.assert_within(nnv.layer_norm(x)[0], po.norm(x, None, None, 1e-5)[0], po.norm_bounds(x, None, None, 1e-5)[0], "offset rows")


def test_norm_gradient_against_differences():
    import nnv_amd as nnv
    g = gen(11)
    x, w, b, dy = rand(g, 6, 96), rand(g, 96), rand(g, 96), rand(g, 6, 96)
    _, mean, rstd = nnv.layer_norm(x, w, b)
    grads = nnv.layer_norm_backward(dy, x, mean, rstd, w)
    bounds = po.norm_grad_bounds(dy, x, mean, rstd, w)
    h = 1e-5
    for k, t in enumerate((x, w, b)):
        d = torch.randn(t.shape, generator=g, device="cuda", dtype=torch.float64)
        loss = lambda s: float((po.norm(*[u.double() + (s * d if i == k else 0) for i, u in enumerate((x, w, b))], 1e-5)[0] * dy.double()).sum())  # noqa: E731
        slope = (loss(h) - loss(-h)) / (2 * h)
        size = float((grads[k].double().abs() * d.abs()).sum())
        # the kernel's rounding, that of the statistics it was handed, and the differences' own h^2 and 1e-16 / h
        allowed = float(((bounds[k] + po.U32 * grads[k].double().abs()) * d.abs()).sum()) + 1e-5 * size + 1e-7
        assert abs(float((grads[k].double() * d).sum()) - slope) <= allowed


# ---- attention -------------------------------------------------------------------------------------------


def make(g, b, lq, lk, h, hkv, d, dtype):
    return rand(g, b, lq, h, d, dtype=dtype), rand(g, b, lk, hkv, d, dtype=dtype), rand(g, b, lk, hkv, d, dtype=dtype)


def check_attend(q, k, v, key_lengths=None, key_mask=None, scale=None, backward=True, tag=""):
    import nnv_amd as nnv
    kw = dict(key_lengths=key_lengths, key_mask=key_mask, scale=scale)
    o, lse = nnv.cross_attention(q, k, v, **kw)
    (eo, el), (bo, bl) = po.attend(q, k, v, **kw), po.attend_bounds(q, k, v, **kw)
    po.assert_within(lse, el, bl, tag + " lse")
    po.assert_within(o, eo, bo, tag + " o")
    if not backward:
        return o, lse
    do = rand(gen(q.shape[1]), *q.shape, dtype=q.dtype)
    grads = nnv.cross_attention_backward(do, q, k, v, o, lse, **kw)
    for name, t, got, e, bd in zip(("dq", "dk", "dv"), (q, k, v), grads, po.attend_grad(do, q, k, v, **kw), po.attend_grad_bounds(do, q, k, v, **kw)):
        assert got.dtype == t.dtype
        po.assert_within(got, e, bd, tag + " " + name)
    return o, lse


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("head", [1, 5, 8, 24, 32, 40, 64, 72, 80, 96, 100, 120, 128])
def test_attention_head_sizes(head, dtype):
    g = gen(head)
    for b, lq, lk, h, hkv in ((2, 40, 70, 4, 2), (1, 130, 33, 2, 2), (1, 1, 300, 6, 2)):
        check_attend(*make(g, b, lq, lk, h, hkv, head, dtype), tag="%d queries, head %d" % (lq, head))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("lq", [1, 2, 31, 32, 33, 63, 64, 65, 127, 129, 257])
def test_attention_lengths(lq, dtype):
    g = gen(lq)
    for lk in (1, 2, 31, 32, 33, 64, 65, 127, 128, 129, 200, 515):
        check_attend(*make(g, 1, lq, lk, 2, 1, 64, dtype), tag="%d x %d" % (lq, lk))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("h,hkv", [(1, 1), (3, 3), (8, 1), (12, 4), (40, 1), (64, 2)])
def test_attention_shared_heads(h, hkv, dtype):
    g = gen(h)
    for lq, lk in ((1, 400), (3, 50), (50, 77)):
        check_attend(*make(g, 2, lq, lk, h, hkv, 64, dtype), tag="%d heads, %d queries" % (h, lq))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("lq", [1, 45, 200])
@pytest.mark.parametrize("head", [64, 80, 128])
def test_attention_masks(head, lq, dtype):
    """Lengths of zero, one and beyond, masks that leave nothing, and NaN and infinities in all that does not count."""
    g = gen(lq + head)
    b, lk = 7, 150
    q, k, v = make(g, b, lq, lk, 4, 2, head, dtype)
    lengths = torch.tensor([0, 1, 32, 64, 97, 150, 1000], dtype=torch.int32, device="cuda")
    mask = torch.rand(b, lk, generator=g, device="cuda") < 0.6
    mask[5] = False
    mask[3, :40] = False
    mask[6] = torch.arange(lk, device="cuda") == 149
    for kw in (dict(key_lengths=lengths), dict(key_mask=mask), dict(key_lengths=lengths, key_mask=mask)):
        counts = po.counting(q, k, kw.get("key_lengths"), kw.get("key_mask"))
        bad = [x.clone() for x in (k, v)]
        bad[0][~counts] = math.nan
        bad[1][~counts] = math.inf
        o, lse = check_attend(q, k, v, **kw, tag=str(list(kw)))
        p, m = check_attend(q, *bad, **kw, tag=str(list(kw)) + " with NaN")
        assert torch.equal(o, p) and torch.equal(lse, m)
        empty = ~counts.any(1)
        assert (o[empty] == 0).all() and (lse[empty] == -math.inf).all()


def test_attention_gradient_of_rows_without_keys_is_zero():
    import nnv_amd as nnv
    for dtype in TYPES:
        g = gen(3)
        q, k, v = make(g, 2, 5, 70, 2, 2, 64, dtype)
        q[0], do = math.nan, rand(g, 2, 5, 2, 64, dtype=dtype)
        do[0] = math.inf
        lengths = torch.tensor([0, 70], device="cuda")
        o, lse = nnv.cross_attention(q, k, v, lengths)
        dq, dk, dv = nnv.cross_attention_backward(do, q, k, v, o, lse, lengths)
        for t in (o, dq, dk, dv):
            assert (t[0] == 0).all() and torch.isfinite(t).all()
        # no keys at all, no queries, no sequences
        o, lse = nnv.cross_attention(q, k[:, :0], v[:, :0])
        assert (o == 0).all() and (lse == -math.inf).all()
        dq, dk, dv = nnv.cross_attention_backward(do, q, k[:, :0], v[:, :0], o, lse)
        assert (dq == 0).all() and dk.shape == (2, 0, 2, 64)
        o, lse = nnv.cross_attention(q[:, :0], k, v)
        dq, dk, dv = nnv.cross_attention_backward(o, q[:, :0], k, v, o, lse)
        assert (dk == 0).all() and (dv == 0).all() and dq.numel() == 0 and lse.shape == (2, 2, 0)
        assert nnv.cross_attention(q[:0], k[:0], v[:0])[0].shape == (0, 5, 2, 64)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_attention_strides(dtype):
    """Heads first, keys and values side by side in one tensor, rows at odd places, reversed batches, values not dense."""
    import nnv_amd as nnv
    g = gen(8)
    q = rand(g, 2, 4, 50, 64, dtype=dtype).transpose(1, 2)
    kv = rand(g, 2, 90, 2, 2, 64, dtype=dtype)
    check_attend(q, kv[:, :, 0], kv[:, :, 1], tag="side by side")
    odd = rand(g, 2 * 90 * 2 * 67 + 1, dtype=dtype)[1:].view(2, 90, 2, 67)
    check_attend(q[..., 3:], odd[..., 5:66], odd[..., 1:62], tag="odd places")
    check_attend(q, kv[:, :, 0].expand(2, 90, 2, 64), kv[:1, :, 1].expand(2, 90, 2, 64), tag="one sequence for all")
    check_attend(rand(g, 2, 50, 64, 4, dtype=dtype).transpose(2, 3), kv[:, ::2, 0], kv[:, 1::2, 1], tag="every second key")
    mask = torch.rand(90, 2, generator=g, device="cuda") < 0.5
    check_attend(q, kv[:, :, 0], kv[:, :, 1], key_mask=mask.t(), scale=0.3, tag="transposed mask")
    do = rand(g, 2, 4, 50, 64, dtype=dtype).transpose(1, 2)
    o, lse = nnv.cross_attention(q, kv[:, :, 0], kv[:, :, 1])
    one = nnv.cross_attention_backward(do, q, kv[:, :, 0], kv[:, :, 1], o, lse)
    two = nnv.cross_attention_backward(do.contiguous(), q.contiguous(), kv[:, :, 0].contiguous(), kv[:, :, 1].contiguous(), o.clone(), lse)
    assert all(torch.equal(a, b) for a, b in zip(one, two))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_attention_large_and_negative_scores(dtype):
    """Scores far from zero, a few keys that take everything, the largest one in the last tile and in the first."""
    g = gen(21)
    q, k, v = make(g, 1, 70, 333, 2, 2, 64, dtype)
    for at, by in ((0, 30), (332, 30), (100, -30)):
        kk = k.clone()
        kk[:, at] *= by
        check_attend(q * 4, kk, v, tag="key %d" % at)
    check_attend(q, k, v, scale=-0.125, tag="negative scale")
    check_attend(q, k, v, scale=0.0, tag="no scale")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows", [15, 16, 17, 32, 33, 63, 64, 65])
def test_attention_around_the_forms_for_few_rows(rows, dtype):
    """Rows on either side of what the kernels for few rows take, of one head and of eight that share keys; tiles that the keys end in."""
    g = gen(rows)
    for head in (20, 32, 64, 96, 128):
        check_attend(*make(g, 2, rows, 77, 2, 2, head, dtype), backward=False, tag="%d rows, head %d" % (rows, head))
    if rows % 8 == 0:
        check_attend(*make(g, 1, rows // 8, 700, 8, 1, 64, dtype), tag="%d rows of 8 heads" % rows)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_attention_single_tokens_masks_of_many_tiles(dtype):
    """Masks over more tiles than a wave reads them for at a time, in blocks that take all keys of a sequence; strided keys and values."""
    import nnv_amd as nnv
    g = gen(12)
    b, lk, h, d = 16, 5003, 16, 32
    q = rand(g, b, 1, h, d, dtype=dtype)
    kv = rand(g, b, lk, 2, h, d, dtype=dtype)
    mask = torch.rand(b, lk, generator=g, device="cuda") < 0.3
    mask[1, :4900] = False
    mask[2, 128:] = False
    lengths = torch.randint(0, lk + 1, (b,), generator=g, device="cuda")
    kv[~mask] = math.nan
    clean = torch.where(mask[:, :, None, None, None], kv, 0)
    for kw in (dict(key_mask=mask), dict(key_mask=mask, key_lengths=lengths)):
        o, lse = nnv.cross_attention(q, kv[:, :, 0], kv[:, :, 1], **kw)
        eo, el = po.attend(q, clean[:, :, 0], clean[:, :, 1], **kw)
        bo, bl = po.attend_bounds(q, clean[:, :, 0], clean[:, :, 1], **kw)
        po.assert_within(lse, el, bl, "lse")
        po.assert_within(o, eo, bo, "o")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_attention_long_keys_few_rows(dtype):
    """Single tokens against many keys: the split over the keys and what joins it."""
    g = gen(5)
    for b, lk, h, hkv, d in ((1, 20000, 8, 1, 128), (3, 4100, 4, 4, 64), (2, 9000, 2, 1, 80)):
        q, k, v = make(g, b, 1, lk, h, hkv, d, dtype)
        lengths = torch.randint(0, lk + 1, (b,), generator=g, device="cuda")
        lengths[0] = 33
        check_attend(q, k, v, tag="%d keys" % lk)
        check_attend(q, k, v, key_lengths=lengths, tag="%d keys by length" % lk)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_attention_many_rows_few_keys(dtype):
    """The split of the keys' gradients over the rows."""
    g = gen(6)
    check_attend(*make(g, 1, 2100, 77, 4, 2, 64, dtype), tag="rows")
    check_attend(*make(g, 1, 1030, 20, 8, 1, 128, dtype), tag="rows of shared heads")


def test_attention_offsets_beyond_32_bits():
    import nnv_amd as nnv
    g = gen(9)
    lk = 40000
    store = torch.empty(lk * 65536, dtype=BF16, device="cuda")   # 2.6e9 elements, 5.2 GB
    k = store.view(lk, 65536)[:, :64].view(1, lk, 1, 64)
    v = store.view(lk, 65536)[:, 64:128].view(1, lk, 1, 64)
    k.copy_(rand(g, 1, lk, 1, 64, dtype=BF16))
    v.copy_(rand(g, 1, lk, 1, 64, dtype=BF16))
    for lq in (1, 40):
        q = rand(g, 1, lq, 2, 64, dtype=BF16)
        a, b = nnv.cross_attention(q, k, v), nnv.cross_attention(q, k.contiguous(), v.contiguous())
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        do = rand(g, 1, lq, 2, 64, dtype=BF16)
        c, d = (nnv.cross_attention_backward(do, q, x, y, *a) for x, y in ((k, v), (k.contiguous(), v.contiguous())))
        assert all(torch.equal(s, t) for s, t in zip(c, d))


def test_attention_gives_the_same_bits_again():
    import nnv_amd as nnv
    g = gen(10)
    for dtype in TYPES:
        for lq, lk, h, hkv in ((1, 5000, 8, 2), (300, 400, 4, 2), (1500, 60, 2, 1)):
            q, k, v = make(g, 2, lq, lk, h, hkv, 64, dtype)
            do = rand(g, *q.shape, dtype=dtype)
            o, lse = nnv.cross_attention(q, k, v)
            grads = nnv.cross_attention_backward(do, q, k, v, o, lse)
            for _ in range(3):
                again = nnv.cross_attention(q, k, v)
                assert torch.equal(o, again[0]) and torch.equal(lse, again[1])
                assert all(torch.equal(a, b) for a, b in zip(grads, nnv.cross_attention_backward(do, q, k, v, o, lse)))


def test_attention_gradient_against_differences():
    import nnv_amd as nnv
    g = gen(12)
    t = make(g, 2, 9, 40, 4, 2, 24, F32)
    mask = torch.rand(2, 40, generator=g, device="cuda") < 0.7
    do = rand(g, 2, 9, 4, 24)
    o, lse = nnv.cross_attention(*t, key_mask=mask)
    grads = nnv.cross_attention_backward(do, *t, o, lse, key_mask=mask)
    bounds = po.attend_grad_bounds(do, *t, key_mask=mask)
    h = 1e-5
    for i in range(3):
        d = torch.randn(t[i].shape, generator=g, device="cuda", dtype=torch.float64)
        loss = lambda s: float((po.attend(*[u.double() + (s * d if j == i else 0) for j, u in enumerate(t)], key_mask=mask)[0] * do.double()).sum())  # noqa: E731
        slope = (loss(h) - loss(-h)) / (2 * h)
        allowed = float(((bounds[i] + po.U32 * grads[i].double().abs()) * d.abs()).sum()) + 1e-7 * float((grads[i].double().abs() * d.abs()).sum()) + 1e-7
        assert abs(float((grads[i].double() * d).sum()) - slope) <= allowed


# ---- clipping --------------------------------------------------------------------------------------------


def check_clip(grads, threshold, out=None):
    import nnv_amd as nnv
    before = [x.clone() for x in grads]
    got, norm = nnv.clip_gradients(grads, threshold, out=out)
    exact, n = po.clip(before, threshold)
    assert norm.dtype == F32 and norm.dim() == 0
    # squares and sums in f64, one rounding to f32
    assert abs(float(norm) - n) <= 2 * po.U32 * n
    assert len(got) == len(grads)
    for k, (a, e) in enumerate(zip(got, exact)):
        assert a.dtype == before[k].dtype and a.shape == before[k].shape
        po.assert_within(a, e, 6 * po.U32 * e.abs(), "tensor %d" % k)
    if n <= threshold:
        assert all(torch.equal(a, b) for a, b in zip(got, before))
    return got, norm


@pytest.mark.parametrize("count", [1, 2, 5, 95, 96, 97, 250])
def test_clip_many_tensors(count):
    g = gen(count)
    sizes = [(k * 7919) % 9001 for k in range(count)]   # the first is empty
    grads = [rand(g, n, dtype=TYPES[k % 3], scale=0.1) for k, n in enumerate(sizes)]
    for threshold in (0.5, 1e6):
        check_clip(grads, threshold)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_clip_sizes_and_places(dtype):
    g = gen(2)
    # around a pack, a tile and the tiles of all blocks; starting at odd elements; of several dimensions
    store = rand(g, 9_000_000, dtype=dtype)
    for n in (1, 7, 8, 9, 4095, 4096, 4097, 8191, 8193, 8_388_609):
        check_clip([store[3:3 + n]], 0.25)
    check_clip([rand(g, 3, 50, 7, dtype=dtype), rand(g, 20, 30, dtype=dtype).t(), rand(g, 40, 40, dtype=dtype)[::2, ::3]], 0.1)


def test_clip_in_place_into_views_and_at_the_threshold():
    import nnv_amd as nnv
    g = gen(3)
    grads = [rand(g, 3000, dtype=t) for t in TYPES]
    keep = [x.clone() for x in grads]
    got, norm = check_clip(grads, 1.0, out=grads)
    assert all(a is b for a, b in zip(got, grads))
    again, less = check_clip(grads, 1e9, out=grads)
    assert abs(float(less) - 1.0) < 0.01
    views = [torch.zeros(50, 60, device="cuda", dtype=t).t() for t in TYPES]
    got, _ = check_clip([x.view(60, 50) for x in keep], 1.0, out=views)
    assert all(a is b for a, b in zip(got, views))
    x = torch.tensor([3.0, 4.0], device="cuda")
    got, norm = nnv.clip_gradients([x], 5.0)          # a norm at the threshold is not over it
    assert float(norm) == 5.0 and torch.equal(got[0], x)
    got, norm = nnv.clip_gradients([], 1.0)
    assert got == [] and float(norm) == 0
    got, norm = nnv.clip_gradients([x[:0], x * 0], 1.0)
    assert float(norm) == 0 and (got[1] == 0).all()


def test_clip_large_infinite_and_missing_values():
    import nnv_amd as nnv
    x = torch.full((1000,), 1e30, device="cuda")       # squares beyond f32
    got, norm = nnv.clip_gradients([x], 1.0)
    exact, n = po.clip([x], 1.0)
    assert abs(float(norm) / n - 1) < 1e-6
    po.assert_within(got[0], exact[0], 6 * po.U32 * exact[0], "large")
    x[5] = math.inf
    got, norm = nnv.clip_gradients([x], 1.0)
    assert float(norm) == math.inf and torch.isnan(got[0][5]) and (got[0][:5] == 0).all()
    x[5] = math.nan
    got, norm = nnv.clip_gradients([x], 1.0)
    assert torch.isnan(norm) and torch.equal(got[0][:5], x[:5]) and torch.isnan(got[0][5])


# ---- how they are called ------------------------------------------------------------------------------


def test_other_streams_and_graphs():
    """The calls follow torch's current stream: behind what it already holds, and into a graph that is replayed on new inputs."""
    import nnv_amd as nnv
    g = gen(13)
    q, k, v = make(g, 2, 40, 300, 4, 2, 64, BF16)
    x, w = rand(g, 200, 512, dtype=BF16), rand(g, 512, dtype=BF16)

    def everything(q, k, v, x, w):
        y, mean, rstd = nnv.layer_norm(x, w, None)
        o, lse = nnv.cross_attention(q, k, v)
        one, _ = nnv.cross_attention(q[:, :1], k, v)
        grads = list(nnv.cross_attention_backward(o, q, k, v, o, lse)) + list(nnv.layer_norm_backward(y, x, mean, rstd, w))
        clipped, norm = nnv.clip_gradients(grads, 0.5)
        return [y, mean, rstd, o, lse, one, *grads, *clipped, norm]

    expected = everything(q, k, v, x, w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = [torch.zeros_like(t) for t in (q, k, v, x, w)]
        spin = torch.randn(2048, 2048, device="cuda")
        for _ in range(20):
            spin = spin @ spin * 1e-3
        for t, s in zip(late, (q, k, v, x, w)):
            t.copy_(s)
        got = everything(*late)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, expected))

    inputs = [t.clone() for t in (q, k, v, x, w)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = everything(*inputs)
    for seed in (1, 2, 3):
        for t, s in zip(inputs, (q, k, v, x, w)):
            t.copy_(s * seed)
        graph.replay()
        torch.cuda.synchronize()
        fresh = everything(*inputs)
        assert all(torch.equal(a, b) for a, b in zip(held, fresh)), seed


def test_refusals_on_the_gpu():
    import nnv_amd as nnv
    x = torch.zeros(4, 8, device="cuda")
    q = torch.zeros(2, 3, 4, 16, device="cuda")
    bad = [
        (nnv.layer_norm, (x.double(),), "float32, bfloat16 or float16"),
        (nnv.layer_norm, (x[:, :0],), "at least one value"),
        (nnv.layer_norm, (x, x[0, :7]), "one value per channel"),
        (nnv.layer_norm, (x, x[0].half()), "type of the values"),
        (nnv.layer_norm, (x.half(), x[0].half(), x[0]), "the same type"),
        (nnv.layer_norm, (x, x[0].cpu()), "on one GPU"),
        (nnv.layer_norm, (x, None, None, -1.0), "epsilon"),
        (nnv.layer_norm_backward, (x[:2], x, x[:, 0], x[:, 0]), "shape and type of x"),
        (nnv.layer_norm_backward, (x, x, x[:2, 0], x[:, 0]), "what layer_norm returned"),
        (nnv.cross_attention, (q[0], q, q), "batch x tokens"),
        (nnv.cross_attention, (q, q[:, :, :3], q[:, :, :3]), "multiple"),
        (nnv.cross_attention, (q, q[:1], q[:1]), "do not fit"),
        (nnv.cross_attention, (q, q, q[:, :2]), "do not fit"),
        (nnv.cross_attention, (q, q.half(), q.half()), "one type"),
        (nnv.cross_attention, (q, q, q, torch.zeros(3, device="cuda")), "key_lengths"),
        (nnv.cross_attention, (q, q, q, torch.zeros(2, device="cuda")), "key_lengths"),
        (nnv.cross_attention, (q, q, q, None, torch.ones(2, 4, device="cuda", dtype=torch.bool)), "key_mask"),
        (nnv.cross_attention, (q, q, q, None, torch.ones(2, 3, device="cuda")), "key_mask"),
        (nnv.cross_attention, tuple(torch.zeros(1, 2, 1, 136, device="cuda") for _ in range(3)), "1 to 128"),
        (nnv.cross_attention_backward, (q[:1], q, q, q, q, q[..., 0]), "shape and type of q"),
        (nnv.cross_attention_backward, (q, q, q, q, q, q[..., 0]), "what cross_attention returned"),
        (nnv.clip_gradients, ([x], 0.0), "threshold"),
        (nnv.clip_gradients, ([x], math.nan), "threshold"),
        (nnv.clip_gradients, ([x.long()], 1.0), "float32, bfloat16 or float16"),
        (nnv.clip_gradients, ([x, x.cpu()], 1.0), "on one GPU"),
        (nnv.clip_gradients, ([x], 1.0, [x[0]]), "out must have"),
        (nnv.clip_gradients, ([x], 1.0, []), "tensors to write to"),
    ]
    for fn, args, text in bad:
        with pytest.raises(ValueError, match=text):
            fn(*args)
    with pytest.raises(TypeError):
        nnv.layer_norm([1.0, 2.0])


def test_library_refuses_a_small_workspace():
    import ctypes as C

    import nnv_amd as nnv
    from nnv_amd import _lib, points
    ctx = nnv.default_context()
    x = torch.zeros(4000, 64, device="cuda")
    n = C.c_int64()
    _lib.check(ctx.lib.nnvhip_layer_norm_backward_workspace(0, 4000, 64, C.byref(n)))
    assert n.value > 0
    work = torch.zeros(n.value, dtype=torch.uint8, device="cuda")
    args = [ctx.handle, 0, 0, 4000, 64, x.data_ptr(), 64, x.data_ptr(), 64, x.data_ptr(), x.data_ptr(), None, x.data_ptr(), x.data_ptr(), x.data_ptr()]
    with pytest.raises(_lib.NNVHipError, match="workspace"):
        _lib.check(ctx.lib.nnvhip_layer_norm_backward(*args, work.data_ptr(), n.value - 4, None))
    with pytest.raises(_lib.NNVHipError, match="workspace"):
        _lib.check(ctx.lib.nnvhip_layer_norm_backward(*args, None, n.value, None))
    d = points._ATTENTION.pack(0, 1, 1, 9000, 1, 1, 64, 0.125, *[0] * 25)
    with pytest.raises(_lib.NNVHipError, match="null pointer"):
        _lib.check(ctx.lib.nnvhip_cross_attention(ctx.handle, d, work.data_ptr(), 1 << 40, None))


def test_layers_forward_and_backward():
    import nnv_amd as nnv
    g = gen(14)
    norm = nnv.LayerNormalizationLayer(Scale=rand(g, 128, shift=1.0), Offset=rand(g, 128))
    attend = nnv.CrossAttentionLayer(NumHeads=4, NumKeyValueHeads=2)
    x, k, v = rand(g, 2, 10, 128), rand(g, 2, 30, 64), rand(g, 2, 30, 64)
    y, saved = norm.forward(x)
    assert torch.equal(y, norm.evaluate(x))
    o, kept = attend.forward(y, k, v)
    assert o.shape == x.shape and torch.equal(o, attend.evaluate(y, k, v))
    dy, dk, dv = attend.backward(o, kept)
    dx, (dscale, doffset) = norm.backward(dy, saved)
    assert dk.shape == k.shape and dx.shape == x.shape and dscale.shape == doffset.shape == (128,)
    with pytest.raises(ValueError, match="number of channels"):
        norm.evaluate(x[..., :64])
    with pytest.raises(ValueError, match="multiple of the number of heads"):
        attend.evaluate(y[..., :126], k, v)
