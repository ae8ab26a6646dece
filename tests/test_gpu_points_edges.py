"""The operators on points (nnv_amd.points) on the GPU, where calls are rare: lengths in 64 bits, infinite values in keys that count, scores far
from zero, weights far below one, gradients whose norm passes f32, many sequences of many keys, and the steady state of the kernels that keep
several tiles on their way."""
import math

import pytest
import torch

from tests import points_oracle as po
from tests.test_gpu_points import BF16, F16, F32, IDS, TYPES, check_attend, gen, make, rand

pytestmark = pytest.mark.gpu


# ---- lengths -------------------------------------------------------------------------------------------------


def test_lengths_in_64_bits():
    """A length beyond the keys is taken as all of them, one below zero as none, whatever its upper half says."""
    import nnv_amd as nnv
    lengths = torch.tensor([2 ** 31, 2 ** 32, 2 ** 63 - 1, 2 ** 32 + 5, -2 ** 63, -2 ** 32 + 3, -1, 3, 70], device="cuda")
    plain = torch.tensor([70, 70, 70, 70, 0, 0, 0, 3, 70], dtype=torch.int32, device="cuda")
    for dtype in (F32, BF16):
        g = gen(1)
        q, k, v = make(g, 9, 5, 70, 2, 1, 64, dtype)
        do = rand(g, *q.shape, dtype=dtype)
        o, lse = nnv.cross_attention(q, k, v, lengths)
        eo, el = nnv.cross_attention(q, k, v, plain)
        assert torch.equal(o, eo) and torch.equal(lse, el)
        for a, b in zip(nnv.cross_attention_backward(do, q, k, v, o, lse, lengths), nnv.cross_attention_backward(do, q, k, v, o, lse, plain)):
            assert torch.equal(a, b)


# ---- infinite values that count --------------------------------------------------------------------------------


def check_infinite_values(rows, head, dtype):
    import nnv_amd as nnv
    g = gen(rows + head)
    q, k, v = make(g, 2, rows, 90, 2, 2, head, dtype)
    v[0, 3, 0, 1], v[0, 70, 0, 1] = math.inf, math.inf
    v[0, 89, 1, 4] = -math.inf
    o, lse = nnv.cross_attention(q, k, v)
    po.assert_within(lse, po.attend(q, k, v)[1], po.attend_bounds(q, k, v)[1], "%d rows, head %d: lse" % (rows, head))
    po.assert_within(o, po.attend(q, k, v)[0], po.attend_bounds(q, k, v)[0], "%d rows, head %d" % (rows, head))
    v[1, 5, 0, 2], v[1, 60, 0, 2], v[1, 7, 1, 3] = math.inf, -math.inf, math.nan
    o, _ = nnv.cross_attention(q, k, v)
    none = torch.zeros_like(o, dtype=torch.bool)
    none[1, :, 0, 2] = none[1, :, 1, 3] = True
    assert torch.equal(torch.isnan(o), none)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 16, 17, 32, 33, 64, 65, 200])
def test_infinite_values_of_keys_that_count_in_16_bits(rows, dtype):
    """A weight is above zero, so that an infinite value makes the result infinite, and nothing else, however many rows there are."""
    for head in (40, 64, 128):
        check_infinite_values(rows, head, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows", [1, 16, 17, 32, 33, 64, 65, 200])
def test_infinite_values_where_products_are_cut(rows, dtype):
    """The same in f32, and in 16 bits with rows that cannot be moved in 16-byte pieces."""
    for head in (5, 40, 64, 99, 128) if dtype == F32 else (5, 99):
        check_infinite_values(rows, head, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows", [1, 16, 17, 32, 33, 64, 65, 200])
def test_scores_of_minus_infinity(rows, dtype):
    """A key whose scores are all -inf, by an infinity in it or in the queries, has no weight."""
    import nnv_amd as nnv
    for head in (5, 40, 64, 128):
        g = gen(rows + head)
        q, k, v = make(g, 1, rows, 90, 2, 2, head, dtype)
        q[..., 1] = -q[..., 1].abs() - 0.25
        k[0, 31, :, 1] = math.inf
        check_attend(q, k, v, backward=False, tag="%d rows, head %d, keys" % (rows, head))
        q, k, v = make(g, 1, rows, 90, 2, 2, head, dtype)
        q[0, rows // 2, :, 2] = math.inf
        k[..., 2] = -k[..., 2].abs() - 0.25
        k[0, 50, :, 2] = 0.0                      # inf * 0: no number
        o, _ = nnv.cross_attention(q, k, v)
        none = torch.zeros_like(o, dtype=torch.bool)
        none[0, rows // 2] = True
        assert torch.equal(torch.isnan(o), none)


# ---- products of f32 -------------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows", [1, 20, 4096])
def test_products_of_f32_are_rounded_like_f32(rows):
    """One key, heads of one value: lse is the product.  It is rounded as a product, times scale / ln 2 (a rounded number), in the sum with the
    logarithm of one, and times ln 2 (a rounded number): five roundings of 2^-24 at most, and what the pieces leave out, below 2^-24."""
    import nnv_amd as nnv
    g = gen(rows)
    q = 1 + torch.rand(64, rows, 1, 1, generator=g, device="cuda")
    k = 1 + torch.rand(64, 1, 1, 1, generator=g, device="cuda")
    q[32:], k[32:] = 1.0078124 - (q[32:] - 1) * 2.0 ** -18, 1.0078124    # the largest numbers behind seven zeros
    q[:, ::2] *= -1
    _, lse = nnv.cross_attention(q, k, torch.ones_like(k), scale=1.0)
    exact = (q.double() * k.double())[:, :, 0, 0]
    err = ((lse[:, 0] - exact) / exact.abs()).abs()
    assert float(err.max()) <= 6 * po.U32, "%.2f" % (float(err.max()) / po.U32)


def test_sums_of_f32_products_have_no_drift():
    """The mean error of many products is a small part of one rounding, if those go either way: 2^18 of them, each within six, leave a
    mean below 1/8 beside what the two rounded constants are off."""
    import nnv_amd as nnv
    g = gen(3)
    q = 1 + torch.rand(64, 4096, 1, 1, generator=g, device="cuda")
    k = 1 + torch.rand(64, 1, 1, 1, generator=g, device="cuda")
    _, lse = nnv.cross_attention(q, k, torch.ones_like(k), scale=1.0)
    f = lambda x: float(torch.tensor(x, dtype=F32))  # noqa: E731
    exact = (q.double() * k.double())[:, :, 0, 0] * (f(1 / math.log(2)) * f(math.log(2)))
    assert abs(float(((lse[:, 0] - exact) / exact).mean())) <= po.U32 / 8


# ---- scores and weights at the ends of their range ---------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("head", [64, 128])
def test_scores_beyond_the_integers_of_f32(head, dtype):
    """Scores of some 2^28 to 2^32, whose roundings are larger than the distance of any two exponents: the key with the largest score takes all."""
    import nnv_amd as nnv
    for rows in (1, 20, 70, 130):
        g = gen(rows)
        q, k, v = make(g, 2, rows, 300, 2, 1, head, dtype)
        size = (1 + torch.rand(2, rows, 2, 1, generator=g, device="cuda") * 3) * 4000
        q = size.expand(-1, -1, -1, head).to(dtype)
        order = torch.stack([torch.randperm(300, generator=g, device="cuda") for _ in range(2)])
        k = (8000.0 + 16 * order)[:, :, None, None].expand(-1, -1, 1, head).to(dtype) * (1 if dtype != BF16 else 1)
        if dtype == BF16:   # fewer different numbers: the largest one alone
            k = torch.where(order[:, :, None, None] == 299, 16000.0, 8000.0).expand(-1, -1, 1, head).to(dtype)
        o, lse = nnv.cross_attention(q, k, v)
        best = order.argmax(1)
        expected = torch.stack([v[i, best[i]] for i in range(2)])[:, None].expand(2, rows, 2, head)
        assert torch.equal(o, expected), "%d rows" % rows
        exact = (q.double().permute(0, 2, 1, 3)[..., 0] * torch.stack([k[i, best[i], 0, 0] for i in range(2)]).double()[:, None, None]) * head ** 0.5
        assert float(((lse - exact) / exact).abs().max()) <= (head + 8) * po.U32


@pytest.mark.parametrize("batch,rows", [(256, 1), (256, 33), (512, 65)])
def test_many_small_weights_of_f16(batch, rows):
    """Eight keys of weight 1, one in the first tile of each wave of a block, and 2^20 of some 2^-26: f16's smallest number is 2^-24, and what they hold
    together is 2^-9 of the result.  A weight may be off by half of f16's last place, or, with the largest at 2^7 or more, by 2^-32.  (The sequences are
    as many as keep a block with all keys of one; they share their keys.)"""
    import nnv_amd as nnv
    n = 1 << 20
    q = torch.ones(1, rows, 1, 8, dtype=F16, device="cuda").expand(batch, -1, -1, -1)
    k = torch.full((1, n + 8, 1, 8), -18.02 / 8, dtype=F16, device="cuda")
    v = torch.ones(1, n + 8, 1, 8, dtype=F16, device="cuda")
    w = n * math.exp(float(k[0, 0, 0].double().sum()))
    k[0, :256:32], v[0, :256:32] = 0.0, 0.0
    o, lse = nnv.cross_attention(q, k.expand(batch, -1, -1, -1), v.expand(batch, -1, -1, -1), scale=1.0)
    exact = w / (8 + w)
    assert float((o.double() - exact).abs().max()) <= (n * 2.0 ** -32 + 2 * 2.0 ** -11 * w) / 8
    # (a sum of n terms, as in the oracle's bounds)
    assert float((lse.double() - math.log(8 + w)).abs().max()) <= (n + 32) * po.U32


# ---- sizes ---------------------------------------------------------------------------------------------------


def test_many_sequences_of_many_keys():
    """A token each for 64 sequences of 65536 keys, 64 heads on 8: 17 GB of keys and values, were the sequences not one and the same here."""
    import nnv_amd as nnv
    g = gen(4)
    q, k, v = make(g, 1, 1, 65536, 64, 8, 128, BF16)
    lengths = torch.arange(64, 0, -1, device="cuda", dtype=torch.int32) * 1024
    o, lse = nnv.cross_attention(q.expand(64, -1, -1, -1), k.expand(64, -1, -1, -1), v.expand(64, -1, -1, -1), lengths)
    for i in (0, 1, 40, 63):
        n = int(lengths[i])
        (eo, el), (bo, bl) = po.attend(q, k[:, :n], v[:, :n]), po.attend_bounds(q, k[:, :n], v[:, :n])
        po.assert_within(lse[i:i + 1], el, bl, "lse of sequence %d" % i)
        po.assert_within(o[i:i + 1], eo, bo, "sequence %d" % i)


# ---- arguments -----------------------------------------------------------------------------------------------


def test_scales_that_are_no_numbers_and_heads_of_nothing_are_refused():
    import nnv_amd as nnv
    for dtype in TYPES:
        q = torch.zeros(1, 2, 2, 16, device="cuda", dtype=dtype)
        o, lse = nnv.cross_attention(q, q, q)
        for scale in (math.nan, math.inf, -math.inf, 1e39):
            with pytest.raises(ValueError, match="scale"):
                nnv.cross_attention(q, q, q, scale=scale)
            with pytest.raises(ValueError, match="scale"):
                nnv.cross_attention_backward(q, q, q, q, o, lse, scale=scale)
        with pytest.raises(ValueError, match="1 to 128"):
            nnv.cross_attention(q[..., :0], q[..., :0], q[..., :0])

def test_tensors_that_require_gradients_are_refused_unless_nobody_asks():
    """The results are not part of torch's graph: where torch records one, a call says so."""
    import nnv_amd as nnv
    x, w = torch.randn(4, 8, device="cuda"), torch.ones(8, device="cuda", requires_grad=True)
    q, k = torch.randn(1, 2, 2, 16, device="cuda"), torch.randn(1, 3, 2, 16, device="cuda", requires_grad=True)
    with torch.no_grad():
        y, mean, rstd = nnv.layer_norm(x, w)
        o, lse = nnv.cross_attention(q, k, k)
    for call in (lambda: nnv.layer_norm(x, w), lambda: nnv.layer_norm_backward(x, x, mean, rstd, w), lambda: nnv.cross_attention(q, k, k),
                 lambda: nnv.cross_attention_backward(q, q, k, k, o, lse), lambda: nnv.clip_gradients([x, w], 1.0),
                 lambda: nnv.clip_gradients([x], 1.0, out=[torch.empty_like(x).requires_grad_()])):
        with pytest.raises(ValueError, match="no_grad"):
            call()
        with torch.no_grad():
            call()
    assert torch.equal(y, nnv.layer_norm(x, w.detach())[0]) and torch.equal(o, nnv.cross_attention(q, k.detach(), k.detach())[0])


# ---- clipping ------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_clip_a_norm_beyond_f32(dtype):
    """Finite gradients whose norm f32 does not hold: it is told as infinite, and the gradients are scaled by what it is."""
    import nnv_amd as nnv
    grads = [torch.full((1000,), 2e38, device="cuda", dtype=dtype), torch.full((3, 50), -3e38, device="cuda", dtype=dtype),
             torch.full((20,), 1e30, device="cuda", dtype=dtype)]
    exact, n = po.clip(grads, 1.0)
    assert n > 3.5e38
    got, norm = nnv.clip_gradients(grads, 1.0)
    assert float(norm) == math.inf
    for a, e in zip(got, exact):
        po.assert_within(a, e, 6 * po.U32 * e.abs(), "beyond f32")
    got, _ = nnv.clip_gradients(grads, 1e39)
    for a, e in zip(got, po.clip(grads, 1e39)[0]):
        po.assert_within(a, e, 6 * po.U32 * e.abs(), "a threshold beyond f32")
    got, _ = nnv.clip_gradients(grads, 1e300)
    assert all(torch.equal(a, b) for a, b in zip(got, grads))

def test_clip_refuses_outputs_that_share_memory():
    """Blocks would read what others have written: the same tensor twice, two in the wrong order, one shifted against its gradient."""
    import nnv_amd as nnv
    g = gen(5)
    store = rand(g, 100000)
    a, b = store[:40000], store[50000:90000]
    for grads, out in (([a, a], [a, a]), ([a, b], [b, a]), ([a], [store[1:40001]]), ([b], [store[49999:89999]]),
                       ([a, b], [torch.empty_like(a), store[39999:79999]]), ([a, store[100:200]], [a, store[100:200]])):
        with pytest.raises(ValueError, match="overlaps"):
            nnv.clip_gradients(grads, 1.0, out=out)
    before = store.clone()
    exact, _ = po.clip([a, a, b, a[:0]], 1.0)
    got, _ = nnv.clip_gradients([a, a, b, a[:0]], 1.0)      # read twice, written to new memory
    assert torch.equal(store, before)
    for x, e in zip(got, exact):
        po.assert_within(x, e, 6 * po.U32 * e.abs(), "the same gradient twice")
    exact, _ = po.clip([a, b, a[:0]], 1.0)
    got, _ = nnv.clip_gradients([a, b, a[:0]], 1.0, out=[a, torch.empty_like(b), a[:0]])
    for x, e in zip(got, exact):
        po.assert_within(x, e, 6 * po.U32 * e.abs(), "in place and not")
    # next to one another
    half = [store[:50000], store[50000:]]
    exact, _ = po.clip(half, 0.5)
    got, _ = nnv.clip_gradients(half, 0.5, out=half)
    for x, e in zip(got, exact):
        po.assert_within(x, e, 6 * po.U32 * e.abs(), "neighbours")


# ---- the steady state of kernels that keep several tiles on their way ------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("head", [48, 72, 80, 96, 128])
def test_many_tiles_of_keys(head, dtype):
    """More tiles of keys than the forms for many rows hold at a time, and keys that end next to a tile's and a round's end."""
    g = gen(head)
    for rows in (65, 129, 257, 300):
        for keys in (191, 192, 193, 255, 256, 257, 321, 515):
            q, k, v = make(g, 2, rows, keys, 2, 1, head, dtype)
            lengths = torch.tensor([keys, 1 + keys * 3 // 4], dtype=torch.int32, device="cuda")
            check_attend(q, k, v, backward=keys in (257, 515), tag="%d x %d, head %d" % (rows, keys, head))
            check_attend(q, k, v, key_lengths=lengths, backward=keys == 321, tag="%d x %d by length, head %d" % (rows, keys, head))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("batch,kv_heads,head", [(1, 2, 128), (1, 2, 32), (8, 32, 72), (8, 32, 128), (8, 64, 32)])
def test_masks_over_many_tiles_of_keys(batch, kv_heads, head, dtype):
    """2177 keys, more than a mask is read for at a time, in blocks that take them all (256 of heads above 64, 512 of others) and in blocks
    that share them; whatever is left out is NaN."""
    import nnv_amd as nnv
    g = gen(batch + head)
    keys = 2177
    q, k, v = make(g, batch, 65, keys, kv_heads, kv_heads, head, dtype)
    mask = torch.rand(batch, keys, generator=g, device="cuda") < 0.5
    mask[0, :2100] = False
    lengths = torch.randint(2050, keys + 1, (batch,), generator=g, device="cuda")
    for kw in (dict(key_mask=mask), dict(key_mask=mask, key_lengths=lengths)):
        counts = po.counting(q, k, kw.get("key_lengths"), mask)[:, :, None, None]
        o, lse = nnv.cross_attention(q, torch.where(counts, k, math.nan), torch.where(counts, v, math.nan), **kw)
        for i in range(0, batch, 7):     # (a sequence at a time: the oracle's 64-bit scores)
            one = dict(key_mask=counts[i:i + 1, :, 0, 0])
            (eo, el), (bo, bl) = po.attend(q[i:i + 1], k[i:i + 1], v[i:i + 1], **one), po.attend_bounds(q[i:i + 1], k[i:i + 1], v[i:i + 1], **one)
            po.assert_within(lse[i:i + 1], el, bl, "lse")
            po.assert_within(o[i:i + 1], eo, bo, "o")


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("head", [32, 64, 80, 128])
def test_masks_of_single_tokens_over_many_tiles_of_keys(head, dtype):
    """9001 keys in blocks that take them all: eight waves of heads up to 64, four of others, read a mask for 32 tiles each at a time."""
    import nnv_amd as nnv
    g = gen(head)
    batch, keys, heads = 16, 9001, 16
    q = rand(g, batch, 1, heads, head, dtype=dtype)
    kv = rand(g, batch, keys, 2, heads, head, dtype=dtype)
    mask = torch.rand(batch, keys, generator=g, device="cuda") < 0.3
    mask[1, :8900] = False
    mask[2, 8000:] = False
    clean = kv.clone()
    kv[~mask] = math.nan
    o, lse = nnv.cross_attention(q, kv[:, :, 0], kv[:, :, 1], key_mask=mask)
    for i in (0, 1, 2, 15):
        s = slice(i, i + 1)
        args, kw = (q[s], clean[s, :, 0], clean[s, :, 1]), dict(key_mask=mask[s])
        (eo, el), (bo, bl) = po.attend(*args, **kw), po.attend_bounds(*args, **kw)
        po.assert_within(lse[s], el, bl, "lse")
        po.assert_within(o[s], eo, bo, "o")
