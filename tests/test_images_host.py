"""The operators on points that are images or videos as far as they go without a GPU: their refusals, their workspaces, and their
plain forms in 64 bits (tests/images_oracle.py) against torch's own differentiation."""
import ctypes as C
import math
import os

import numpy as np
import pytest
import torch

from tests import images_oracle as io

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nnv_amd", "libnnvhip.so")
built = pytest.mark.skipif(not os.path.exists(LIB), reason="library not built (python -m nnv_amd.build)")


class OnGpu(torch.Tensor):
    """A host tensor that says it is on GPU 0, for what is checked before anything is launched."""

    @staticmethod
    def __new__(cls, t):
        return t.as_subclass(cls)

    def get_device(self):
        return 0


@pytest.fixture
def no_gpu(monkeypatch):
    """The operators' checks without a GPU: a context that has no library."""
    from nnv_amd import images, points

    class Context:
        lib, handle, device = None, None, 0

    context = Context()
    monkeypatch.setattr(points, "context_on", lambda index: context)
    monkeypatch.setattr(points, "_stream_of", lambda index: 0)
    return images


def refused(match, call, *args, error=ValueError, **kw):
    with pytest.raises(error, match=match):
        call(*args, **kw)


def test_tensors_on_the_host_are_refused():
    import nnv_amd as nnv
    x = torch.zeros(2, 3, 4, 8)
    refused("on the GPU", nnv.group_norm, x, 2)
    refused("on the GPU", nnv.group_norm_backward, x, x, torch.zeros(2, 2), torch.zeros(2, 2))
    refused("on the GPU", nnv.rotate_positions, x, torch.zeros(3, 1, dtype=torch.int32), [2])
    refused("expected torch tensors", nnv.group_norm, 3.0, 2, error=TypeError)
    refused("expected torch tensors", nnv.rotate_positions, [3.0], x, [2], error=TypeError)


def test_refusals_of_group_norm(no_gpu):
    x, w = OnGpu(torch.zeros(2, 3, 4, 8)), OnGpu(torch.zeros(8))
    call = no_gpu.group_norm
    for groups in (0, 3, -2, 2.0, None):
        refused("equal groups", call, x, groups)
    refused("batch x", call, OnGpu(torch.zeros(8)), 2)
    refused("at least one place", call, OnGpu(torch.zeros(2, 0, 8)), 2)
    refused("activation", call, x, 2, activation="tanh")
    refused("activation", call, x, 2, activation=False)
    refused("float32, bfloat16 or float16", call, OnGpu(torch.zeros(2, 3, 8, dtype=torch.float64)), 2)
    refused("one value per channel", call, x, 2, OnGpu(torch.zeros(4)))
    refused("type of the values", call, OnGpu(x.bfloat16()), 2, OnGpu(w.half()))
    refused("same type", call, OnGpu(x.bfloat16()), 2, OnGpu(w.bfloat16()), w)
    refused("epsilon", call, x, 2, epsilon=-1e-5)
    refused("epsilon", call, x, 2, epsilon=math.nan)
    refused("requires a gradient", call, x, 2, OnGpu(torch.zeros(8)).requires_grad_())
    back, stats = no_gpu.group_norm_backward, OnGpu(torch.zeros(2, 4))
    refused("shape and type of x", back, OnGpu(torch.zeros(2, 3, 4, 4)), x, stats, stats)
    refused("shape and type of x", back, OnGpu(x.half()), x, stats, stats)
    refused("what group_norm returned", back, x, x, stats, OnGpu(torch.zeros(2, 2)))
    refused("what group_norm returned", back, x, x, OnGpu(torch.zeros(3, 4)), OnGpu(torch.zeros(3, 4)))
    refused("what group_norm returned", back, x, x, OnGpu(stats.double()), OnGpu(stats.double()))
    refused("equal groups", back, x, x, OnGpu(torch.zeros(2, 3)), OnGpu(torch.zeros(2, 3)))


def test_refusals_of_rotary_positions(no_gpu):
    x, at = OnGpu(torch.zeros(2, 5, 3, 8)), OnGpu(torch.zeros(5, 2, dtype=torch.int32))
    call = no_gpu.rotate_positions
    refused("at least one tensor", call, [], at, [2, 2])
    for sections in ([], [0, 0], [-1, 3], [1.5, 2], [200, 57]):
        refused("sections", call, x, at, sections)
    refused("do not hold", call, x, at, [3, 2])
    refused("base", call, x, at, [2, 2], base=0.0)
    refused("base", call, x, at, [2, 2], base=math.inf)
    refused("alike", call, OnGpu(torch.zeros(2, 5, 8)), at, [2, 2])
    for other in (torch.zeros(2, 4, 3, 8), torch.zeros(2, 5, 3, 4), torch.zeros(2, 5, 3, 8, dtype=torch.bfloat16)):
        refused("alike", call, [x, OnGpu(other)], at, [2, 2])
    for bad in (torch.zeros(5, 3, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(3, 5, 2, dtype=torch.int32),
                torch.zeros(5, 2, dtype=torch.float64), torch.zeros(2, dtype=torch.int32)):
        refused("positions", call, x, OnGpu(bad), [2, 2])
    refused("float32, bfloat16 or float16", call, OnGpu(x.double()), at, [2, 2])


def test_sections_that_are_no_whole_numbers_are_refused_whatever_was_called_before(no_gpu):
    x, at = OnGpu(torch.zeros(2, 5, 3, 8)), OnGpu(torch.zeros(5, 3, dtype=torch.int32))   # (positions of other axes: refused after the sections)
    for accepted in ([1, 2], (np.int64(1), np.int32(2)), np.array([1, 2])):
        refused("positions", no_gpu.rotate_positions, x, at, accepted)
        for sections in ([1.0, 2.0], [1, 2.0], (np.float32(1), 2), [1, None], ["1", 2]):
            refused("sections", no_gpu.rotate_positions, x, at, sections)


def test_frequencies_live_as_long_as_a_call_that_reads_them(no_gpu, monkeypatch):
    """The library is handed their addresses: other calls, which push them out of the caches meanwhile, must not free them."""
    import gc
    import weakref

    from nnv_amd import points

    held, read = [], []

    class Library:
        @staticmethod
        def nnvhip_rotate_positions(handle, d, stream):
            no_gpu._turns.cache_clear()
            no_gpu._frequencies.cache_clear()
            gc.collect()
            read.append([array() is not None for array in held])
            return 0

    class Context:
        lib, handle, device = Library, None, 0

    monkeypatch.setattr(points, "context_on", lambda index: Context)
    held += [weakref.ref(array) for array in no_gpu._frequencies((2, 1), 77.0, False)]
    x, at = OnGpu(torch.zeros(2, 5, 3, 8)), OnGpu(torch.zeros(5, 2, dtype=torch.int32))
    no_gpu.rotate_positions([x] * 5, at, [2, 1], base=77.0)
    assert read == [[True, True]] * 2


@built
def test_workspaces_and_their_refusals():
    from nnv_amd import _lib, images
    lib, n = _lib.load(), C.c_int64()

    def group(backward=False, **kw):
        s = dict(type=1, param_type=1, activation=2, batch=4, places=1000, channels=64, groups=8)
        s.update(kw)
        fn = lib.nnvhip_group_norm_backward_workspace if backward else lib.nnvhip_group_norm_workspace
        _lib.check(fn(images._GROUP.pack(*s.values(), 1e-5, *[0] * 14), C.byref(n)))
        return n.value

    # sums of parts of the places, where they are too many for a block; sums of the channels in the backward pass
    assert group() == 0 and group(places=1 << 20) >= 4 * 8 * 16 and group(backward=True) >= 4 * 64 * 8 and group(batch=0) == 0
    assert group(backward=True, places=1 << 20) >= group(places=1 << 20) + 4 * 64 * 8
    # what is kept of long places stays a small part of them
    assert group(backward=True, places=1 << 24, batch=1) < (1 << 24) * 64 * 2 / 16
    assert group(channels=1 << 20, groups=1) > 0 and group(channels=5000, groups=5000) > 0
    for kw in (dict(type=3), dict(param_type=2), dict(activation=3), dict(groups=7), dict(groups=0), dict(places=0), dict(channels=0), dict(batch=-1),
               dict(batch=1 << 23), dict(channels=1 << 24, groups=1), dict(places=1 << 40), dict(batch=1 << 22, channels=2048), dict(places=1 << 39), dict(places=1 << 36, channels=1, groups=1)):
        for backward in (False, True):
            with pytest.raises((ValueError, _lib.NNVHipError)):
                group(backward, **kw)


@pytest.mark.parametrize("activation", [None, "relu", "silu"])
def test_plain_group_norm_is_differentiated_right(activation):
    torch.manual_seed(3)
    x, w, b = (torch.randn(*s, dtype=torch.float64, requires_grad=True) for s in ((3, 4, 5, 12), (12,), (12,)))
    dy = torch.randn(3, 4, 5, 12, dtype=torch.float64)
    y, mean, rstd = io.group(x, 4, w, b, 1e-5, activation)
    y.backward(dy)
    for got, t in zip(io.group_grad(dy, x.detach(), mean.detach(), rstd.detach(), w.detach(), b.detach(), activation), (x, w, b)):
        assert torch.allclose(got, t.grad, rtol=1e-11, atol=1e-11)
    plain = torch.nn.functional.group_norm(x.permute(0, 3, 1, 2), 4, w, b, 1e-5).permute(0, 2, 3, 1)
    act = {None: lambda u: u, "relu": torch.relu, "silu": torch.nn.functional.silu}[activation]
    assert torch.allclose(y, act(plain), rtol=1e-11, atol=1e-11)


def test_plain_rotation_by_hand():
    x = torch.arange(1.0, 9.0, dtype=torch.float64).view(1, 1, 1, 8)
    at = torch.tensor([[2, 5]])
    y = io.rotate(x, at, [1, 2], base=100.0)[0, 0, 0]
    for i, (t, a, b) in enumerate([(2.0, 1, 4), (5.0, 2, 5), (0.5, 3, 6)]):
        assert torch.allclose(y[[i, i + 3]], torch.tensor([a * math.cos(t) - b * math.sin(t), a * math.sin(t) + b * math.cos(t)], dtype=torch.float64))
    assert torch.equal(y[6:], x[0, 0, 0, 6:])
    z = io.rotate(x, at, [1, 2], base=100.0, shared=True, interleaved=True)[0, 0, 0]
    for i, t in enumerate([2.0, 5 * 100 ** (-1 / 3), 5 * 100 ** (-2 / 3)]):
        a, b = x[0, 0, 0, 2 * i], x[0, 0, 0, 2 * i + 1]
        assert torch.allclose(z[[2 * i, 2 * i + 1]], torch.stack([a * math.cos(t) - b * math.sin(t), a * math.sin(t) + b * math.cos(t)]))
    # turned back: the gradient
    assert torch.allclose(io.rotate(io.rotate(x, at, [2, 2]), at, [2, 2], inverse=True), x)
    # frequencies as the operator forms them
    from nnv_amd.images import _frequencies
    f, axes = _frequencies((1, 2), 100.0, True)
    assert list(axes) == [0, 1, 1] and [round(v, 12) for v in f] == [round(100.0 ** (-i / 3), 12) for i in range(3)]
    f, axes = _frequencies((2, 1), 100.0, False)
    assert list(axes) == [0, 0, 1] and list(f) == [1.0, 0.1, 1.0]


def test_refusals_of_differential_attention(no_gpu):
    import nnv_amd as nnv
    x = torch.zeros(2, 3, 4, 8)
    refused("on the GPU", nnv.differential_attention, x, x, torch.zeros(2, 3, 2, 16), torch.zeros(2))
    q, k, v, w = (OnGpu(torch.zeros(*s)) for s in ((2, 5, 8, 16), (2, 7, 4, 16), (2, 7, 2, 32), (4,)))
    call = no_gpu.differential_attention
    refused("batch x tokens", call, OnGpu(q[0]), k, v, w)
    for bad in ((2, 7, 2, 16), (2, 6, 4, 16), (1, 7, 4, 16), (2, 7, 4, 8)):
        refused("fit together", call, q, OnGpu(torch.zeros(bad)), v, w)
    for bad in ((2, 7, 2, 16), (2, 7, 4, 32), (2, 8, 2, 32)):
        refused("fit together", call, q, k, OnGpu(torch.zeros(bad)), w)
    refused("one type", call, q, OnGpu(k.half()), v, w)
    refused("float32, bfloat16 or float16", call, *(OnGpu(t.double()) for t in (q, k, v)), w)
    refused("1 to 128", call, *(OnGpu(torch.zeros(*s)) for s in ((2, 5, 8, 129), (2, 7, 4, 129), (2, 7, 2, 258))), w)
    refused("two maps", call, OnGpu(q[:, :, :7]), k, v, w)
    refused("two maps", call, OnGpu(q[:, :, :6]), k, v, w)
    refused("two maps", call, OnGpu(q[:, :, :0]), k, v, w)
    refused("one value per head", call, q, k, v, OnGpu(torch.zeros(8)))
    refused("type of the values", call, *(OnGpu(t.half()) for t in (q, k, v)), OnGpu(w.bfloat16()))
    refused("float32, bfloat16 or float16", call, q, k, v, OnGpu(w.double()))
    refused("key_lengths", call, q, k, v, w, OnGpu(torch.zeros(3, dtype=torch.int32)))
    refused("key_lengths", call, q, k, v, w, OnGpu(torch.zeros(2)))
    refused("key_mask", call, q, k, v, w, key_mask=OnGpu(torch.zeros(2, 5, dtype=torch.bool)))
    refused("finite", call, q, k, v, w, scale=math.inf)
    refused("finite", call, q, k, v, w, scale=math.nan)
    back, o, lse = no_gpu.differential_attention_backward, OnGpu(torch.zeros(2, 5, 4, 32)), OnGpu(torch.zeros(2, 8, 5))
    for bad in (None, OnGpu(torch.zeros(2, 5, 4, 16)), OnGpu(o.half())):
        refused("for_backward", back, o, q, k, v, w, o, lse, bad)
    refused("for_backward", back, OnGpu(o[:1]), q, k, v, w, o, lse, o)
    for bad in (OnGpu(torch.zeros(2, 4, 5)), OnGpu(lse.double())):
        refused("lse", back, o, q, k, v, w, o, bad, o)
    refused("requires a gradient", call, q, k, v, OnGpu(torch.zeros(4)).requires_grad_())


@built
def test_workspaces_of_differential_attention_and_their_refusals():
    from nnv_amd import _lib, images
    lib, n = _lib.load(), C.c_int64()

    def differ(backward=False, **kw):
        s = dict(type=1, weight_type=1, batch=2, queries=100, keys=200, heads=4, kv_heads=2, head=64, causal=0)
        s.update(kw)
        fn = lib.nnvhip_differential_attention_backward_workspace if backward else lib.nnvhip_differential_attention_workspace
        _lib.check(fn(images._DIFFER.pack(*s.values(), 0.125, *[0] * 28), C.byref(n)))
        return n.value

    # one token against many keys is split, a large batch is not; D of both maps' rows in the backward pass
    assert differ(queries=1, keys=60000) > 0
    assert differ(batch=64, queries=4096, keys=4096, heads=32, kv_heads=32) == 0
    assert differ(backward=True) >= 4 * 2 * 2 * 4 * 100
    for kw in (dict(type=3), dict(weight_type=2), dict(head=0), dict(head=129), dict(heads=3), dict(kv_heads=0), dict(keys=-1), dict(queries=1 << 40),
               dict(batch=1 << 20), dict(heads=32768), dict(keys=1 << 31), dict(queries=1 << 31), dict(batch=65535, queries=1 << 20),
               dict(batch=65535, heads=32767, kv_heads=32767, queries=(1 << 31) - 256, keys=(1 << 31) - 256)):
        for backward in (False, True):
            with pytest.raises((ValueError, _lib.NNVHipError)):
                differ(backward, **kw)
    for kw in (dict(batch=64, heads=32, kv_heads=32, queries=32768, keys=4096), dict(batch=64, heads=64, kv_heads=8, queries=1, keys=65536), dict(heads=8, batch=1, queries=1, keys=1 << 26), dict(batch=1, queries=0), dict(keys=0)):
        for t in range(3):
            assert differ(type=t, weight_type=t, **kw) >= 0 and differ(True, type=t, weight_type=t, **kw) >= 0


@pytest.mark.parametrize("causal", [False, True])
def test_plain_differential_attention_is_differentiated_right(causal):
    torch.manual_seed(4)
    q, k, v, w = (torch.randn(*s, dtype=torch.float64, requires_grad=True) for s in ((2, 5, 8, 6), (2, 7, 4, 6), (2, 7, 2, 12), (4,)))
    kw = dict(key_mask=torch.rand(2, 7) < 0.8, key_lengths=torch.tensor([7, 3]), causal=causal)
    do = torch.randn(2, 5, 4, 12, dtype=torch.float64)
    o, lse, second = io.differ(q, k, v, w, **kw)
    o.backward(do)
    for got, t in zip(io.differ_grad(do, q.detach(), k.detach(), v.detach(), w.detach(), **kw), (q, k, v, w)):
        assert torch.allclose(got, t.grad, rtol=1e-10, atol=1e-12)
    # one row by hand: head 3, whose keys are the second key/value head's
    at = [j for j in range(7) if kw["key_mask"][0, j] and (not causal or j < 7 - 5 + 2 + 1)]
    p = [torch.softmax(torch.stack([(q[0, 2, 6 + m] * k[0, j, 2 + m]).sum() * 6 ** -0.5 for j in at]), 0) for m in (0, 1)]
    assert torch.allclose(o[0, 2, 3], (p[0] - w[3] * p[1]) @ v[0, at, 1]) and torch.allclose(second[0, 2, 3], p[1] @ v[0, at, 1])
    if causal:     # three keys for five queries: the first two see none
        assert (o[1, :2] == 0).all() and (lse[1, :, :2] == -math.inf).all()
