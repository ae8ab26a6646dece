"""The operators on points as far as they go without a GPU: their workspaces, their refusals, and their plain forms in 64 bits
(tests/points_oracle.py) against torch's own differentiation."""
import ctypes as C
import math
import os

import pytest
import torch

from tests import points_oracle as po

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nnv_amd", "libnnvhip.so")
built = pytest.mark.skipif(not os.path.exists(LIB), reason="library not built (python -m nnv_amd.build)")


def test_tensors_on_the_host_are_refused():
    import nnv_amd as nnv
    x = torch.zeros(2, 3, 4, 8)
    for call in (lambda: nnv.layer_norm(x), lambda: nnv.cross_attention(x, x, x), lambda: nnv.clip_gradients([x], 1.0)):
        with pytest.raises(ValueError, match="on the GPU"):
            call()
    with pytest.raises(TypeError):
        nnv.layer_norm(3.0)
    with pytest.raises(AttributeError):
        nnv.no_such_operator
    assert "layer_norm" in dir(nnv)


@built
def test_workspaces_and_their_refusals():
    from nnv_amd import _lib, points
    lib, n = _lib.load(), C.c_int64()

    def attention(backward=False, **kw):
        s = dict(type=1, batch=2, queries=100, keys=200, heads=4, kv_heads=2, head=64)
        s.update(kw)
        d = points._ATTENTION.pack(*s.values(), 0.125, *[0] * 25)
        fn = lib.nnvhip_cross_attention_backward_workspace if backward else lib.nnvhip_cross_attention_workspace
        _lib.check(fn(d, C.byref(n)))
        return n.value

    # one token against many keys is split, a large batch is not; D of every row in the backward pass
    assert attention(queries=1, keys=60000) > 0
    assert attention(batch=64, queries=4096, keys=4096, heads=32, kv_heads=32) == 0
    assert attention(backward=True) >= 4 * 2 * 4 * 100
    for kw in (dict(type=3), dict(head=0), dict(head=129), dict(heads=3), dict(kv_heads=0), dict(keys=-1), dict(queries=1 << 40), dict(batch=1 << 20)):
        with pytest.raises((ValueError, _lib.NNVHipError)):
            attention(**kw)
    _lib.check(lib.nnvhip_layer_norm_backward_workspace(0, 3, 64, C.byref(n)))
    assert n.value == 0                                    # one block: no partial sums
    _lib.check(lib.nnvhip_layer_norm_backward_workspace(0, 100000, 64, C.byref(n)))
    assert 0 < n.value <= 512 * 2 * 64 * 4
    for args in ((5, 3, 64), (0, -1, 64), (0, 3, 0), (0, 1 << 32, 64)):
        with pytest.raises((ValueError, _lib.NNVHipError)):
            _lib.check(lib.nnvhip_layer_norm_backward_workspace(*args, C.byref(n)))
    with pytest.raises(ValueError):
        _lib.check(lib.nnvhip_clip_gradients_workspace(-1, C.byref(n)))


def test_plain_norm_is_differentiated_right():
    torch.manual_seed(1)
    x, w, b = (torch.randn(*s, dtype=torch.float64, requires_grad=True) for s in ((5, 33), (33,), (33,)))
    dy = torch.randn(5, 33, dtype=torch.float64)
    y, mean, rstd = po.norm(x, w, b, 1e-5)
    y.backward(dy)
    for got, t in zip(po.norm_grad(dy, x.detach(), mean.detach(), rstd.detach(), w.detach()), (x, w, b)):
        assert torch.allclose(got, t.grad, rtol=1e-12, atol=1e-12)
    assert torch.allclose(y, torch.nn.functional.layer_norm(x, (33,), w, b, 1e-5), rtol=1e-12, atol=1e-12)


def test_plain_attention_is_differentiated_right():
    torch.manual_seed(2)
    q, k, v = (torch.randn(*s, dtype=torch.float64, requires_grad=True) for s in ((2, 5, 4, 8), (2, 7, 2, 8), (2, 7, 2, 8)))
    mask = torch.rand(2, 7) < 0.7
    mask[:, 0] = True
    do = torch.randn(2, 5, 4, 8, dtype=torch.float64)
    o, lse = po.attend(q, k, v, key_mask=mask)
    o.backward(do)
    for got, t in zip(po.attend_grad(do, q.detach(), k.detach(), v.detach(), key_mask=mask), (q, k, v)):
        assert torch.allclose(got, t.grad, rtol=1e-10, atol=1e-12)
    # one row by hand
    s = torch.stack([(q[1, 2, 3] * k[1, j, 1]).sum() * 8 ** -0.5 for j in range(7)])[mask[1]]
    assert torch.allclose(lse[1, 3, 2], torch.logsumexp(s, 0)) and torch.allclose(o[1, 2, 3], torch.softmax(s, 0) @ v[1, mask[1], 1])
    o, lse = po.attend(q, k, v, key_lengths=torch.tensor([0, 7]))
    assert (o[0] == 0).all() and (lse[0] == -math.inf).all()
    assert all((g[0] == 0).all() for g in po.attend_grad(do, q, k, v, key_lengths=torch.tensor([0, 7])))


def test_plain_clip():
    got, n = po.clip([torch.tensor([3.0]), torch.tensor([[4.0]])], 2.5)
    assert n == 5.0 and float(got[0]) == 1.5 and float(got[1]) == 2.0
