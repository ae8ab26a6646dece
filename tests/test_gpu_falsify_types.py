"""The search for counterexamples in 16 bits on the GPU, in a box whose bounds have 64: what it finds lies in the box and in the HalfSpace."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
def test_a_counterexample_of_every_type(dtype):
    import nnv_amd as nnv
    net = nnv.CrossAttentionClassifier.random(48, 32, 5, NumHeads=4, NumKeyValueHeads=2, head=24, seed=3, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(4)
    x, states = torch.randn(9, 48, generator=g, device="cuda", dtype=torch.float64), torch.randn(70, 32, generator=g, device="cuda").to(dtype)
    scores = net.evaluate(x[None].to(dtype), states[None])[0].float()
    label, other = (int(i) for i in scores.topk(2).indices)
    G = np.zeros((1, 5))
    G[0, label], G[0, other] = 1.0, -1.0              # unsafe: the other class scores at least as high
    unsafe, lb, ub = nnv.HalfSpace(G, [0.0]), (x - 1.0).cpu().numpy(), (x + 1.0).cpu().numpy()
    lengths = torch.tensor([61], device="cuda")
    for kw in ({}, dict(key_lengths=lengths), dict(key_mask=(torch.arange(70, device="cuda") % 9 != 4)[None])):
        found = nnv.falsify_point(net, lb, ub, states, unsafe, **kw)
        assert found is not None
        point = np.asarray(found, dtype=np.float64)
        assert (point >= lb).all() and (point <= ub).all()
        # (alone and among the starts, a product may be summed in another order: a place of the scores' type)
        again = net.evaluate(torch.as_tensor(found, device="cuda").to(dtype)[None], states[None], **kw)[0].double().cpu().numpy()
        slack = float(torch.finfo(dtype).eps) * 8 * np.abs(again).max()
        assert again[label] - again[other] <= slack
