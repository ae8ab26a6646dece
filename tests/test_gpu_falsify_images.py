"""The network for images and videos of nnv_amd.falsify: group normalization, positions, differential attention and their gradients together, against
torch's own differentiation in 64 bits on the host; the search and the training step on it."""
import numpy as np
import pytest
import torch

from tests import images_oracle as io

pytestmark = pytest.mark.gpu

GRID, STATES, GROUPS, HEADS, KV, SECTIONS = (2, 3, 5), (2, 4, 7), 4, 4, 2, (2, 4, 6)


def differentiable_rotation(x, positions, sections):
    total = sum(sections)
    angles = torch.cat([positions[:, a, None].double() * 10000.0 ** -(torch.arange(n, dtype=torch.float64) / n) for a, n in enumerate(sections)], 1)
    c, s = torch.cos(angles)[None, :, None], torch.sin(angles)[None, :, None]
    u, w = x[..., :total], x[..., total:2 * total]
    return torch.cat([u * c - w * s, u * s + w * c, x[..., 2 * total:]], -1)


def plain_scores(p, x, states, mask, positions, state_positions):
    """The network's definition, on the host in 64 bits."""
    y = io.group(x, GROUPS, p["Scale"], p["Offset"], 1e-5, "silu")[0]
    q, k, v = ((t).unflatten(2, (h, -1)) for t, h in ((y @ p["Wq"], 2 * HEADS), (states @ p["Wk"], 2 * KV), (states @ p["Wv"], KV)))
    q, k = differentiable_rotation(q, positions, SECTIONS), differentiable_rotation(k, state_positions, SECTIONS)
    o = io.differ(q, k, v, p["Weights"], key_mask=mask)[0].flatten(2)
    return (x + o @ p["Wo"]).mean(1) @ p["Wc"] + p["bc"]


def case(seed=0, dtype=torch.float32):
    import nnv_amd as nnv
    net = nnv.GridAttentionClassifier.random(40, 24, 5, GRID, STATES, GROUPS, HEADS, SECTIONS, KV, head=32, seed=seed, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    x, states = torch.randn(6, 30, 40, generator=g, device="cuda"), torch.randn(6, 56, 24, generator=g, device="cuda")
    return net, x.to(dtype), states.to(dtype), torch.rand(6, 56, generator=g, device="cuda") < 0.7


def test_network_and_its_gradients():
    net, x, states, mask = case()
    scores, saved = net.forward(x, states, key_mask=mask)
    assert torch.equal(net.evaluate(x, states, key_mask=mask), scores)
    w = torch.randn(scores.shape, device="cuda")
    dx, grads = net.backward(w, saved)
    p = {n: t.double().cpu().requires_grad_() for n, t in net.parameters.items()}
    x64 = x.double().cpu().requires_grad_()
    exact = plain_scores(p, x64, states.double().cpu(), mask.cpu(), net.positions.cpu(), net.state_positions.cpu())
    (exact * w.double().cpu()).sum().backward()
    # products and sums of at most a few hundred f32 terms one behind the other: some 1e3 roundings of 2^-24, of the tensor's scale
    for name, got, e in [("scores", scores, exact.detach()), ("dx", dx, x64.grad)] + [(n, t, p[n].grad) for n, t in zip(net.PARAMETERS, grads)]:
        assert got.shape == e.shape, name
        assert (got.double().cpu() - e).abs().max() <= 1e3 * 2.0 ** -24 * e.abs().max().clamp_min(1e-3), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
def test_search_and_training_step_run(dtype):
    import nnv_amd as nnv
    net, x, states, mask = case(3, dtype)
    centre = x[0].double().cpu().numpy()
    scores = net.evaluate(x[:1], states[:1]).float().cpu().numpy()[0]
    # unsafe: the smallest score's class is the largest's peer; and everything
    order = scores.argsort()
    G = np.zeros((1, 5))
    G[0, order[-1]], G[0, order[-2]] = 1.0, -1.0
    found = nnv.falsify_point(net, centre - 0.5, centre + 0.5, states[0], nnv.HalfSpace(G, [0.0]), steps=3)
    assert found is None or (found >= centre - 0.5).all() and (found <= centre + 0.5).all()
    anything = nnv.falsify_point(net, centre - 0.5, centre + 0.5, states[0], nnv.HalfSpace(G, [1e4]), steps=0)
    assert anything is not None and anything.shape == centre.shape
    labels = torch.tensor([0, 1, 2, 3, 4, 0], device="cuda")
    before = {n: t.clone() for n, t in net.parameters.items()}
    loss, norm = nnv.train_step(net, x, states, labels, rate=0.1, threshold=1.0, key_mask=mask)
    assert bool(torch.isfinite(loss)) and bool(torch.isfinite(norm))
    # a step has a norm of 0.1 at most; one below half a place of a 16-bit parameter (2^-9 of a scale of one) leaves it as it is
    steps = {n: (t - before[n]).float().norm() for n, t in net.parameters.items()}
    assert any(float(s) > 0 for s in steps.values()) and (dtype != torch.float32 or all(float(s) > 0 for s in steps.values()))
    assert all(float(s) <= 0.1 + float((torch.finfo(dtype).eps / 2 * before[n].float()).norm() + (torch.finfo(dtype).eps * 0.1)) for n, s in steps.items())


def test_layers_and_their_refusals():
    import nnv_amd as nnv
    net, x, states, _ = case(4)
    with pytest.raises(ValueError, match="parameters missing"):
        nnv.GridAttentionClassifier(GRID, STATES, GROUPS, HEADS, SECTIONS)
    with pytest.raises(ValueError, match="same axes"):
        nnv.GridAttentionClassifier(GRID, STATES[:2], GROUPS, HEADS, SECTIONS, KV, **net.parameters)
    with pytest.raises(ValueError, match="number of channels"):
        net.norm.evaluate(x[..., :20])
    with pytest.raises(ValueError, match="need positions"):
        net.attend.evaluate(x @ net.parameters["Wq"], states @ net.parameters["Wk"], states @ net.parameters["Wv"])
    with pytest.raises(ValueError, match="multiple of the number of heads"):
        net.attend.evaluate(x[..., :39], states, states, net.positions, net.state_positions)
    # causal self-attention whose queries and keys have one grid, without positions and with them
    w = torch.full((2,), 0.4, device="cuda")
    q, k, v = (torch.randn(3, 30, n, device="cuda") for n in (4 * 16, 4 * 16, 2 * 32))
    for sections, at in ((None, None), (SECTIONS[:1] + (3, 3), net.positions)):
        layer = nnv.DifferentialAttentionLayer(2, w, Causal=True, Sections=sections)
        o, saved = layer.forward(q, k, v, at, at)
        grads = layer.backward(torch.ones_like(o), saved)
        assert [t.shape for t in grads] == [q.shape, k.shape, v.shape, w.shape]
        split = [t.unflatten(2, (n, -1)) for t, n in ((q, 4), (k, 4), (v, 2))]
        if at is not None:
            split[:2] = [io.rotate(t, at, sections) for t in split[:2]]
        e = io.differ(*[t.double() for t in split], w, causal=True)[0].flatten(2)
        assert (o - e).abs().max() <= 1e3 * 2.0 ** -24 * e.abs().max()
