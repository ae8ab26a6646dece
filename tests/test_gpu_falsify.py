"""The search for counterexamples and the training step of nnv_amd.falsify: its network against torch's own differentiation in 64 bits
on the host, a counterexample that is one, and a loss that falls."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def plain_scores(p, x, states, mask, heads, kv_heads):
    """The network's definition, on the host in 64 bits."""
    mean, c = x.mean(-1, keepdim=True), x - x.mean(-1, keepdim=True)
    y = c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-5) * p["Scale"] + p["Offset"]
    q, k, v = (t.unflatten(2, (h, -1)).transpose(1, 2) for t, h in ((y @ p["Wq"], heads), (states @ p["Wk"], kv_heads), (states @ p["Wv"], kv_heads)))
    k, v = (t.repeat_interleave(heads // kv_heads, dim=1) for t in (k, v))
    s = (q @ k.transpose(2, 3)) * q.shape[-1] ** -0.5
    o = torch.softmax(s.masked_fill(~mask[:, None, None, :], -torch.inf), -1) @ v
    return (x + o.transpose(1, 2).flatten(2) @ p["Wo"]).mean(1) @ p["Wc"] + p["bc"]


def case(seed=0):
    import nnv_amd as nnv
    net = nnv.CrossAttentionClassifier.random(48, 32, 5, NumHeads=4, NumKeyValueHeads=2, head=24, seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    x, states = torch.randn(6, 9, 48, generator=g, device="cuda"), torch.randn(6, 70, 32, generator=g, device="cuda")
    mask = torch.rand(6, 70, generator=g, device="cuda") < 0.7
    return net, x, states, mask


def test_network_and_its_gradients():
    net, x, states, mask = case()
    scores, saved = net.forward(x, states, key_mask=mask)
    w = torch.randn(scores.shape, device="cuda")
    dx, grads = net.backward(w, saved)
    p = {n: t.double().cpu().requires_grad_() for n, t in net.parameters.items()}
    x64 = x.double().cpu().requires_grad_()
    exact = plain_scores(p, x64, states.double().cpu(), mask.cpu(), 4, 2)
    (exact * w.double().cpu()).sum().backward()
    # six products and sums of at most a few hundred f32 terms one behind the other: some 1e3 roundings of 2^-24, of the tensor's scale
    for name, got, e in [("scores", scores, exact.detach()), ("dx", dx, x64.grad)] + [(n, t, p[n].grad) for n, t in zip(net.PARAMETERS, grads)]:
        assert got.shape == e.shape, name
        assert (got.double().cpu() - e).abs().max() <= 1e3 * 2.0 ** -24 * e.abs().max().clamp_min(1e-3), name


def test_a_counterexample_is_one():
    import nnv_amd as nnv
    net, x, states, mask = case(3)
    centre, label = x[0], int(net.evaluate(x[:1], states[:1])[0].argmax())
    other = int(net.evaluate(x[:1], states[:1])[0].topk(2).indices[1])
    G = np.zeros((1, 5))
    G[0, label], G[0, other] = 1.0, -1.0              # unsafe: the other class scores at least as high
    unsafe = nnv.HalfSpace(G, [0.0])
    found = nnv.falsify_point(net, centre - 1.0, centre + 1.0, states[0], unsafe)
    assert found is not None
    point = torch.as_tensor(found, device="cuda")
    assert bool((point >= centre - 1.0).all()) and bool((point <= centre + 1.0).all())
    assert unsafe.contains(net.evaluate(point[None], states[:1])[0].double().cpu().numpy())
    # a box of one point is that point, and it is safe
    assert nnv.falsify_point(net, centre, centre, states[0], unsafe, starts=2, steps=2) is None
    with pytest.raises(TypeError, match="HalfSpace"):
        nnv.falsify_point(net, centre, centre, states[0], None)
    with pytest.raises(ValueError, match="bounds of a box"):
        nnv.falsify_point(net, centre + 1, centre, states[0], unsafe)
    with pytest.raises(ValueError, match="parameters missing"):
        nnv.CrossAttentionClassifier(4)


def test_training_on_points_lowers_their_loss():
    import nnv_amd as nnv
    net, x, states, mask = case(5)
    labels = torch.tensor([0, 1, 2, 3, 4, 0], device="cuda")
    losses = [float(nnv.train_step(net, x, states, labels, rate=0.3, threshold=1.0, key_mask=mask)[0]) for _ in range(30)]
    assert losses[-1] < 0.5 * losses[0]
    _, norm = nnv.train_step(net, x, states, labels, rate=0.0, threshold=1e-3, key_mask=mask)
    assert float(norm) > 1e-3
