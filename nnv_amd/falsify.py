"""Search for counterexamples along gradients, and training on the ones found: how the operators of ``nnv_amd.points`` work
together on a network that the set layers do not cover.

A verifier looks for a counterexample before it reaches (the reference's NN evaluates samples of the input box, nn/NN.m); where a
gradient is to be had, the search follows it.  ``CrossAttentionClassifier`` is a small network for that: points are sequences of
tokens that attend to the states of another sequence.  ``falsify_point`` moves points of a box towards a HalfSpace of unsafe outputs
and returns one whose output lies in it, checked against the HalfSpace itself; ``train_step`` is one step of gradient descent on
the cross entropy of labelled points, e.g. of counterexamples, with the norm of all gradients bounded.
"""
from __future__ import annotations

import numpy as np
import torch

from .points import CrossAttentionLayer, LayerNormalizationLayer, clip_gradients
from .verify import HalfSpace


class CrossAttentionClassifier:
    """scores = mean over tokens of (x + attention(norm(x) Wq; states Wk, states Wv) Wo) Wc + bc.

    x: batch x tokens x channels; states: batch x keys x (their channels), with key_lengths or a key_mask where they are padded."""

    PARAMETERS = ("Scale", "Offset", "Wq", "Wk", "Wv", "Wo", "Wc", "bc")

    def __init__(self, NumHeads, NumKeyValueHeads=None, **parameters):
        missing = [n for n in self.PARAMETERS if n not in parameters]
        if missing:
            raise ValueError("parameters missing: " + ", ".join(missing))
        self.parameters = {n: parameters[n] for n in self.PARAMETERS}
        self.norm = LayerNormalizationLayer(Scale=parameters["Scale"], Offset=parameters["Offset"])
        self.attend = CrossAttentionLayer(NumHeads, NumKeyValueHeads)

    @staticmethod
    def random(channels, state_channels, classes, NumHeads, NumKeyValueHeads=None, head=64, seed=0, dtype=torch.float32, device="cuda"):
        """A network with random weights, for examples and tests."""
        g = torch.Generator().manual_seed(seed)
        kv = NumKeyValueHeads or NumHeads

        def w(n_in, n_out):
            return (torch.randn(n_in, n_out, generator=g) / n_in ** 0.5).to(dtype).to(device)

        return CrossAttentionClassifier(NumHeads, NumKeyValueHeads, Scale=torch.ones(channels, dtype=dtype, device=device),
                                        Offset=torch.zeros(channels, dtype=dtype, device=device), Wq=w(channels, NumHeads * head),
                                        Wk=w(state_channels, kv * head), Wv=w(state_channels, kv * head), Wo=w(NumHeads * head, channels),
                                        Wc=w(channels, classes), bc=torch.zeros(classes, dtype=dtype, device=device))

    def evaluate(self, x, states, key_lengths=None, key_mask=None):
        return self.forward(x, states, key_lengths, key_mask)[0]

    def forward(self, x, states, key_lengths=None, key_mask=None):
        """(scores: batch x classes, what backward takes)."""
        p = self.parameters
        y, norm = self.norm.forward(x)
        o, attend = self.attend.forward(y @ p["Wq"], states @ p["Wk"], states @ p["Wv"], key_lengths, key_mask)
        pooled = (x + o @ p["Wo"]).mean(1)
        return pooled @ p["Wc"] + p["bc"], (x, states, y, norm, o, attend, pooled)

    def backward(self, dscores, saved):
        """(dx, gradients of the parameters in the order of PARAMETERS)."""
        p = self.parameters
        x, states, y, norm, o, attend, pooled = saved

        def by_weights(inputs, gradient):      # sum over batch and tokens
            return inputs.flatten(0, -2).t() @ gradient.flatten(0, -2)

        dz = ((dscores @ p["Wc"].t()) / x.shape[1])[:, None, :].expand(x.shape).contiguous()
        dq, dk, dv = self.attend.backward(dz @ p["Wo"].t(), attend)
        dx, (dscale, doffset) = self.norm.backward(dq @ p["Wq"].t(), norm)
        return dz + dx, [dscale, doffset, by_weights(y, dq), by_weights(states, dk), by_weights(states, dv), by_weights(o, dz),
                         pooled.t() @ dscores, dscores.sum(0)]


def _bounds_within(lb, ub, like):
    """(lb, ub) in like's type and on its device, rounded towards the inside of the box that they are given as; None where none of
    the type's numbers lies between them."""
    lb, ub = (torch.as_tensor(t, dtype=torch.float64, device="cpu") for t in (lb, ub))
    if lb.shape != ub.shape or lb.dim() != 2 or not bool((lb <= ub).all()) or not bool((lb.isfinite() & ub.isfinite()).all()):
        raise ValueError("lb and ub are the bounds of a box of tokens x channels")
    low, high = lb.to(like.dtype), ub.to(like.dtype)
    low = torch.where(low.double() < lb, torch.nextafter(low, torch.full_like(low, torch.inf)), low)
    high = torch.where(high.double() > ub, torch.nextafter(high, torch.full_like(high, -torch.inf)), high)
    return (low.to(like.device), high.to(like.device)) if bool((low <= high).all()) else None


@torch.no_grad()
def falsify_point(network, lb, ub, states, unsafe, starts=8, steps=50, step=0.1, seed=0, key_lengths=None, key_mask=None):
    """A point of the box [lb, ub] (tokens x channels) whose scores lie in the HalfSpace `unsafe` (G y <= g), as a host array of the
    states' type (f32 for bf16); None if none was found, which says nothing about there being none.

    `starts` points drawn from the box (the first is its centre) descend on the largest row of G y - g, each coordinate by `step` times the
    box's width against the sign of its gradient, and stay in the box, whose bounds may be finer than the states' type.  states: keys x
    channels."""
    if not isinstance(unsafe, HalfSpace):
        raise TypeError("unsafe must be a HalfSpace")
    bounds = _bounds_within(lb, ub, states)
    if bounds is None:
        return None
    lb, ub = bounds
    G = torch.as_tensor(np.asarray(unsafe.G), dtype=states.dtype, device=states.device)
    g = torch.as_tensor(np.asarray(unsafe.g).reshape(-1), dtype=states.dtype, device=states.device)
    r = torch.Generator(device=states.device).manual_seed(seed)
    x = lb + (ub - lb) * torch.rand((starts,) + lb.shape, generator=r, device=states.device, dtype=states.dtype)
    x[0] = lb / 2 + ub / 2
    x = torch.minimum(torch.maximum(x, lb), ub)   # (sums are rounded)
    kept = states.expand((starts,) + states.shape).contiguous()   # (one matrix of all tokens for the products with the weights)
    spread = None if key_lengths is None else key_lengths.expand(starts).contiguous()
    mask = None if key_mask is None else key_mask.expand(starts, -1)
    for k in range(steps + 1):
        scores, saved = network.forward(x, kept, spread, mask)
        margins = scores @ G.t() - g
        worst, row = margins.max(1)
        best = int(worst.nan_to_num(torch.inf, torch.inf, -torch.inf).argmin())   # (a start without scores is not the best one)
        if float(worst[best]) <= 0 and unsafe.contains(scores[best].double().cpu().numpy()):
            point = x[best].cpu()
            return (point.float() if point.dtype == torch.bfloat16 else point).numpy()
        if k == steps:
            return None
        dx, _ = network.backward(G[row].contiguous(), saved)
        x = torch.minimum(torch.maximum(x - step * (ub - lb) * dx.sign(), lb), ub)


@torch.no_grad()
def train_step(network, x, states, labels, rate, threshold, key_lengths=None, key_mask=None):
    """One step of gradient descent on the cross entropy, the norm of all gradients bounded to `threshold`.  The network's parameters
    are updated in place; returns (loss, norm) as they were before the step, both left on the GPU."""
    scores, saved = network.forward(x, states, key_lengths, key_mask)
    logs = torch.log_softmax(scores.float(), 1)
    picked = torch.nn.functional.one_hot(labels, scores.shape[1]).to(logs.dtype)
    loss = -(logs * picked).sum(1).mean()
    _, gradients = network.backward(((logs.exp() - picked) / len(labels)).to(scores.dtype), saved)
    gradients, norm = clip_gradients(gradients, threshold, out=gradients)
    for name, gradient in zip(network.PARAMETERS, gradients):
        network.parameters[name].sub_(gradient, alpha=rate)
    return loss, norm
