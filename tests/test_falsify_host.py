"""The search for counterexamples (nnv_amd.falsify) on networks of a few torch operations on the host: what it hands back lies in
the box that it was given."""
import numpy as np
import pytest
import torch


class Linear:
    """scores = W times the sum over tokens of x, with the gradient that falsify_point follows."""

    def __init__(self, weights):
        self.weights = weights   # classes x channels

    def forward(self, x, states, key_lengths=None, key_mask=None):
        return x.sum(1) @ self.weights.t(), x.shape

    def backward(self, dscores, saved):
        return (dscores @ self.weights)[:, None, :].expand(saved), []


def box64(lb, ub, dtype, weights, g, **kw):
    import nnv_amd as nnv
    net = Linear(torch.tensor(weights, dtype=dtype))
    states = torch.zeros(1, 1, dtype=dtype)
    return nnv.falsify_point(net, np.asarray(lb), np.asarray(ub), states, nnv.HalfSpace(np.eye(len(weights)), np.asarray(g)), **kw)


@pytest.mark.parametrize("dtype,kept", [(torch.float32, np.float32), (torch.bfloat16, np.float32), (torch.float16, np.float16)],
                         ids=["f32", "bf16", "f16"])
def test_a_point_of_every_type_is_handed_back(dtype, kept):
    """numpy has no bf16: such a point comes as f32, which holds it."""
    found = box64([[0.0, 1.0]], [[1.0, 2.0]], dtype, [[1.0, 1.0]], [1e4], starts=1)
    assert found.dtype == kept and (found == np.array([[0.5, 1.5]])).all()
