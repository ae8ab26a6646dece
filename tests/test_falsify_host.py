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
        return (dscores @ self.weights)[:, None, :].expand(saved), [dscores.sum(0)]


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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_a_point_on_the_boxs_border_is_inside(dtype, sign):
    """Bounds in 64 bits that the states' type does not hold: the search ends on a border, and that has to be on this side of it."""
    at = np.array([[0.1, 0.3, 1 / 3, 0.7, 1.1, 2.3]])
    lb, ub = (at - 1.0, at) if sign > 0 else (-at, 1.0 - at)
    # only within a hundredth of the largest sums of x: what the steps reach on the border alone
    limit = -sign * float((ub if sign > 0 else lb).sum())
    found = box64(lb, ub, dtype, [[-sign] * 6], [limit + 0.1], steps=40)
    assert found is not None
    point = np.asarray(found, dtype=np.float64)
    assert (point >= lb).all() and (point <= ub).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
def test_the_first_points_are_inside(dtype):
    """Every point is a counterexample, so that the starts themselves are handed back: one of each seed."""
    r = np.random.default_rng(1)
    for seed in range(40):
        lb = r.normal(size=(1, 300))
        ub = lb + np.maximum(10.0 ** r.uniform(-3, 0), abs(lb) / 64)   # wider than two of bf16's numbers are apart
        for starts in (1, 2):
            found = box64(lb, ub, dtype, [[1.0] + [0.0] * 299], [1e4], starts=starts, steps=0, seed=seed)
            assert found is not None
            point = np.asarray(found, dtype=np.float64)
            assert (point >= lb).all() and (point <= ub).all()


def test_a_box_without_a_point_of_the_type():
    assert box64([[0.1]], [[0.1]], torch.float32, [[1.0]], [1e4]) is None
    assert box64([[0.125]], [[0.125]], torch.float32, [[1.0]], [1e4]) == 0.125


def test_boxes_that_are_none():
    for lb, ub in (([[0.2]], [[0.1]]), ([[np.nan]], [[0.1]]), ([[-np.inf]], [[0.1]]), ([0.1], [0.2])):
        with pytest.raises(ValueError, match="bounds of a box"):
            box64(lb, ub, torch.float32, [[1.0]], [1e4])


def test_a_start_without_scores_hides_no_other():
    """A network that gives NaN for some points: the others are still looked at, and moved."""

    class Broken(Linear):
        def forward(self, x, states, key_lengths=None, key_mask=None):
            scores, saved = super().forward(x, states)
            return torch.where(torch.arange(len(x))[:, None] == 1, torch.nan, scores), saved

    import nnv_amd as nnv
    states = torch.zeros(1, 1)
    for limit in (1e4, -0.4):   # met by the first points, and by steps to the lower border
        found = nnv.falsify_point(Broken(torch.ones(1, 2)), np.zeros((1, 2)) - 0.25, np.ones((1, 2)), states, nnv.HalfSpace([[1.0]], [limit]))
        assert found is not None and found.sum() <= limit


def test_searches_and_training_steps_record_no_gradients():
    """They follow gradients of their own: weights that require one are no obstacle, and train_step may write to them."""
    import nnv_amd as nnv

    class Asked(Linear):
        def forward(self, *args, **kw):
            assert not torch.is_grad_enabled()
            return super().forward(*args, **kw)

    net = Asked(torch.ones(1, 2, requires_grad=True))
    assert nnv.falsify_point(net, np.zeros((1, 2)), np.ones((1, 2)), torch.zeros(1, 1), nnv.HalfSpace([[1.0]], [0.5])) is not None
    with pytest.raises(ValueError, match="on the GPU"):      # as far as a step goes on the host: to the clipping
        nnv.train_step(net, torch.ones(2, 1, 2), None, torch.tensor([0, 0]), 0.1, 1.0)
