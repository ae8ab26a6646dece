"""How the operators on points choose the GPU they work on, without one: the context of the tensors' GPU."""
import pytest


class Tensor:
    requires_grad = False

    def __init__(self, index):
        self.index = index

    def get_device(self):
        return self.index


@pytest.fixture
def contexts(monkeypatch):
    """Contexts without a GPU, and none made so far; the list of those made."""
    from nnv_amd import _lib, points
    made = []

    class Context:
        lib, handle = "library", "handle"

        def __init__(self, device=0):
            self.device = device
            made.append(device)

    monkeypatch.setattr(_lib, "Context", Context)
    monkeypatch.setattr(_lib, "_default_ctx", None)
    monkeypatch.setattr(_lib, "_other_ctx", {}, raising=False)
    monkeypatch.delenv("NNVHIP_DEVICE", raising=False)
    monkeypatch.setattr(points, "_stream_of", lambda index: 100 + index)
    return made


def test_tensors_of_any_gpu_find_its_context(contexts, monkeypatch):
    from nnv_amd import _lib, points
    one = points._enter("call", None, Tensor(1), None, Tensor(1))
    assert (one[0].device, one[2]) == (1, 101) and contexts == [1]      # GPU 0 is left alone
    assert points._enter("call", None, Tensor(1))[0] is one[0]
    zero = points._enter("call", None, Tensor(0))[0]
    assert zero is _lib.default_context() and points._enter("call", None, Tensor(0))[0] is zero and contexts == [1, 0]
    assert points._enter("call", one[0], Tensor(1))[0] is one[0]
    with pytest.raises(ValueError, match="the context is GPU 1's"):
        points._enter("call", one[0], Tensor(0))
    with pytest.raises(ValueError, match="on one GPU"):
        points._enter("call", None, Tensor(0), Tensor(1))
    with pytest.raises(ValueError, match="on the GPU"):
        points._enter("call", None, Tensor(-1))


def test_the_default_contexts_gpu_is_the_environments(contexts, monkeypatch):
    from nnv_amd import _lib, points
    monkeypatch.setenv("NNVHIP_DEVICE", "2")
    assert points._enter("call", None, Tensor(2))[0] is _lib.default_context() and contexts == [2]
    assert points._enter("call", None, Tensor(0))[0].device == 0


def test_gradients_that_nobody_records_are_not_lost_silently(contexts):
    from nnv_amd import points
    torch = pytest.importorskip("torch")

    class Learnt(Tensor):
        requires_grad = True

    with pytest.raises(ValueError, match="no_grad"):
        points._enter("call", None, Tensor(0), None, Learnt(0))
    with torch.no_grad():
        assert points._enter("call", None, Tensor(0), None, Learnt(0))[0].device == 0
    assert points._enter("call", None, Tensor(0), None, Tensor(0))[0].device == 0
