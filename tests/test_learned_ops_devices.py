"""Tensors of another device than the current one, and things that are no tensors, are
refused by the learned-choice and orthogonalisation operators.  CPU only."""
import numpy as np
import pytest

from tatara_amd import _lib, ops

FAKE = 4096  # an address that a refused call never reads


class Elsewhere:
    """Stands for a tensor on the second GPU."""

    is_cuda, device = True, "cuda:1"

    def __init__(self, *shape, dtype="float32"):
        self.shape, self.dtype = shape, np.dtype(dtype)

    def get_device(self):
        return 1

    def data_ptr(self):
        return FAKE

    def stride(self):
        return tuple(int(np.prod(self.shape[i + 1:])) for i in range(len(self.shape)))

    def is_contiguous(self):
        return True


def whole(*shape):
    return Elsewhere(*shape, dtype="int32")


E = Elsewhere
CALLS = {
    "norm": lambda: ops.LayerNorm(8).forward(E(3, 8), E(8), E(8), E(3, 8), E(3), E(3)),
    "norm_grad": lambda: ops.LayerNorm(8).backward(E(3, 8), E(3, 8), E(8), E(3), E(3), E(3, 8), E(8), E(8)),
    "gate": lambda: ops.BucketGate(9).forward(E(3, 9), whole(3, 1), E(3, 1), whole(9), E(9), whole(1), E(1)),
    "gate_grad": lambda: ops.BucketGate(9).backward(E(3, 9), whole(3, 1), whole(9), whole(1), E(3, 9), E(3, 1)),
    "orthogonalise": lambda: ops.Orthogonaliser(2, 3, 4)(E(2, 3, 4), E(2, 3, 4)),
    "muon": lambda: ops.Muon(2, 3, 4).step(E(2, 3, 4), E(2, 3, 4), E(2, 3, 4), 0.1),
}


@pytest.mark.parametrize("call", list(CALLS))
def test_another_device_is_refused(call):
    with pytest.raises(ValueError, match="on device 1"):
        CALLS[call]()


@pytest.mark.parametrize("x", [None, 3.0, np.float32(1), [1, 2]])
def test_no_tensors_are_refused(x):
    with pytest.raises(ValueError, match="x must"):
        ops.LayerNorm(8).forward(x, None, None, x)
    with pytest.raises(ValueError, match="dy must|x must"):
        ops.LayerNorm(8).backward(x, x, None, x, x, x)
    gate = ops.BucketGate(9)
    with pytest.raises(ValueError, match="logits must"):
        gate.forward(x, x, x, x, x, x, x)
    with pytest.raises(ValueError, match="logits must"):
        gate.backward(x, x, x, x, x)


def test_current_device():
    assert _lib.load().tatara_get_device(None) == -3
