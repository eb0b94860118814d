"""Which stream a learned-choice or orthogonalisation call goes to.  CPU only."""
import ctypes as C

import pytest

from tatara_amd import _lib, ops
from test_learned_ops_devices import Elsewhere


class TorchStream:
    def __init__(self, device, native):
        self.device_index, self.cuda_stream = device, native


class OwnStream:
    def __init__(self, handle):
        self.handle = handle


class Array:
    """Stands for the library's own array."""


def torch_is_there(monkeypatch, current_stream):
    monkeypatch.setattr(ops, "_torch_device", lambda: 0, raising=False)
    monkeypatch.setattr(ops, "_torch_stream", current_stream, raising=False)


def queue(x, stream):
    return ops._place(x, stream)[1]


@pytest.fixture
def side_stream(monkeypatch):
    """torch's current stream is one of its own."""
    torch_is_there(monkeypatch, lambda device: 0x1000 + device)


def test_torch_tensors_go_to_torchs_current_stream(side_stream):
    x = Elsewhere(3, 8)
    h = queue(x, None)
    assert h and h == queue(x, None)
    assert queue(Array(), None) is None  # the library's arrays: the null stream


def test_torchs_default_stream_is_the_null_stream(monkeypatch):
    torch_is_there(monkeypatch, lambda device: 0)
    assert queue(Elsewhere(3, 8), None) is None


def test_streams_that_are_given(side_stream):
    x = Elsewhere(3, 8)
    assert queue(x, TorchStream(0, 0x1000)) == queue(x, None)
    assert queue(Array(), TorchStream(0, 0x2000)) not in (None, queue(x, None))
    assert queue(x, OwnStream(77)) == 77


def test_a_closed_stream_is_refused():
    """It would stand for the null stream."""
    with pytest.raises(ValueError, match="closed"):
        queue(Array(), OwnStream(None))
    with pytest.raises(ValueError, match="closed"):
        queue(Elsewhere(3, 8), OwnStream(None))


def test_wrapped_streams():
    lib = _lib.load()
    assert lib.tatara_stream_wrap(0, None, None) == -3
    h = C.c_void_p()
    assert lib.tatara_stream_wrap(-1, None, C.byref(h)) == -3 and h.value is None
    assert lib.tatara_stream_wrap(0, 0x1000, C.byref(h)) == 0 and h.value
    assert lib.tatara_stream_destroy(h) == 0  # the stream itself is another library's
