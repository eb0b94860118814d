"""Without a stream a call goes where its first tensor's stream says, whatever the others
are.  CPU only."""
import pytest

from tatara_amd import ops

CALLS = {
    "layer norm": lambda t: ops.LayerNorm(8).forward(t, *[None] * 3),
    "layer norm backward": lambda t: ops.LayerNorm(8).backward(t, *[None] * 5),
    "gate": lambda t: ops.BucketGate(9).forward(t, *[None] * 6),
    "gate backward": lambda t: ops.BucketGate(9).backward(t, *[None] * 4),
    "orthogonaliser": lambda t: ops.Orthogonaliser(1, 4, 4)(t, None),
    "muon": lambda t: ops.Muon(1, 4, 4).step(t, None, None, 0.1),
    "RMS norm": lambda t: ops.RMSNorm(8).forward(t, None, None),
    "RMS norm in 8 bits": lambda t: ops.RMSNorm(8).forward_8bit(t, None, None, None),
    "RMS norm backward": lambda t: ops.RMSNorm(8).backward(t, *[None] * 4),
    "dropout": lambda t: ops.Dropout(8, 0.1).forward(t, None),
    "dropout backward": lambda t: ops.Dropout(8, 0.1).backward(t, None),
    "sort": lambda t: ops.BucketRows(9, 8).sort(t, *[None] * 3),
    "gather": lambda t: ops.BucketRows(9, 8).gather(t, *[None] * 3),
    "gather backward": lambda t: ops.BucketRows(9, 8).gather_backward(t, None, None),
    "combine": lambda t: ops.BucketRows(9, 8).combine(t, *[None] * 3),
    "combine backward": lambda t: ops.BucketRows(9, 8).combine_backward(t, *[None] * 5),
    "embedding": lambda t: ops.Embedding(9, 8, 4).forward(t, None, None),
    "embedding backward": lambda t: ops.Embedding(9, 8, 4).backward(t, None, None),
}


class Asked(Exception):
    pass


@pytest.mark.parametrize("name", list(CALLS))
def test_the_stream_is_the_first_tensors(name, monkeypatch):
    def place(x, stream):
        raise Asked(x)

    monkeypatch.setattr(ops, "_place", place)
    first = object()
    with pytest.raises(Asked) as asked:
        CALLS[name](first)
    assert asked.value.args[0] is first
