"""Learned-choice and orthogonalisation calls on torch's streams: ordered with the work that
made their inputs, and recorded into a graph."""
import pytest
import torch

from tatara_amd import ops
from tatara_amd.runtime import Stream

pytestmark = pytest.mark.gpu


class Step:
    """One call of every operator, on inputs that are made on the GPU from one tensor."""

    def __init__(self):
        g = torch.Generator().manual_seed(0)
        self.norm, self.gate = ops.LayerNorm(96), ops.BucketGate(9, 2, renormalise=True)
        self.ortho, self.muon = ops.Orthogonaliser(2, 80, 96), ops.Muon(2, 16, 96)
        self.source = torch.randn(320, 96, generator=g).cuda()

    def buffers(self):
        def empty(*shape, dtype=torch.float32):
            return torch.full(shape, 7, dtype=dtype, device="cuda")

        b = dict(x=empty(320, 96), y=empty(320, 96), mean=empty(320), rstd=empty(320), dx=empty(320, 96), dw=empty(96),
                 db=empty(96), logits=empty(320, 9), bucket=empty(320, 2, dtype=torch.int32), share=empty(320, 2),
                 count=empty(9, dtype=torch.int32), prob=empty(9), counted=empty(1, dtype=torch.int32), loss=empty(1),
                 dlogits=empty(320, 9), out=empty(2, 80, 96), w=torch.zeros(2, 16, 96, device="cuda"),
                 m=torch.zeros(2, 16, 96, device="cuda"))
        torch.cuda.synchronize()
        return b

    def __call__(self, b, scale, stream=None):
        x = b["x"]
        x.copy_(self.source * scale)
        b["logits"].copy_(self.source[:, :9] * scale)
        if stream is not None:  # torch's work above is on torch's stream
            torch.cuda.current_stream().synchronize()
        self.norm.forward(x, None, None, b["y"], b["mean"], b["rstd"], stream=stream)
        self.norm.backward(b["y"], x, None, b["mean"], b["rstd"], b["dx"], b["dw"], b["db"], stream=stream)
        self.gate.forward(b["logits"], b["bucket"], b["share"], b["count"], b["prob"], b["counted"], b["loss"],
                          stream=stream)
        self.gate.backward(b["logits"], b["bucket"], b["count"], b["counted"], b["dlogits"], b["share"],
                           stream=stream)
        self.ortho(x.view(4, 80, 96)[:2], b["out"], stream=stream)
        self.muon.step(b["w"], b["m"], x[:32].view(2, 16, 96), 0.1, stream=stream)


def same(a, b):
    return [k for k in a if not torch.equal(a[k], b[k])] == []


@pytest.fixture(scope="module")
def step(gpu):
    return Step()


def test_torchs_current_stream(step):
    """Work that takes milliseconds stands ahead of the inputs on the stream."""
    want = step.buffers()
    step(want, 1.5)
    torch.cuda.synchronize()
    long = torch.zeros(1 << 28, device="cuda")
    side = torch.cuda.Stream()
    got = step.buffers()
    with torch.cuda.stream(side):
        for _ in range(20):
            long.add_(1.0)
        step(got, 1.5)
        side.synchronize()
    assert same(want, got)


def test_a_torch_stream_that_is_given(step):
    want, got = step.buffers(), step.buffers()
    step(want, 0.5)
    side = torch.cuda.Stream()
    step(got, 0.5, stream=side)
    side.synchronize()
    torch.cuda.synchronize()
    assert same(want, got)


def test_a_closed_stream_is_refused(step):
    s = Stream()
    s.close()
    x = step.source
    with pytest.raises(ValueError, match="closed"):
        step.norm.forward(x, None, None, torch.empty_like(x), stream=s)


def test_graph(step):
    """Every replay gives what the calls give, with other work between them."""
    warm = step.buffers()
    step(warm, 1.0)  # makes the workspaces
    torch.cuda.synchronize()
    b = step.buffers()
    scale = torch.ones(1, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(b, scale)
    b["w"].zero_()
    b["m"].zero_()
    want = step.buffers()
    for k in range(4):
        scale.fill_(1.0 + k)
        graph.replay()
        torch.cuda.synchronize()
        step(want, 1.0 + k)
        torch.cuda.synchronize()
        assert same(want, b), k
