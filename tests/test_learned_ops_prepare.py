"""An operator's workspace, made ahead of its first call."""
import pytest

from tatara_amd import ops

MAKE = {"norm": lambda: ops.LayerNorm(64), "gate": lambda: ops.BucketGate(9),
        "orthogonalise": lambda: ops.Orthogonaliser(1, 80, 96), "muon": lambda: ops.Muon(1, 80, 96)}


@pytest.mark.parametrize("name", list(MAKE))
def test_prepare_makes_one_workspace_a_device(name, monkeypatch):
    made, device = [], [0]
    monkeypatch.setattr(ops, "_Workspace", lambda nbytes: made.append((device[0], nbytes)) or object())
    monkeypatch.setattr(ops, "_here", lambda: device[0])
    op = MAKE[name]()
    op.prepare()
    op.prepare()
    assert len(made) == 1 and made[0][1] > 0
    device[0] = 1
    op.prepare()
    assert [d for d, _ in made] == [0, 1]


@pytest.mark.gpu
def test_the_first_call_is_recorded_into_a_graph(gpu):
    import torch

    g = torch.Generator().manual_seed(0)
    x = torch.randn(1, 80, 96, generator=g).cuda()
    w, m = torch.zeros_like(x), torch.zeros_like(x)
    out, want = torch.empty_like(x), torch.empty_like(x)
    gate, ortho, muon = ops.BucketGate(9), ops.Orthogonaliser(1, 80, 96), ops.Muon(1, 80, 96)
    for op in (gate, ortho, muon):
        op.prepare()
    logits = torch.randn(3000, 9, generator=g).cuda()
    o = [torch.empty(3000, 1, dtype=torch.int32, device="cuda"), torch.empty(3000, 1, device="cuda"),
         torch.empty(9, dtype=torch.int32, device="cuda"), torch.empty(9, device="cuda"),
         torch.empty(1, dtype=torch.int32, device="cuda"), torch.empty(1, device="cuda")]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gate.forward(logits, *o)
        ortho(x, out)
        muon.step(w, m, x, 0.1)
    w_want, m_want = torch.zeros_like(x), torch.zeros_like(x)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in o]
        ops.Orthogonaliser(1, 80, 96)(x, want)
        ops.Muon(1, 80, 96).step(w_want, m_want, x, 0.1)
        gate.forward(logits, *o)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(w, w_want) and torch.equal(m, m_want)
        assert all(torch.equal(a, b) for a, b in zip(got, o))
