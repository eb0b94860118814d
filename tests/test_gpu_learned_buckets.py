"""The example that trains a learned bucket choice, end to end on the GPU."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

SPEC = importlib.util.spec_from_file_location(
    "learned_buckets", Path(__file__).resolve().parents[1] / "examples" / "learned_buckets.py")


@pytest.fixture(scope="module")
def example():
    m = importlib.util.module_from_spec(SPEC)
    SPEC.loader.exec_module(m)
    return m


def test_training_lowers_the_error_and_keeps_buckets_in_use(gpu, example):
    h = example.train(steps=40, positions=1024)
    first, last = h[0]["error"], sum(r["error"] for r in h[-5:]) / 5
    assert last < 0.5 * first, (first, last)
    assert sum(h[-1]["counts"]) == 1024 * 2
    assert sum(c > 0 for c in h[-1]["counts"]) >= 5


def test_gradients_of_the_whole_step(gpu, example):
    """The step's gradients against torch's autograd of the same model in 64 bits."""
    n, d, buckets, top = 64, 96, 6, 2
    m = example.LearnedBuckets(n, d, buckets, top, 0.3, seed=4)
    x = example.features(n, d, 3)
    target = torch.rand(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    w0, layers0, weight0 = m.w.clone(), m.layers.clone(), m.weight.clone()
    seen = {}
    m.muon_w.step = lambda w, mom, g, lr: seen.update(w=g.clone())
    m.muon_layers.step = lambda w, mom, g, lr: seen.update(layers=g.clone())
    m.step(x, target, 0.0)

    def leaf(t):
        return t.double().cpu().requires_grad_(True)

    w, layers, weight, bias, xd = leaf(w0[0]), leaf(layers0), leaf(weight0), leaf(torch.zeros(d)), leaf(x)
    h = torch.nn.functional.layer_norm(xd, (d,), weight, bias, 1e-5)
    p = torch.softmax(h @ w.t(), 1)
    at = m.bucket.cpu().long()
    share = p.gather(1, at)
    share = share / share.sum(1, keepdim=True)
    a = (h @ layers.reshape(-1, d).t()).view(n, buckets, -1)
    value = a.gather(1, at[:, :, None].expand(n, top, a.shape[2])).clamp(0, 1).mean(2)
    out = (share * value).sum(1)
    balance = 0.3 * buckets / (top * n * n) * (p.sum(0) * m.count.cpu().double()).sum()
    (((out - target.double().cpu()) ** 2).mean() + balance).backward()
    assert abs(float(balance) - float(m.balance_loss)) <= 1e-5 * float(balance)
    for got, exact in ((seen["w"][0], w.grad), (seen["layers"], layers.grad), (m.dx, xd.grad),
                       (m.dweight, weight.grad), (m.dbias, bias.grad)):
        # f32 products and sums of up to 96 values each way
        assert float((got.double().cpu() - exact).norm()) <= 2e-5 * float(exact.norm())
