"""The operators around bucket layers together, as the example has them: embedding, dropout,
norm, gate, rows and back."""
import importlib.util
import sys
from pathlib import Path

import pytest
import torch
from philox import numbers

pytestmark = pytest.mark.gpu

EXAMPLES = Path(__file__).resolve().parents[1] / "examples"


@pytest.fixture(scope="module")
def example():
    sys.path.insert(0, str(EXAMPLES))
    try:
        spec = importlib.util.spec_from_file_location("bucket_layers", EXAMPLES / "bucket_layers.py")
        m = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(m)
    finally:
        sys.path.remove(str(EXAMPLES))
    return m


def batch(example, n, width, stages):
    g = torch.Generator(device="cuda").manual_seed(3)
    stage = torch.randint(-1, stages, (n,), device="cuda", generator=g, dtype=torch.int32)
    return example.features(n, width, 5), stage, torch.rand(n, device="cuda", generator=g)


def test_training_runs(gpu, example):
    h = example.train(steps=5, positions=512, width=96)
    assert len(h) == 5 and all(torch.isfinite(torch.tensor([r["error"], r["balance"]])).all() for r in h)
    assert all(sum(r["counts"]) == 512 * 2 for r in h)


@pytest.mark.parametrize("room", [0.7, 1.5, 3.0])  # 3.0 is room for every position in each of the buckets
def test_gradients_of_the_whole_step(gpu, example, room):
    """Against torch's autograd of the same model in 64 bits, with the same choices and mask."""
    n, width, e, k, stages, p, seed = 200, 96, 6, 2, 9, 0.25, 77
    m = example.BucketLayers(n, width, e, k, stages, hidden=24, p=p, balance=0.3, room=room, seed=seed)
    m.step_count.fill_(12)
    x, stage, target = batch(example, n, width, stages)
    out = m.forward(x, stage)
    m.backward(2.0 * (out - target) / n, stage)

    def leaf(t):
        return t.double().cpu().requires_grad_(True)

    table, weight, w, l, u, v = (leaf(t) for t in (m.table, m.weight, m.w[0], m.l, m.u, m.v))
    st, slot, at = stage.cpu().long(), m.slot.cpu(), m.bucket.cpu().long()
    looked_up = torch.where(st[:, None] >= 0, table[st.clamp(min=0)], 0.0)
    keep = torch.from_numpy(numbers(n, width, seed, 12).astype("int64")) >= round(p * 2.0**32)
    s = x.double().cpu() + torch.where(keep, looked_up / (1.0 - p), 0.0)
    h = s * (s.square().mean(1, keepdim=True) + m.norm.eps).rsqrt() * weight
    prob = torch.softmax(h @ w.t(), 1)
    share = prob.gather(1, at)
    share = share / share.sum(1, keepdim=True)
    a = torch.einsum("nd,ehd->neh", h, l).clamp(0.0, 1.0)
    up = torch.einsum("neh,edh->ned", a, u).gather(1, at[:, :, None].expand(n, k, width))
    y = (torch.where(slot >= 0, share, 0.0)[:, :, None] * up).sum(1)
    value = (s + y) @ v / width
    # too few rows for all choices, or one for each whatever they are
    assert (slot < 0).any() if room < 1.0 else room < 3.0 or not (slot < 0).any()
    # f32 products and sums of up to 96 values, one after the other
    assert float((out.double().cpu() - value.detach()).norm()) <= 2e-5 * float(value.detach().norm())
    balance = 0.3 * e / (k * n * n) * (prob.sum(0) * m.count.cpu().double()).sum()
    (((value - target.double().cpu()) ** 2).mean() + balance).backward()
    for got, exact in ((m.dtable, table.grad), (m.dweight, weight.grad), (m.dw[0], w.grad), (m.dl, l.grad),
                       (m.du, u.grad), (m.dv, v.grad)):
        assert float((got.double().cpu() - exact).norm()) <= 2e-5 * float(exact.norm())


def state(m):
    return {k: t.clone() for k, t in vars(m).items() if torch.is_tensor(t)}


def same(a, b):
    return [k for k in a if not torch.equal(a[k], b[k])]


def made(example, seed=1):
    m = example.BucketLayers(320, 96, 9, 2, 32, seed=seed)
    for t in vars(m).values():  # what is only written begins alike
        if torch.is_tensor(t) and t.data_ptr() not in {w.data_ptr() for w in (m.w, m.l, m.u, m.v, m.table, m.weight)}:
            t.zero_()
    return m


def test_a_step_in_a_graph(gpu, example):
    """Every replay is the next step, with the mask of its own, and eager steps between the replays
    do not change it."""
    x, stage, target = batch(example, 320, 96, 32)
    want, m = made(example), made(example)
    first = state(m)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            m.step(x, stage, target, 0.02)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.step(x, stage, target, 0.02)
    for k, t in first.items():
        getattr(m, k).copy_(t)
    for t in m.momentum:
        t.zero_()
    masks = []
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        want.step(x, stage, target, 0.02)
        torch.cuda.synchronize()
        names = [k for k in first if k not in ("step_count",)]
        a, b = state(m), state(want)
        assert same({k: a[k] for k in names}, b) == []
        masks.append((a["dropped"] == 0.0) & (a["looked_up"] != 0.0))
    assert not torch.equal(masks[0], masks[1]) and int(m.step_count) == 4


def test_torchs_current_stream(gpu, example):
    """Work that takes milliseconds stands ahead of the inputs on the stream."""
    x, stage, target = batch(example, 320, 96, 32)
    want, m = made(example), made(example)
    want.step(x, stage, target, 0.02)
    torch.cuda.synchronize()
    long = torch.zeros(1 << 28, device="cuda")
    late = torch.empty_like(x)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(20):
            long.add_(1.0)
        late.copy_(x)
        m.step(late, stage, target, 0.02)
        side.synchronize()
    assert same(state(want), state(m)) == []


def test_every_call_takes_a_stream(gpu):
    """The library's own stream and a torch stream that is given, with the same results."""
    from tatara_amd import ops
    from tatara_amd.runtime import Stream

    n, c, e, k = 500, 64, 9, 2
    g = torch.Generator().manual_seed(0)
    x, res = torch.randn(n, c, generator=g).cuda(), torch.randn(n, c, generator=g).cuda()
    bucket = torch.stack([torch.randperm(e, generator=g)[:k] for _ in range(n)]).int().cuda()
    token, gate = torch.randint(0, 40, (n,), generator=g, dtype=torch.int32).cuda(), torch.rand(n, k, generator=g).cuda()
    table = torch.randn(40, c, generator=g).cuda()
    norm, drop, rows, emb = ops.RMSNorm(c), ops.Dropout(c, 0.3, seed=5), ops.BucketRows(e, c, k), ops.Embedding(40, c, n)

    def run(stream):
        def empty(*shape, dtype=torch.float32):
            return torch.full(shape, 7, dtype=dtype, device="cuda")

        o = [empty(n, c) for _ in range(8)] + [empty(n), empty(c), empty(n, 1), empty(40, c), empty(n, k)]
        i = [empty(n, k, dtype=torch.int32), empty(n * k, dtype=torch.int32), empty(e + 1, dtype=torch.int32)]
        q, r = torch.zeros(n, c, dtype=torch.float8_e4m3fn, device="cuda"), [empty(n * k, c), empty(n * k, c)]
        torch.cuda.synchronize()
        norm.forward(x, None, o[0], o[8], res, o[1], stream=stream)
        norm.forward_8bit(x, None, q, o[10], residual=res, stream=stream)
        norm.backward(x, o[1], None, o[8], o[2], o[9], res, stream=stream)
        drop.forward(x, o[3], 4, residual=res, stream=stream)
        drop.backward(x, o[4], 4, stream=stream)
        rows.sort(bucket, *i, stream=stream)
        rows.gather(x, i[0], i[1], r[0], stream=stream)
        rows.combine(r[0], i[0], gate, o[5], stream=stream)
        rows.gather_backward(r[0], i[0], o[6], stream=stream)
        rows.combine_backward(res, r[0], i[0], i[1], gate, r[1], o[12], stream=stream)
        emb.forward(token, table, o[7], stream=stream)
        emb.backward(x, token, o[11], stream=stream)
        stream.synchronize() if stream else torch.cuda.synchronize()
        return o + i + r + [q.float()]

    want = run(None)
    with Stream() as own:
        assert all(torch.equal(a, b) for a, b in zip(want, run(own)))
    assert all(torch.equal(a, b) for a, b in zip(want, run(torch.cuda.Stream())))
    closed = Stream()
    closed.close()
    for call in (lambda: drop.forward(x, x, stream=closed), lambda: rows.sort(bucket, bucket, token, token, stream=closed)):
        with pytest.raises(ValueError, match="closed"):
            call()


def test_library_arrays(gpu):
    """DeviceArray operands: bf16 as uint16, e4m3 as uint8."""
    import numpy as np

    from tatara_amd import ops
    from tatara_amd.trainer import DeviceArray

    g = torch.Generator().manual_seed(2)
    x = torch.randn(30, 96, generator=g).bfloat16()
    X, R = DeviceArray(x.view(torch.uint16).numpy()), DeviceArray.empty((30, 96), np.uint16)
    Q, S = DeviceArray.empty((30, 96), np.uint8), DeviceArray.empty((30, 3), np.float32)
    norm = ops.RMSNorm(96, "bf16", group=32)
    norm.forward_8bit(X, None, Q, S)
    q, s, total = torch.empty(30, 96, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(30, 3, device="cuda"), None
    norm.forward_8bit(x.cuda(), None, q, s, total=total)
    torch.cuda.synchronize()
    assert np.array_equal(Q.to_host(), q.view(torch.uint8).cpu().numpy()) and np.array_equal(S.to_host(), s.cpu().numpy())
    T, D = DeviceArray(np.array([5], np.int64)), ops.Dropout(96, 0.5, "bf16", seed=8)
    D.forward(X, R, step=2, more_steps=T)
    y = torch.empty(30, 96, dtype=torch.bfloat16, device="cuda")
    D.forward(x.cuda(), y, step=7)
    torch.cuda.synchronize()
    assert np.array_equal(R.to_host(), y.view(torch.uint16).cpu().numpy())
