"""The bucket gate on the GPU against its formulas in 64 bits.

Whole numbers (choices, counts) are equal.  A probability carries the rounding
of l - max (2^-24 of it), expf (2 ulp), the sum over at most 1024 buckets (16 a
lane, 6 shuffles) and the division: (64 + 2 |l - max|) 2^-24 of it bounds them.
"""
import math

import pytest
import torch

from tatara_amd import ops
from tatara_amd.runtime import Stream

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}
TINY = {"f32": 2.0**-126, "f16": 2.0**-25, "bf16": 2.0**-126}
EPS32 = 2.0**-24

CASES = [(1, 1, 1), (1, 9, 1), (1, 8, 2), (3, 2, 2), (257, 9, 1), (1000, 8, 2), (513, 16, 3), (300, 17, 4),
         (129, 64, 4), (77, 65, 8), (100, 200, 5), (50, 257, 16), (33, 512, 2), (20, 700, 6), (9, 1024, 16),
         (70001, 9, 1), (40000, 33, 2)]


def inputs(n, e, dtype, masked, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    l = torch.randn(n, e + pad, generator=g) * 2
    valid = None
    if masked:
        l[torch.rand(n, e + pad, generator=g) < 0.3] = -math.inf
        l[torch.rand(n, generator=g) < 0.1] = -math.inf
        valid = (torch.rand(n, generator=g) < 0.8).to(torch.uint8)
    return l.to(TYPES[dtype])[:, pad // 2:pad // 2 + e], valid


def reference(l, valid, k, share, balance):
    n, e = l.shape
    l = l.double()
    counted = (l > -math.inf).any(1)
    if valid is not None:
        counted &= valid != 0
    top = l.amax(1, keepdim=True)
    z = torch.exp(l - torch.where(top > -math.inf, top, 0.0))
    p = torch.where(counted[:, None], z / z.sum(1, keepdim=True), 0.0)
    value, order = torch.sort(l, dim=1, descending=True, stable=True)
    taken = (value[:, :k] > -math.inf) & counted[:, None]
    bucket = torch.where(taken, order[:, :k], -1)
    gate = torch.where(taken, p.gather(1, order[:, :k]), 0.0)
    if share:
        gate = gate / torch.where(counted, gate.sum(1), 1.0)[:, None]
    count = torch.bincount(bucket[taken], minlength=e)
    c = int(counted.sum())
    loss = balance * e / k * float((count.double() * p.sum(0)).sum()) / max(c, 1) ** 2
    off = (64 + 2 * torch.where(torch.isfinite(l), (l - top).abs(), 0.0)).amax(1, keepdim=True) * EPS32
    return dict(p=p, bucket=bucket, gate=gate, count=count, prob=p.sum(0), counted=c, loss=loss, off=off)


def outputs(n, e, k):
    return (torch.full((n, k), 77, dtype=torch.int32, device="cuda"), torch.full((n, k), 7.0, device="cuda"),
            torch.full((e,), 77, dtype=torch.int32, device="cuda"), torch.full((e,), 7.0, device="cuda"),
            torch.full((1,), 77, dtype=torch.int32, device="cuda"), torch.full((1,), 7.0, device="cuda"))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,e,k", CASES)
@pytest.mark.parametrize("masked,share", [(False, False), (True, True)])
def test_forward(gpu, n, e, k, dtype, masked, share):
    l, valid = inputs(n, e, dtype, masked, n + e + k, pad=(n + e) % 4)
    r = reference(l, valid, k, share, 0.02)
    bucket, gate, count, prob, counted, loss = outputs(n, e, k)
    op = ops.BucketGate(e, k, dtype, share, 0.02)
    lg = torch.empty(n, e + 5, dtype=l.dtype, device="cuda")[:, 2:e + 2].copy_(l)
    op.forward(lg, bucket, gate, count, prob, counted, loss, valid=None if valid is None else valid.cuda())
    assert torch.equal(bucket.cpu().long(), r["bucket"])
    assert torch.equal(count.cpu().long(), r["count"]) and int(counted) == r["counted"]
    assert ((gate.double().cpu() - r["gate"]).abs() <= 2 * r["off"] * r["gate"] + TINY["f32"]).all()
    # sums of a lane's positions in order (n / 256 blocks), then shuffles, waves and workgroups
    chain = n / (256 * 8) + 64
    assert ((prob.double().cpu() - r["prob"]).abs()
            <= (r["p"] * r["off"]).sum(0) + chain * EPS32 * r["prob"] + TINY["f32"]).all()
    assert abs(float(loss) - r["loss"]) <= (float(r["off"].max()) + (chain + 4) * EPS32) * r["loss"]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,e,k", CASES)
@pytest.mark.parametrize("masked,share", [(False, True), (True, False)])
def test_backward(gpu, n, e, k, dtype, masked, share):
    l, valid = inputs(n, e, dtype, masked, n + 2 * e + k, pad=(n + e) % 4)
    r = reference(l, valid, k, share, 0.02)
    g = torch.Generator().manual_seed(3)
    dgate = torch.randn(n, k, generator=g)
    dloss = 3.0 * n
    x = l.double().requires_grad_(True)
    # autograd through the formula, the counts held fixed
    keep = r["p"].sum(1) > 0
    top = torch.where(keep[:, None], x.amax(1, keepdim=True), 0.0).detach()
    z = torch.exp(x - top)
    p = torch.where(keep[:, None], z / torch.where(keep, z.sum(1), 1.0)[:, None], 0.0)
    taken = r["bucket"] >= 0
    gate = torch.where(taken, p.gather(1, r["bucket"].clamp(min=0)), 0.0)
    if share:
        gate = gate / torch.where(keep, gate.sum(1), 1.0)[:, None]
    loss = 0.02 * e / k / max(r["counted"], 1) ** 2 * (p.sum(0) * r["count"]).sum()
    ((gate * dgate).sum() + dloss * loss).backward()
    exact = torch.where(torch.isfinite(l), x.grad, 0.0)
    wide = torch.full((n, e + 2), 7.0, dtype=TYPES[dtype], device="cuda")
    d = wide[:, 1:e + 1]
    ops.BucketGate(e, k, dtype, share, 0.02).backward(
        l.cuda(), r["bucket"].int().cuda(), r["count"].int().cuda(),
        torch.tensor([r["counted"]], dtype=torch.int32, device="cuda"), d, dgate.cuda(), dloss,
        None if valid is None else valid.cuda())
    # sizes of what is summed: |h| of every bucket, through p
    h = (dloss * 0.02 * e / k / max(r["counted"], 1) ** 2 * r["count"]).double().expand(n, e).clone()
    inner = dgate.double().abs()
    if share:
        total = torch.where(keep, torch.where(taken, r["p"].gather(1, r["bucket"].clamp(min=0)), 0.0).sum(1), 1.0)
        inner = (inner + (inner * r["gate"]).sum(1, keepdim=True)) / total[:, None]
    h.scatter_add_(1, r["bucket"].clamp(min=0), torch.where(taken, inner, 0.0))
    size = r["p"] * (h + (r["p"] * h).sum(1, keepdim=True))
    tol = UNIT[dtype] * exact.abs() + 4 * r["off"] * size + TINY[dtype]
    assert ((d.double().cpu() - exact).abs() <= tol).all()
    assert (wide[:, 0] == 7.0).all() and (wide[:, -1] == 7.0).all()


def test_gradient_against_differences(gpu):
    """The kernel's own loss and gates, moved along a direction that changes no choice."""
    n, e, k, step = 40, 12, 3, 2.0**-7
    g = torch.Generator().manual_seed(0)
    l = torch.stack([torch.randperm(e, generator=g) for _ in range(n)]).double() * 0.3  # gaps of 0.3
    v = torch.rand(n, e, generator=g).double() * 2 - 1
    dgate = torch.randn(n, k, generator=g).double()
    op = ops.BucketGate(e, k, "f32", True, 5.0)

    def value(t):
        bucket, gate, count, prob, counted, loss = outputs(n, e, k)
        op.forward((l + t * v).float().cuda(), bucket, gate, count, prob, counted, loss)
        return float((gate.double().cpu() * dgate).sum()) + float(loss), (bucket, count, counted)

    def exact_value(t):
        r = reference(l + t * v, None, k, True, 5.0)
        return float((r["gate"] * dgate).sum()) + r["loss"]

    _, (bucket, count, counted) = value(0.0)
    d = torch.empty(n, e, device="cuda")
    op.backward(l.float().cuda(), bucket, count, counted, d, dgate.float().cuda())
    seen = (value(step)[0] - value(-step)[0]) / (2 * step)
    cut = 2 * abs((exact_value(step) - exact_value(-step)) / (2 * step)
                  - (exact_value(step / 2) - exact_value(-step / 2)) / step)
    rounding = 200 * EPS32 * (float(dgate.abs().sum()) + 5.0) / step
    assert abs(seen - float((d.double().cpu() * v).sum())) <= cut + rounding


def test_ties_zeros_and_lowest_values(gpu):
    low = torch.finfo(torch.float32).min
    l = torch.tensor([[1.0, 1.0, 1.0, 0.0], [0.0, -0.0, 0.0, -0.0], [low, low, low, low],
                      [low, 3.0, low, -math.inf], [-math.inf] * 4, [-math.inf, -math.inf, 2.0, -math.inf]])
    n, e, k = 6, 4, 3
    bucket, gate, count, prob, counted, loss = outputs(n, e, k)
    ops.BucketGate(e, k).forward(l.cuda(), bucket, gate, count, prob, counted, loss)
    assert bucket.tolist() == [[0, 1, 2], [0, 1, 2], [0, 1, 2], [1, 0, 2], [-1, -1, -1], [2, -1, -1]]
    assert gate[1].tolist() == [0.25] * 3 and gate[2].tolist() == [0.25] * 3  # all alike, also at the type's lowest
    assert gate[3].tolist() == [1.0, 0.0, 0.0] and not gate[4].any() and gate[5].tolist() == [1.0, 0.0, 0.0]
    assert int(counted) == 5 and count.tolist() == [4, 4, 5, 0]


def test_nothing_counts(gpu):
    for n in (0, 5, 3000):
        bucket, gate, count, prob, counted, loss = outputs(n, 9, 2)
        l, valid = torch.randn(n, 9, device="cuda"), torch.zeros(n, dtype=torch.uint8, device="cuda")
        op = ops.BucketGate(9, 2)
        op.forward(l, bucket, gate, count, prob, counted, loss, valid=valid)
        assert not count.any() and not prob.any() and not counted.any() and not loss.any()
        assert (bucket == -1).all() and not gate.any()
        d = torch.full((n, 9), 7.0, device="cuda")
        op.backward(l, bucket, count, counted, d, torch.ones(n, 2, device="cuda"), valid=valid)
        assert not d.any()


def test_nan_and_infinity(gpu):
    l = torch.randn(3, 9, generator=torch.Generator().manual_seed(0))
    l[0, 4] = math.nan
    l[1, 7] = math.inf
    bucket, gate, count, prob, counted, loss = outputs(3, 9, 2)
    ops.BucketGate(9, 2).forward(l.cuda(), bucket, gate, count, prob, counted, loss)
    assert int(bucket[0, 0]) == 4 and int(bucket[1, 0]) == 7 and int(counted) == 3
    assert torch.isnan(gate[:2]).all() and torch.isfinite(gate[2]).all()
    assert torch.isnan(prob).all() and torch.isnan(loss).all()


def test_choices_out_of_range_are_passed_over(gpu):
    l = torch.randn(4, 9, device="cuda")
    count, counted = torch.ones(9, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    dg, out = torch.ones(4, 1, device="cuda"), []
    for v in (-1, 9, 2**31 - 1):
        d = torch.empty(4, 9, device="cuda")
        bucket = torch.full((4, 1), v, dtype=torch.int32, device="cuda")
        ops.BucketGate(9).backward(l, bucket, count, counted, d, dg)
        out.append(d)
    assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])


def test_same_result_every_time_and_on_another_stream(gpu):
    l = torch.randn(50000, 9, device="cuda")
    op, got = ops.BucketGate(9, 2), []
    with Stream() as s:
        for stream in (None, None, s):
            o = outputs(50000, 9, 2)
            torch.cuda.synchronize()
            op.forward(l, *o, stream=stream)
            stream.synchronize() if stream else torch.cuda.synchronize()
            got.append(o)
    assert all(torch.equal(a, b) for o in got[1:] for a, b in zip(got[0], o))
