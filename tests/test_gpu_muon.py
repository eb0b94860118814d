"""Orthogonalised updates on the GPU against Newton-Schulz steps in 64 bits.

A step's own error is at most e = 2^-20 of |X|: operands of 22 bits (2^-22 each)
and f32 sums.  An error that enters is multiplied by at most a = 3.4445 in a
later step, so five steps leave at most e (1 + a + ... + a^4) = 198 e = 1.9e-4;
the result is rounded once to its type.
"""
import math

import pytest
import torch

from tatara_amd import ops
from tatara_amd.runtime import Stream

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}
A, B, C = 3.4445, -4.7750, 2.0315


def bound(steps=5):
    return 2.0**-20 * sum(A**i for i in range(steps))


def reference(u, steps=5):
    u = u.double()
    x = u / (torch.linalg.vector_norm(u, dim=(1, 2), keepdim=True) + 1e-7)
    flip = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2) if flip else x
    for _ in range(steps):
        g = x @ x.transpose(1, 2)
        x = A * x + (B * g + C * g @ g) @ x
    return x.transpose(1, 2) if flip else x


def off(got, exact):
    return float((got.double().cpu() - exact).norm() / exact.norm())


def matrices(batch, rows, cols, seed, low_rank=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(batch, rows, cols, generator=g)
    if low_rank:
        r = min(4, rows, cols)
        x = torch.randn(batch, rows, r, generator=g) @ torch.randn(batch, r, cols, generator=g) + 0.05 * x
    return x * 1e-3


SHAPES = [(1, 1, 1), (3, 1, 5), (2, 5, 1), (9, 32, 30), (9, 8, 768), (2, 16, 1536), (1, 64, 64), (2, 65, 64),
          (1, 100, 300), (3, 300, 100), (1, 128, 129), (2, 193, 257), (1, 512, 32), (1, 520, 390), (7, 33, 1000)]
# batches that take each size of a product's tiles, upright and lying
TILES = [(14, 150, 130), (18, 130, 150), (25, 130, 150), (60, 150, 130), (300, 140, 150), (300, 150, 140)]
SHAPES += TILES


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("batch,rows,cols", SHAPES)
def test_orthogonalise(gpu, batch, rows, cols, dtype):
    u = matrices(batch, rows, cols, batch + rows + cols, low_rank=rows % 2 == 0).to(TYPES[dtype])
    if dtype == "f16":
        u = u * 64  # clear of its subnormals
    out = torch.empty_like(u, device="cuda")
    ops.Orthogonaliser(batch, rows, cols, dtype)(u.cuda(), out)
    assert off(out, reference(u)) <= bound() + UNIT[dtype]


def test_singular_values_come_near_one(gpu):
    u = matrices(1, 200, 320, 1)
    out = torch.empty_like(u, device="cuda")
    ops.Orthogonaliser(1, 200, 320)(u.cuda(), out)
    s = torch.linalg.svdvals(out.double().cpu())
    assert float(s.max()) < 1.25 and float(s.min()) > 0.6


@pytest.mark.parametrize("steps", [1, 2, 8])
def test_steps(gpu, steps):
    u = matrices(2, 70, 90, 4)
    out = torch.empty_like(u, device="cuda")
    ops.Orthogonaliser(2, 70, 90, steps=steps)(u.cuda(), out)
    assert off(out, reference(u, steps)) <= bound(steps)


@pytest.mark.parametrize("rows,cols", [(20, 33), (150, 75)])
def test_strides_and_in_place(gpu, rows, cols):
    wide = torch.zeros(3, rows + 2, cols + 7, device="cuda")
    x = wide[:, 1:rows + 1, 3:cols + 3]
    u = matrices(3, rows, cols, 9)
    x.copy_(u)
    op = ops.Orthogonaliser(3, rows, cols)
    out = torch.full((3, rows, cols + 1), 7.0, device="cuda")
    op(x, out[:, :, :cols])
    assert off(out[:, :, :cols], reference(u)) <= bound()
    assert (out[:, :, cols] == 7.0).all()
    op(x, x)
    assert torch.equal(x, out[:, :, :cols])
    x.zero_()
    assert not wide.any(), "values beside the matrices were written"


def test_zeros_sizes_and_special_values(gpu):
    u = matrices(5, 40, 50, 2)
    u[0] = 0
    u[1] *= 1e33  # squares pass f32's range
    u[2] = 0
    u[2, 3, 4] = 1e-3  # one entry: its own orthogonal factor
    u[3, 1, 1] = math.nan
    u[4, 2, 2] = math.inf
    out = torch.empty_like(u, device="cuda")
    ops.Orthogonaliser(5, 40, 50)(u.cuda(), out)
    out = out.cpu()
    assert not out[0].any()
    assert off(out[1:2], reference(u[1:2])) <= bound()
    assert off(out[2:3], reference(u[2:3])) <= bound()
    assert torch.isnan(out[3]).all() and torch.isnan(out[4]).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("batch,rows,cols", [(9, 16, 200), (1, 96, 32), (2, 130, 140)] + TILES[:5])
def test_muon_steps(gpu, batch, rows, cols, nesterov, dtype):
    w = 0.05 * torch.randn(batch, rows, cols, generator=torch.Generator().manual_seed(0))
    m = torch.zeros(batch, rows, cols)
    beta, lr, decay, scale, cap = 0.9, 0.05, 0.1, 1.5, 0.08
    op = ops.Muon(batch, rows, cols, beta, nesterov, decay, dtype, min_w=-cap, max_w=cap)
    W, M = w.cuda(), m.cuda()
    ew, em = w.double(), m.double()
    for k in range(3):
        g = (matrices(batch, rows, cols, 10 + k) * 64).to(TYPES[dtype])
        op.step(W, M, g.cuda(), lr, scale)
        em = beta * em + (1 - beta) * g.double()
        o = reference((1 - beta) * g.double() + beta * em if nesterov else em)
        ew = (ew * (1 - lr * decay) - lr * scale * o).clamp(-cap, cap)
        assert off(M, em) <= 4 * 2.0**-24 * (k + 1)
        # the update's error and two roundings of the weights, a step
        tol = (k + 1) * (lr * scale * bound() * float(o.norm()) + 2.0**-23 * float(ew.norm()))
        assert float((W.double().cpu() - ew).norm()) <= tol
    assert float(W.abs().max()) <= cap


def test_no_learning_rate_keeps_the_weights(gpu):
    w = torch.randn(2, 30, 40, generator=torch.Generator().manual_seed(0))
    W, M = w.cuda(), torch.zeros(2, 30, 40, device="cuda")
    ops.Muon(2, 30, 40).step(W, M, matrices(2, 30, 40, 1).cuda(), 0.0)
    assert torch.equal(W.cpu(), w)


def test_same_result_every_time_and_on_another_stream(gpu):
    u = matrices(3, 200, 160, 5).cuda()
    op, got = ops.Orthogonaliser(3, 200, 160), []
    with Stream() as s:
        for stream in (None, None, s):
            out = torch.empty_like(u)
            torch.cuda.synchronize()
            op(u, out, stream=stream)
            stream.synchronize() if stream else torch.cuda.synchronize()
            got.append(out)
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_broadcast_input(gpu):
    """Matrices that share one input, by a stride of zero."""
    u = matrices(1, 24, 48, 6).cuda()
    out = torch.empty(4, 24, 48, device="cuda")
    ops.Orthogonaliser(4, 24, 48)(u.expand(4, 24, 48), out)
    assert all(torch.equal(out[0], o) for o in out[1:])
    assert off(out[:1], reference(u.cpu())) <= bound()
