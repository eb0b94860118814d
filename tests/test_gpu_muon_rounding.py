"""16-bit results of the Newton-Schulz steps carry their type's rounding and little more.

The result's own rounding, norm-wise, is that of the exact result rounded to the
type.  Beside it stands what products leave, e (1 + a + ... + a^4) with e = 2^-20 of
a step (operands of 22 bits and f32 sums) and a = 3.4445 the most that a later step
multiplies it by.
"""
import pytest
import torch

from tatara_amd import ops

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
A, B, C = 3.4445, -4.7750, 2.0315


def left_over(steps):
    return 2.0**-20 * sum(A**i for i in range(steps))


def exact(u, steps):
    u = u.double()
    x = u / (torch.linalg.vector_norm(u, dim=(1, 2), keepdim=True) + 1e-7)
    flip = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2) if flip else x
    for _ in range(steps):
        g = x @ x.transpose(1, 2)
        x = A * x + (B * g + C * g @ g) @ x
    return x.transpose(1, 2) if flip else x


def full_rank(batch, rows, cols, g):
    return torch.randn(batch, rows, cols, generator=g)


def nearly_low_rank(batch, rows, cols, g):
    return (torch.randn(batch, rows, 4, generator=g) @ torch.randn(batch, 4, cols, generator=g)
            + 0.005 * torch.randn(batch, rows, cols, generator=g))


def graded(batch, rows, cols, g):
    """Rows of falling size."""
    return torch.randn(batch, rows, cols, generator=g) * torch.logspace(0, -3, rows)[:, None]


def alike(batch, rows, cols, g):
    """One singular value, which is at 1 from the start."""
    return torch.full((batch, rows, cols), 3.0)


def low_rank(batch, rows, cols, g):
    """Whole numbers of rank 3, exact in 16 bits."""
    return (torch.randint(-2, 3, (batch, rows, 3), generator=g) @ torch.randint(-2, 3, (batch, 3, cols),
                                                                              generator=g)).float()


def check(dtype, batch, rows, cols, kind, steps, seed):
    u = kind(batch, rows, cols, torch.Generator().manual_seed(seed)).to(TYPES[dtype])
    out = torch.empty_like(u, device="cuda")
    ops.Orthogonaliser(batch, rows, cols, dtype, steps)(u.cuda(), out)
    e = exact(u, steps)
    for got, want in zip(out.double().cpu(), e):
        rounding = float((want.to(TYPES[dtype]).double() - want).norm() / want.norm())
        off = float((got - want).norm() / want.norm())
        assert off <= rounding + left_over(steps), (off, rounding)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kind", [full_rank, nearly_low_rank, graded, alike, low_rank])
@pytest.mark.parametrize("batch,rows,cols", [(2, 65, 66), (1, 65, 100), (1, 100, 72), (1, 66, 1000), (1, 33, 1100),
                                             (3, 129, 127), (1, 128, 512), (2, 257, 256), (1, 511, 600),
                                             (1, 512, 513)])
def test_rounding_of_the_type_alone(gpu, batch, rows, cols, kind, dtype):
    check(dtype, batch, rows, cols, kind, 5, batch + rows + cols)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("steps", [1, 2, 3, 6])
@pytest.mark.parametrize("rows,cols", [(70, 90), (140, 130), (512, 520)])
def test_rounding_with_other_steps(gpu, rows, cols, steps, dtype):
    check(dtype, 1, rows, cols, full_rank, steps, rows + steps)
