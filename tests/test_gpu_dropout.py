"""Dropout on the GPU: which values stay is a whole number's comparison and what they become
one product and one sum in f32, so results are equal, bit for bit."""
import numpy as np
import pytest
import torch
from philox import numbers

from tatara_amd import ops

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SHAPES = [(1, 1), (3, 2), (5, 7), (1, 8), (2, 1536), (70, 130), (33, 257), (1021, 96), (2, 40000), (3000, 5)]
SEED = 0x1234567890ABCDEF


def kept(rows, cols, p, seed, step, first_row=0):
    return torch.from_numpy(numbers(rows, cols, seed, step, first_row) >= np.uint64(round(p * 2.0**32)))


def expected(x, residual, keep, p):
    y = torch.where(keep.cuda(), x.float() * (1.0 / (1.0 - p)), 0.0)
    return (y if residual is None else y + residual.float()).to(x.dtype)


def rows_of(g, rows, cols, pad, dtype):
    return torch.randn(rows, cols + pad, generator=g).to(TYPES[dtype]).cuda()[:, pad // 2:pad // 2 + cols]


@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("p", [0.1, 0.5])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward_and_backward(gpu, rows, cols, dtype, p, add):
    g = torch.Generator().manual_seed(rows + cols)
    pad = (0, 1, 6)[(rows + cols) % 3]
    x, dy = rows_of(g, rows, cols, pad, dtype), rows_of(g, rows, cols, pad, dtype)
    res = rows_of(g, rows, cols, pad + 1, dtype) if add else None
    wide = torch.full((rows, cols + 3), 7.0, dtype=TYPES[dtype], device="cuda")
    y, step = wide[:, 1:cols + 1], 5 * 2**32 + 77 + rows
    op = ops.Dropout(cols, p, dtype, SEED)
    op.forward(x, y, step, res)
    keep = kept(rows, cols, p, SEED, step)
    assert torch.equal(y, expected(x, res, keep, p))
    assert (wide[:, 0] == 7.0).all() and (wide[:, cols + 1:] == 7.0).all()
    dx = torch.empty_like(dy)
    op.backward(dy, dx, step)
    assert torch.equal(dx, expected(dy, None, keep, p))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(3, 2), (700, 7), (5000, 130), (40, 1537), (3, 40000)])
def test_in_place(gpu, rows, cols, dtype):
    g = torch.Generator().manual_seed(cols)
    x, res = rows_of(g, rows, cols, 5, dtype), rows_of(g, rows, cols, 5, dtype)
    op, y = ops.Dropout(cols, 0.4, dtype, SEED), torch.empty(rows, cols, dtype=TYPES[dtype], device="cuda")
    op.forward(x, y, 9, res)
    for to in (0, 1):
        pair = [x.clone(), res.clone()]
        op.forward(pair[0], pair[to], 9, pair[1])
        assert torch.equal(pair[to], y)
    op.forward(x, y, 9)
    op.backward(x, x, 9)
    assert torch.equal(x, y)


def test_a_part_of_a_batch_and_steps_on_the_device(gpu):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(300, 77, generator=g).cuda()
    op, y, z = ops.Dropout(77, 0.3, seed=3), torch.empty_like(x), torch.empty_like(x)
    op.forward(x, y, 2**40 + 5)
    more = torch.tensor([2**40 - 7], device="cuda")
    op.forward(x[:100], z[:100], 12, more_steps=more)
    op.forward(x[100:], z[100:], 12, more_steps=more, first_row=100)
    assert torch.equal(y, z)
    last = 2**32 - 300
    op.forward(x, y, first_row=last)
    assert torch.equal(y, expected(x, None, kept(300, 77, 0.3, 3, 0, last), 0.3))


def test_no_and_nearly_all(gpu):
    x = torch.randn(50, 90, generator=torch.Generator().manual_seed(1)).cuda()
    y = torch.empty_like(x)
    ops.Dropout(90, 0.0, seed=9).forward(x, y)
    assert torch.equal(x, y)
    ops.Dropout(90, 1.0 - 2.0**-53, seed=9).forward(x, y)
    keep = torch.from_numpy(numbers(50, 90, 9, 0) >= np.uint64(2**32 - 1))
    assert not y.cpu()[~keep].any()


def test_share_that_is_dropped(gpu):
    """Of 2^24 values: five standard deviations of a binomial count."""
    n, p = 1 << 24, 0.1
    x = torch.ones(n // 4096, 4096, device="cuda")
    y, z = torch.empty_like(x), torch.empty_like(x)
    op = ops.Dropout(4096, p, seed=11)
    op.forward(x, y, 1)
    op.forward(x, z, 2)
    a, b = y == 0, z == 0
    for count, q in ((a.sum(), p), (b.sum(), p), ((a & b).sum(), p * p), ((a[:, 1:] & a[:, :-1]).sum(), p * p),
                     ((a[1:] & a[:-1]).sum(), p * p)):
        assert abs(int(count) - q * n) <= 5 * (q * n) ** 0.5 + 2 * p * p * n / 4096


def test_dropped_values_are_zero_whatever_they_were(gpu):
    x = torch.full((40, 100), float("nan"), device="cuda")
    y = torch.empty_like(x)
    ops.Dropout(100, 0.5, seed=1).forward(x, y)
    keep = kept(40, 100, 0.5, 1, 0).cuda()
    assert torch.isnan(y[keep]).all() and (y[~keep] == 0).all()


def test_no_rows(gpu):
    none = torch.empty(0, 9, device="cuda")
    ops.Dropout(9, 0.5).forward(none, none)


def test_more_pieces_than_a_grid_holds(gpu):
    """2^20 workgroups of 1024 rows, and some: in bf16 of one column, 2 GiB."""
    rows = (1 << 30) + 12345
    x = torch.ones(rows, 1, dtype=torch.bfloat16, device="cuda")
    y = torch.full_like(x, 7.0)
    ops.Dropout(1, 0.5, "bf16", 21).forward(x, y)
    for first in (0, 1 << 29, rows - 5000):
        keep = kept(5000, 1, 0.5, 21, 0, first)
        assert torch.equal(y[first:first + 5000], expected(x[:5000], None, keep, 0.5))
