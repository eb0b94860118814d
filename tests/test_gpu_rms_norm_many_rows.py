"""RMS norm where a workgroup takes one row after another: more rows than a grid has
workgroups, an output in 8 bits (4096 workgroups at most), sixteen waves a row backward.

Tolerances are those of test_gpu_rms_norm.py, from the same chains; the formulas in 64 bits
are computed on the GPU.
"""
import pytest
import torch

from tatara_amd import ops
from test_gpu_rms_norm import EPS32, NORM, TINY, TYPES, UNIT

pytestmark = pytest.mark.gpu

GRID = 1 << 20     # workgroups of the forward pass at most
BITS8_GRID = 4096  # of an output in 8 bits


def randn(g, rows, cols, dtype, pad=0, scale=1.0):
    x = torch.randn(rows, cols + pad, device="cuda", generator=g, dtype=TYPES[dtype])
    return x.mul_(scale)[:, pad // 2:pad // 2 + cols]


def inside(rows, cols, dtype):
    """A tensor inside a wider one, and what lies beside it."""
    wide = torch.full((rows, cols + 3), 7.0, dtype=TYPES[dtype], device="cuda")
    return wide[:, 1:cols + 1], lambda: (wide[:, :1] == 7.0).all() and (wide[:, cols + 1:] == 7.0).all()


def formula(s, w, eps=1e-6):
    s = s.double()
    rstd = 1.0 / torch.sqrt((s * s).mean(1) + eps)
    return s * rstd[:, None] * w.double(), rstd


# columns, and the rows that a workgroup takes at once: two lanes a row, a wave, four and sixteen
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("dtype,cols,at_once", [("f32", 5, 128), ("bf16", 257, 4), ("f32", 129, 4), ("bf16", 1537, 1),
                                                ("bf16", 8193, 1)])
def test_forward_beyond_the_grid(gpu, dtype, cols, at_once, add):
    rows = at_once * (GRID + 251) + at_once // 2
    assert rows > GRID * at_once
    g = torch.Generator(device="cuda").manual_seed(cols)
    x, w = randn(g, rows, cols, dtype), 1 + 0.2 * torch.randn(cols, device="cuda", generator=g)
    res = randn(g, rows, cols, dtype) if add else None
    first = GRID * at_once
    parts = [slice(0, 50), slice(first - 300, first + 300), slice(rows - 300, rows)]  # of both turns
    sums = [x[p] if res is None else (x[p].float() + res[p].float()).to(x.dtype) for p in parts]
    y, rstd = torch.empty_like(x), torch.full((rows,), 7.0, device="cuda")
    ops.RMSNorm(cols, dtype).forward(x, w, y, rstd, res, res)  # the sum into the residual
    for p, s in zip(parts, sums):
        ey, er = formula(s, w)
        assert ((rstd[p].double() / er - 1).abs() <= NORM).all()
        assert ((y[p].double() - ey).abs() <= (UNIT[dtype] + NORM) * ey.abs() + TINY[dtype]).all()
        assert res is None or torch.equal(res[p], s)
    assert (rstd != 7.0).all()


def values(q, out8):
    return q.float().double() if out8 == "e4m3" else q.double()


# rows that share a wave, a wave, four and sixteen waves a row: three turns at least of one form in each
MANY = [(1600003, 9), (140001, 100), (40001, 257), (9001, 2049), (9001, 8193)]


@pytest.mark.parametrize("out8,group", [("e4m3", 0), ("i8", 64), ("i8", 0), ("e4m3", 128)])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", MANY)
def test_several_rows_a_workgroup_in_8_bits(gpu, rows, cols, dtype, out8, group):
    assert rows > 2 * BITS8_GRID
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    pad = (1, 0, 6)[(rows + cols + group // 64) % 3]
    x, res = randn(g, rows, cols, dtype, pad, 0.7), randn(g, rows, cols, dtype, pad)
    # rows of other sizes than their neighbours: a maximum of the wrong row shows
    x *= torch.linspace(0.01, 3.0, 7, device="cuda")[torch.arange(rows, device="cuda") % 7, None].to(x.dtype)
    w = 1 + 0.2 * torch.randn(cols, device="cuda", generator=g)
    t8 = torch.float8_e4m3fn if out8 == "e4m3" else torch.int8
    wide = torch.full((rows, cols + 3), 3, dtype=torch.uint8, device="cuda")
    q = wide.view(t8)[:, 1:cols + 1]
    op = ops.RMSNorm(cols, dtype, 1e-6, out8, group)
    scale, total, rstd = torch.empty(rows, op.groups, device="cuda"), torch.empty_like(x), torch.empty(rows, device="cuda")
    op.forward_8bit(x, w, q, scale, rstd, res, total)
    for a in range(0, rows, 200000):
        at = slice(a, min(a + 200000, rows))
        s = (x[at].float() + res[at].float()).to(x.dtype)
        assert torch.equal(total[at], s)
        ey, er = formula(s, w)
        assert ((rstd[at].double() / er - 1).abs() <= NORM).all()
        most, size = 448.0 if out8 == "e4m3" else 127.0, group or cols
        top = torch.stack([p.abs().amax(1) for p in ey.split(size, 1)], 1)
        assert ((scale[at].double() / (top.clamp(min=2.0**-100) / most) - 1).abs() <= NORM + 2 * EPS32).all()
        got, v = values(q[at], out8), ey / scale[at].double().repeat_interleave(size, 1)[:, :cols]
        off = v.abs() * (NORM + 3 * EPS32)
        half = torch.clamp((v.abs() + off) * 2.0**-4, min=2.0**-10) if out8 == "e4m3" else 0.5
        assert ((got - v).abs() <= half + off).all()
    assert (wide[:, 0] == 3).all() and (wide[:, cols + 1:] == 3).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(5, 3), (1029, 33), (1029, 130)] + MANY)
def test_in_8_bits_the_sum_in_place(gpu, rows, cols, dtype):
    g = torch.Generator(device="cuda").manual_seed(cols)
    x, res = randn(g, rows, cols, dtype, 5), randn(g, rows, cols, dtype, 5)
    w, op = torch.randn(cols, device="cuda", generator=g), ops.RMSNorm(cols, dtype, group=32)

    def run(a, b, total):
        q, scale = torch.zeros(rows, cols, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(rows, op.groups, device="cuda")
        op.forward_8bit(a, w, q, scale, None, b, total)
        return q.view(torch.uint8), scale, total.clone()

    want = run(x, res, torch.empty_like(x))
    for to in (0, 1):
        wide = [x.clone(), res.clone()]
        for a, b in zip(run(*wide, wide[to]), want):
            assert torch.equal(a, b)


# sixteen waves a row, rows for two or more turns of 256 or 512 workgroups, above 4 MB: dweight by
# partial sums.  From 16385 columns on (f32, or with dtotal, from 8193) values are made again.
WIDE = [(700, 6145), (700, 8193), (300, 16385), (300, 32768), (2100, 6145)]


@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", WIDE)
def test_wide_rows_backward(gpu, rows, cols, dtype, add):
    assert rows * cols * 2 > 4 << 20 and rows > 256
    g = torch.Generator(device="cuda").manual_seed(rows * 11 + cols)
    pad = (1, 0, 6)[(rows + cols) % 3]
    s, dy = randn(g, rows, cols, dtype, pad, 0.7), randn(g, rows, cols, dtype, pad, 0.5)
    s *= torch.linspace(0.1, 3.0, 7, device="cuda")[torch.arange(rows, device="cuda") % 7, None].to(s.dtype)
    dt = randn(g, rows, cols, dtype, pad + 1, 0.5) if add else None
    w = 1 + 0.2 * torch.randn(cols, device="cuda", generator=g)
    rstd = formula(s, w)[1].float()
    dx, beside = inside(rows, cols, dtype)
    dw = torch.full((cols,), 7.0, device="cuda")
    op = ops.RMSNorm(cols, dtype)
    op.backward(dy, s, w, rstd, dx, dw, dt)
    s64, d64, r64 = s.double(), dy.double(), rstd.double()[:, None]
    h, gr = s64 * r64, d64 * w.double()
    edx = r64 * (gr - h * (gr * h).mean(1, keepdim=True)) + (dt.double() if add else 0.0)
    size = gr.abs() + 3 * h.abs() * (gr * h).abs().mean(1, keepdim=True)
    tol = (UNIT[dtype] + EPS32) * edx.abs() + TINY[dtype] + r64 * 64 * EPS32 * size
    assert ((dx.double() - edx).abs() <= tol).all() and beside()
    # a workgroup's rows, 32 partial sums of a column, 16 of them
    assert ((dw.double() - (d64 * h).sum(0)).abs() <= (rows // 256 + 64) * EPS32 * (d64 * h).abs().sum(0)).all()
    for turn in range(2):  # alike every time, and into dtotal
        again, dw2 = dt.clone() if add and turn else torch.empty_like(dx), torch.full((cols,), 7.0, device="cuda")
        op.backward(dy, s, w, rstd, again, dw2, again if add and turn else dt)
        assert torch.equal(again, dx) and torch.equal(dw2, dw)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(2051, 33), (4097, 130), (1100, 257), (1100, 769)])
def test_narrow_rows_in_place(gpu, rows, cols, dtype):
    """Rows that one wave or a part of it takes, whose last piece overlaps the one ahead."""
    g = torch.Generator(device="cuda").manual_seed(cols)
    x, res, dy, dt = (randn(g, rows, cols, dtype, 4) for _ in range(4))
    w, op = torch.randn(cols, device="cuda", generator=g), ops.RMSNorm(cols, dtype)
    y, total, rstd, dx = torch.empty_like(x), torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty_like(x)
    op.forward(x, w, y, rstd, res, total)
    op.backward(dy, total, w, rstd, dx, None, dt)
    for turn in range(2):
        a, b, y2 = x.clone(), res.clone(), torch.empty_like(x)
        to = (b, a)[turn]
        op.forward(a, w, y2, None, b, to)
        assert torch.equal(y2, y) and torch.equal(to, total)
    op.backward(dy, total, w, rstd, dt, None, dt)
    assert torch.equal(dt, dx)
