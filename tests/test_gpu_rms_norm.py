"""Root-mean-square norm on the GPU against its formulas in 64 bits.

Tolerances follow from the arithmetic: sums are f32 in chains of at most 32 values a
lane, 6 joins of lanes, 16 waves (64 roundings of the summed magnitudes bound them),
and the result is rounded once to the element type.
"""
import pytest
import torch

from tatara_amd import ops

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}  # half an ulp, relative
TINY = {"f32": 0.0, "f16": 2.0**-25, "bf16": 0.0}  # half an ulp of subnormals
EPS32 = 2.0**-24

# either side of a piece, of the widths where more waves share a row, of the rows where one does
SHAPES = [(1, 1), (1, 1536), (3, 7), (5, 64), (2, 65), (70, 256), (33, 257), (9, 770), (2100, 96), (2049, 513),
          (1100, 1536), (1100, 1537), (4, 2049), (3, 6145), (2, 8193), (2, 32768),
          (5000, 33), (4097, 16), (3000, 9), (2051, 128), (1029, 130), (2500, 3)]


def rows_of(g, rows, cols, pad, dtype, scale=1.0):
    x = (torch.randn(rows, cols + pad, generator=g) * scale).to(TYPES[dtype])
    return x.cuda()[:, pad // 2:pad // 2 + cols]


def inside(rows, cols, dtype):
    """A tensor inside a wider one, and what lies beside it."""
    wide = torch.full((rows, cols + 3), 7.0, dtype=TYPES[dtype], device="cuda")
    return wide[:, 1:cols + 1], lambda: (wide[:, :1] == 7.0).all() and (wide[:, cols + 1:] == 7.0).all()


def formula(s, w, eps):
    s = s.double().cpu()
    rstd = 1.0 / torch.sqrt((s * s).mean(1) + eps)
    return s * rstd[:, None] * w.double(), rstd


# y's relative error: half the sum's, and the root's, the quotient's and two products' roundings
NORM = (32 + 6) * EPS32


@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward(gpu, rows, cols, dtype, add):
    g = torch.Generator().manual_seed(rows * 7 + cols)
    pad = (0, 1, 6)[(rows + cols) % 3]
    x = rows_of(g, rows, cols, pad, dtype, 0.7)
    res = rows_of(g, rows, cols, pad + 2, dtype, 1.5) if add else None
    w = 1 + 0.2 * torch.randn(cols, generator=g)
    y, beside_y = inside(rows, cols, dtype)
    total, beside = inside(rows, cols, dtype)
    rstd = torch.empty(rows, device="cuda")
    ops.RMSNorm(cols, dtype, 1e-6).forward(x, w.cuda(), y, rstd, res, total if add else None)
    s = (x.float() + res.float()).to(x.dtype) if add else x
    if add:
        assert torch.equal(total, s) and beside()
    ey, er = formula(s, w, 1e-6)
    assert ((rstd.double().cpu() / er - 1).abs() <= NORM).all()
    assert ((y.double().cpu() - ey).abs() <= (UNIT[dtype] + NORM) * ey.abs() + TINY[dtype]).all()
    assert beside_y()


def values(q, out8):
    return q.float().double().cpu() if out8 == "e4m3" else q.double().cpu()


@pytest.mark.parametrize("out8,group", [("e4m3", 0), ("e4m3", 128), ("i8", 0), ("i8", 32), ("e4m3", 64)])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward_in_8_bits(gpu, rows, cols, dtype, out8, group):
    g = torch.Generator().manual_seed(rows * 5 + cols)
    pad = (1, 0, 6)[(rows + cols) % 3]
    x, res = rows_of(g, rows, cols, pad, dtype, 0.7), rows_of(g, rows, cols, pad, dtype)
    w = 1 + 0.2 * torch.randn(cols, generator=g)
    t8 = torch.float8_e4m3fn if out8 == "e4m3" else torch.int8
    wide = torch.full((rows, cols + 3), 3, dtype=torch.uint8, device="cuda")
    q = wide.view(t8)[:, 1:cols + 1]
    op = ops.RMSNorm(cols, dtype, 1e-6, out8, group)
    scale, total = torch.empty(rows, op.groups, device="cuda"), torch.empty_like(x)
    op.forward_8bit(x, w.cuda(), q, scale, None, res, total)
    s = (x.float() + res.float()).to(x.dtype)
    assert torch.equal(total, s)
    ey, _ = formula(s, w, 1e-6)
    most, size = (448.0, group or cols) if out8 == "e4m3" else (127.0, group or cols)
    parts = ey.split(size, 1)
    # the definition's smallest scale: a group of one column may hold a sum of zero
    top = torch.stack([p.abs().amax(1) for p in parts], 1)
    escale = top.clamp(min=2.0**-100) / most
    assert ((scale.double().cpu() / escale - 1).abs() <= NORM + 2 * EPS32).all()
    got, by = values(q, out8), scale.double().cpu().repeat_interleave(size, 1)[:, :cols]
    # y / scale is off by y's error, the division's and the product's, then rounded to
    # nearest: by 2^-4 of it, or half a step of 2^-9 below 2^-6, or half of one
    v = ey / by
    off = v.abs() * (NORM + 3 * EPS32)
    half = torch.clamp((v.abs() + off) * 2.0**-4, min=2.0**-10) if out8 == "e4m3" else torch.full_like(v, 0.5)
    assert ((got - v).abs() <= half + off).all()
    # the largest fills the range
    assert torch.equal(torch.stack([p.abs().amax(1) for p in got.split(size, 1)], 1), torch.where(top > 0, most, 0.0).double())
    assert (wide[:, 0] == 3).all() and (wide[:, cols + 1:] == 3).all()


@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_backward(gpu, rows, cols, dtype, add):
    g = torch.Generator().manual_seed(rows * 11 + cols)
    pad = (1, 0, 6)[(rows + cols) % 3]
    s, dy = rows_of(g, rows, cols, pad, dtype, 0.7), rows_of(g, rows, cols, pad, dtype, 0.5)
    dt = rows_of(g, rows, cols, pad + 1, dtype, 0.5) if add else None
    w = 1 + 0.2 * torch.randn(cols, generator=g)
    rstd = formula(s, w, 1e-6)[1].float().cuda()
    dx, beside = inside(rows, cols, dtype)
    dw = torch.full((cols,), 7.0, device="cuda")
    ops.RMSNorm(cols, dtype).backward(dy, s, w.cuda(), rstd, dx, dw, dt)
    s64, d64, r64 = s.double().cpu(), dy.double().cpu(), rstd.double().cpu()[:, None]
    h, gr = s64 * r64, d64 * w.double()
    c = (gr * h).mean(1, keepdim=True)
    edx = r64 * (gr - h * c) + (dt.double().cpu() if add else 0.0)
    size = gr.abs() + 3 * h.abs() * (gr * h).abs().mean(1, keepdim=True)
    tol = (UNIT[dtype] + EPS32) * edx.abs() + TINY[dtype] + r64 * 64 * EPS32 * size
    assert ((dx.double().cpu() - edx).abs() <= tol).all()
    # chains: rows of a workgroup's wave, 4 waves, 32 partial sums of a column, 16 of them
    chain = rows // 512 + 64
    assert ((dw.double().cpu() - (d64 * h).sum(0)).abs() <= chain * EPS32 * (d64 * h).abs().sum(0) + 1e-30).all()
    assert beside()


def test_gradient_against_differences(gpu):
    """The kernel's own forward, moved along a direction, changes as its gradient says."""
    g = torch.Generator().manual_seed(5)
    rows, cols, step = 6, 300, 2.0**-6
    x, v, dy = (torch.randn(rows, cols, generator=g).double() for _ in range(3))
    w, vw = (torch.randn(cols, generator=g).double() for _ in range(2))
    op = ops.RMSNorm(cols)

    def value(t):
        y = torch.empty(rows, cols, device="cuda")
        op.forward((x + t * v).float().cuda(), (w + t * vw).float().cuda(), y)
        return float((y.double().cpu() * dy).sum())

    def exact_value(t):
        return float((formula(x + t * v, w + t * vw, 1e-6)[0] * dy).sum())

    y, rstd = torch.empty(rows, cols, device="cuda"), torch.empty(rows, device="cuda")
    op.forward(x.float().cuda(), w.float().cuda(), y, rstd)
    dx, dw = torch.empty(rows, cols, device="cuda"), torch.empty(cols, device="cuda")
    op.backward(dy.float().cuda(), x.float().cuda(), w.float().cuda(), rstd, dx, dw)
    along = float((dx.double().cpu() * v).sum() + (dw.double().cpu() * vw).sum())
    seen = (value(step) - value(-step)) / (2 * step)
    # the difference's own truncation, from 64 bits at half the step (a third of what halving changes,
    # taken whole), and the rounding of x, w and y by 2^-24 of their sizes
    cut = abs((exact_value(step) - exact_value(-step)) / (2 * step)
              - (exact_value(step / 2) - exact_value(-step / 2)) / step) * 2
    rounding = 64 * EPS32 * float((y.double().cpu().abs() * dy.abs()).sum()) / step
    assert abs(seen - along) <= cut + rounding


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(7, 3), (2050, 1537), (1100, 1536), (5, 6145), (3, 20001)])
def test_in_place(gpu, rows, cols, dtype):
    """The sum into the residual or x, the gradient into the sum's own."""
    g = torch.Generator().manual_seed(cols)
    x, res, dy, dt = (rows_of(g, rows, cols, 4, dtype) for _ in range(4))
    w = torch.randn(cols, generator=g).cuda()
    op = ops.RMSNorm(cols, dtype)
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


def test_without_weight_statistics_and_sum(gpu):
    g = torch.Generator().manual_seed(1)
    x, r = torch.randn(37, 130, generator=g).cuda(), torch.randn(37, 130, generator=g).cuda()
    y, z, dx, full = (torch.empty_like(x) for _ in range(4))
    one, dw, rstd = torch.ones(130, device="cuda"), torch.empty(130, device="cuda"), torch.empty(37, device="cuda")
    op = ops.RMSNorm(130, eps=1e-3)
    op.forward(x, None, y, residual=r)
    op.forward(x + r, one, z, rstd)
    assert torch.equal(y, z)
    op.backward(x, x + r, None, rstd, dx)
    op.backward(x, x + r, one, rstd, full, dw)
    assert torch.equal(dx, full)


def test_no_rows(gpu):
    op = ops.RMSNorm(50, group=32)
    none, z = torch.empty(0, 50, device="cuda"), torch.empty(0, device="cuda")
    op.forward(none, None, none, z, none, none)
    op.forward_8bit(none, None, none.to(torch.float8_e4m3fn), torch.empty(0, 2, device="cuda"))
    dw = torch.ones(50, device="cuda")
    op.backward(none, none, None, z, none, dw)
    assert not dw.any()


@pytest.mark.parametrize("out8", ["e4m3", "i8"])
def test_special_values(gpu, out8):
    x = torch.zeros(5, 700)
    x[1, 5] = float("nan")
    x[2, 600] = float("inf")
    x[3] = torch.randn(700, generator=torch.Generator().manual_seed(0)) * 1e-30
    x[4] = torch.randn(700, generator=torch.Generator().manual_seed(0)) * 1e15
    x = x.cuda()
    y = torch.empty_like(x)
    op = ops.RMSNorm(700, eps=0.0, out8=out8, group=128)
    op.forward(x, None, y)
    assert torch.isnan(y[0]).all() and torch.isnan(y[1]).all()  # no spread and no eps: 0 / 0
    assert torch.isnan(y[2, 600]) and (y[2, :600] == 0).all()
    assert torch.isnan(y[3]).sum() == 0  # squares below the smallest number: infinity times a number
    ey, _ = formula(x[4:], torch.ones(700), 0.0)
    assert ((y[4].double().cpu() - ey[0]).abs() <= (UNIT["f32"] + NORM) * ey[0].abs()).all()
    q = torch.empty(5, 700, dtype=torch.float8_e4m3fn if out8 == "e4m3" else torch.int8, device="cuda")
    scale = torch.empty(5, 6, device="cuda")
    op.forward_8bit(x, None, q, scale)
    assert torch.isnan(scale[:2]).all() and not values(q, out8)[:2].any()
    assert torch.isnan(scale[2, 4]) and (scale[2, :4] == scale[2, 5]).all() and not values(q, out8)[2].any()
    op = ops.RMSNorm(700, eps=1e-6, out8=out8, group=128)
    op.forward_8bit(x, None, q, scale)
    assert not values(q, out8)[0].any() and (scale[0] > 0).all() and torch.isfinite(scale[0]).all()


def test_more_rows_than_a_grid_holds(gpu):
    """2^20 workgroups of four rows, and some."""
    rows = 4 * (1 << 20) + 1003
    x = torch.randn(rows, 5, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    y = torch.empty_like(x)
    ops.RMSNorm(5).forward(x, None, y)
    x64 = x.double()
    e = x64 / torch.sqrt((x64 * x64).mean(1, keepdim=True) + 1e-6)
    assert ((y.double() - e).abs() <= (UNIT["f32"] + NORM) * e.abs()).all()


def test_same_result_every_time(gpu):
    g = torch.Generator().manual_seed(2)
    s, dy = torch.randn(5000, 384, generator=g).cuda(), torch.randn(5000, 384, generator=g).cuda()
    rstd = 1 / s.std(1)
    out = []
    for _ in range(3):
        dx, dw = torch.empty_like(s), torch.empty(384, device="cuda")
        ops.RMSNorm(384).backward(dy, s, None, rstd, dx, dw)
        out.append((dx, dw))
    assert all(torch.equal(a, b) for o in out[1:] for a, b in zip(out[0], o))
