"""Layer norm on the GPU against its formulas in 64 bits.

Tolerances follow from the arithmetic: sums are f32 in chains of at most 32
values a lane, 6 shuffles, 16 waves (64 roundings of the summed magnitudes bound
them), and the result is rounded once to the element type.
"""
import numpy as np
import pytest
import torch

from tatara_amd import ops
from tatara_amd.runtime import Event, Stream
from tatara_amd.trainer import DeviceArray

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}  # half an ulp, relative
TINY = {"f32": 0.0, "f16": 2.0**-25, "bf16": 0.0}  # half an ulp of subnormals
EPS32 = 2.0**-24

SHAPES = [(1, 1), (1, 1536), (3, 7), (5, 64), (2, 65), (70, 256), (33, 257), (9, 770), (2100, 96), (2049, 513),
          (4, 2049), (3, 4100), (2, 8193), (2, 32768), (2050, 2048)]
# either side of the widths where more waves share a row
SHAPES += [(1100, 1024), (1100, 1025), (1100, 1536), (1100, 1537), (3, 6144), (3, 6145), (3, 7000), (2, 8192), (2, 16385)]


def rows_of(g, rows, cols, pad, dtype, scale=1.0, shift=0.0):
    x = (torch.randn(rows, cols + pad, generator=g) * scale + shift).to(TYPES[dtype])
    return x.cuda()[:, pad // 2:pad // 2 + cols]


def formula(x, w, b, eps):
    x = x.double().cpu()
    mean = x.mean(1)
    rstd = 1.0 / torch.sqrt(((x - mean[:, None]) ** 2).mean(1) + eps)
    return (x - mean[:, None]) * rstd[:, None] * w + b, mean, rstd


def forward_tolerance(x, w, b, mean, rstd, y, dtype):
    x = x.double().cpu()
    h = ((x - mean[:, None]) * rstd[:, None]).abs()
    size = x.abs().mean(1, keepdim=True) * rstd[:, None]
    return UNIT[dtype] * y.abs() + TINY[dtype] + 64 * EPS32 * (w.abs() * (size + 2 * h) + b.abs())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward(gpu, rows, cols, dtype):
    g = torch.Generator().manual_seed(rows * 7 + cols)
    pad = (0, 1, 6)[(rows + cols) % 3]
    x = rows_of(g, rows, cols, pad, dtype, 0.7, 0.3)
    w, b = 1 + 0.2 * torch.randn(cols, generator=g), 0.1 * torch.randn(cols, generator=g)
    wide = torch.full((rows, cols + 3), 7.0, dtype=TYPES[dtype], device="cuda")
    y = wide[:, 1:cols + 1]
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    ops.LayerNorm(cols, dtype, 1e-5).forward(x, w.cuda(), b.cuda(), y, mean, rstd)
    ey, em, er = formula(x, w.double(), b.double(), 1e-5)
    tol = forward_tolerance(x, w.double(), b.double(), em, er, ey, dtype)
    assert ((y.double().cpu() - ey).abs() <= tol).all()
    assert ((mean.double().cpu() - em).abs() <= 64 * EPS32 * x.double().cpu().abs().mean(1)).all()
    # rstd's error: half that of the variance, whose deviations carry the mean's error squared at most
    assert ((rstd.double().cpu() / er - 1).abs() <= 64 * EPS32 * (1 + (em * er) ** 2 * 64 * EPS32)).all()
    rest = torch.cat([wide[:, :1], wide[:, cols + 1:]], 1)
    assert (rest == 7.0).all(), "values beside the rows were written"


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_backward(gpu, rows, cols, dtype):
    g = torch.Generator().manual_seed(rows * 11 + cols)
    pad = (1, 0, 6)[(rows + cols) % 3]
    x, dy = rows_of(g, rows, cols, pad, dtype, 0.7, 0.3), rows_of(g, rows, cols, pad, dtype, 0.5)
    w = 1 + 0.2 * torch.randn(cols, generator=g)
    _, em, er = formula(x, w.double(), 0.0, 1e-5)
    mean, rstd = em.float().cuda(), er.float().cuda()
    wide = torch.full((rows, cols + 2), 7.0, dtype=TYPES[dtype], device="cuda")
    dx = wide[:, 1:cols + 1]
    dw, db = torch.full((cols,), 7.0, device="cuda"), torch.full((cols,), 7.0, device="cuda")
    ops.LayerNorm(cols, dtype).backward(dy, x, w.cuda(), mean, rstd, dx, dw, db)
    x64, d64, w64 = x.double().cpu(), dy.double().cpu(), w.double()
    m64, r64 = mean.double().cpu()[:, None], rstd.double().cpu()[:, None]
    h, gr = (x64 - m64) * r64, d64 * w64
    a, c = gr.mean(1, keepdim=True), (gr * h).mean(1, keepdim=True)
    edx = r64 * (gr - a - h * c)
    h_off = 2 * EPS32 * (x64.abs() + m64.abs()) * r64  # rounding of h itself
    size = gr.abs() + gr.abs().mean(1, keepdim=True) + 2 * h.abs() * (gr * h).abs().mean(1, keepdim=True)
    tol = UNIT[dtype] * edx.abs() + TINY[dtype] + r64 * (
        64 * EPS32 * size + h_off * c.abs() + h.abs() * (gr.abs() * h_off).mean(1, keepdim=True))
    assert ((dx.double().cpu() - edx).abs() <= tol).all()
    # chains: rows of a workgroup's wave, 4 waves, 32 partial sums of a column, 16 of them
    chain = rows // 512 + 64
    assert ((dw.double().cpu() - (d64 * h).sum(0)).abs()
            <= chain * EPS32 * (d64 * h).abs().sum(0) + (d64.abs() * h_off).sum(0) + 1e-30).all()
    assert ((db.double().cpu() - d64.sum(0)).abs() <= chain * EPS32 * d64.abs().sum(0)).all()
    assert (wide[:, 0] == 7.0).all() and (wide[:, -1] == 7.0).all()


def test_gradient_against_differences(gpu):
    """The kernel's own forward, moved along a direction, changes as its gradient says."""
    g = torch.Generator().manual_seed(5)
    rows, cols, step = 6, 300, 2.0**-6
    x, v, dy = (torch.randn(rows, cols, generator=g, dtype=torch.float64) for _ in range(3))
    x, v, dy = x.float().double(), v.float().double(), dy.float().double()
    w, vw, vb = (torch.randn(cols, generator=g).double() for _ in range(3))
    b = torch.zeros(cols, dtype=torch.float64)
    ln = ops.LayerNorm(cols)

    def value(t):
        y = torch.empty(rows, cols, device="cuda")
        ln.forward((x + t * v).float().cuda(), (w + t * vw).float().cuda(), (b + t * vb).float().cuda(), y)
        return float((y.double().cpu() * dy).sum())

    def exact_value(t):
        y, _, _ = formula(x + t * v, w + t * vw, b + t * vb, 1e-5)
        return float((y * dy).sum())

    y, mean, rstd = (torch.empty(rows, cols, device="cuda"), torch.empty(rows, device="cuda"),
                     torch.empty(rows, device="cuda"))
    ln.forward(x.float().cuda(), w.float().cuda(), b.float().cuda(), y, mean, rstd)
    dx, dw, db = (torch.empty(rows, cols, device="cuda"), torch.empty(cols, device="cuda"),
                  torch.empty(cols, device="cuda"))
    ln.backward(dy.float().cuda(), x.float().cuda(), w.float().cuda(), mean, rstd, dx, dw, db)
    along = float((dx.double().cpu() * v).sum() + (dw.double().cpu() * vw).sum() + (db.double().cpu() * vb).sum())
    seen = (value(step) - value(-step)) / (2 * step)
    # the difference's own truncation, from 64 bits at half the step (a third of what halving changes,
    # taken whole), and the rounding of x, w and y by 2^-24 of their sizes
    cut = abs((exact_value(step) - exact_value(-step)) / (2 * step)
              - (exact_value(step / 2) - exact_value(-step / 2)) / step) * 2
    rounding = 64 * EPS32 * float((y.double().cpu().abs() * dy.abs()).sum()) / step
    assert abs(seen - along) <= cut + rounding


def test_without_parameters_and_statistics(gpu):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(37, 130, generator=g).cuda()
    y, dx = torch.empty_like(x), torch.empty_like(x)
    ln = ops.LayerNorm(130, eps=1e-3)
    ln.forward(x, None, None, y)
    one = torch.ones(130, dtype=torch.float64)
    ey, em, er = formula(x, one, 0 * one, 1e-3)
    assert ((y.double().cpu() - ey).abs() <= forward_tolerance(x, one, 0 * one, em, er, ey, "f32")).all()
    mean, rstd = em.float().cuda(), er.float().cuda()
    full, dw, db = torch.empty_like(x), torch.empty(130, device="cuda"), torch.empty(130, device="cuda")
    ln.backward(x, x, None, mean, rstd, dx)
    ln.backward(x, x, torch.ones(130, device="cuda"), mean, rstd, full, dw, db)
    assert torch.equal(dx, full)
    only = torch.empty_like(db)
    ln.backward(x, x, None, mean, rstd, dx, None, only)
    assert torch.equal(only, db)


def test_more_rows_than_a_grid_holds(gpu):
    """2^20 workgroups of four rows, and some."""
    rows = 4 * (1 << 20) + 1003
    x = torch.randn(rows, 5, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    y, mean = torch.empty_like(x), torch.empty(rows, device="cuda")
    ops.LayerNorm(5).forward(x, None, None, y, mean)
    x64 = x.double()
    em = x64.mean(1, keepdim=True)
    er = 1 / torch.sqrt(((x64 - em) ** 2).mean(1, keepdim=True) + 1e-5)
    h = (x64 - em) * er
    tol = 2.0**-24 * h.abs() + 64 * EPS32 * (x64.abs().mean(1, keepdim=True) * er + 2 * h.abs())
    assert ((y.double() - h).abs() <= tol).all()


def test_no_rows(gpu):
    ln = ops.LayerNorm(50)
    none, z = torch.empty(0, 50, device="cuda"), torch.empty(0, device="cuda")
    ln.forward(none, None, None, none, z, z)
    dw, db = torch.ones(50, device="cuda"), torch.ones(50, device="cuda")
    ln.backward(none, none, None, z, z, none, dw, db)
    assert not dw.any() and not db.any()


def test_constant_rows_and_special_values(gpu):
    x = torch.full((4, 700), 3.0)
    x[1, 5] = float("nan")
    x[2, 6] = float("inf")
    x[3] = torch.randn(700, generator=torch.Generator().manual_seed(0)) * 1e15
    y, mean, rstd = torch.empty(4, 700, device="cuda"), torch.empty(4, device="cuda"), torch.empty(4, device="cuda")
    b = torch.randn(700)
    ops.LayerNorm(700).forward(x.cuda(), None, b.cuda(), y, mean, rstd)
    assert torch.equal(y[0].cpu(), b) and float(mean[0]) == 3.0  # no spread: the bias alone
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all()
    ey, _, _ = formula(x[3:], torch.ones(700).double(), b.double(), 1e-5)
    assert ((y[3].double().cpu() - ey[0]).abs() <= 1e-4).all()  # values to 4, 64 roundings each


def test_same_result_every_time(gpu):
    g = torch.Generator().manual_seed(2)
    x, dy = torch.randn(5000, 384, generator=g).cuda(), torch.randn(5000, 384, generator=g).cuda()
    mean, rstd = x.mean(1), 1 / x.std(1)
    out = []
    for _ in range(3):
        dx, dw, db = torch.empty_like(x), torch.empty(384, device="cuda"), torch.empty(384, device="cuda")
        ops.LayerNorm(384).backward(dy, x, None, mean, rstd, dx, dw, db)
        out.append((dx, dw, db))
    assert all(torch.equal(a, b) for o in out[1:] for a, b in zip(out[0], o))


def test_library_arrays_and_own_stream(gpu):
    """DeviceArray operands (bf16 as uint16), on a stream of the caller's that waits for its inputs."""
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.standard_normal((40, 96)).astype(np.float32)).bfloat16()
    X = DeviceArray(x.view(torch.uint16).numpy())
    Y = DeviceArray.empty((40, 96), np.uint16)
    M, R = DeviceArray.empty((40,), np.float32), DeviceArray.empty((40,), np.float32)
    ready = Event()
    ready.record(None)
    ln = ops.LayerNorm(96, "bf16")
    with Stream() as s:
        s.wait(ready)
        ln.forward(X, None, None, Y, M, R, stream=s)
        s.synchronize()
    one = torch.ones(96, dtype=torch.float64)
    ey, em, er = formula(x, one, 0 * one, 1e-5)
    y = torch.from_numpy(Y.to_host()).view(torch.bfloat16).double()
    assert ((y - ey).abs() <= forward_tolerance(x, one, 0 * one, em, er, ey, "bf16")).all()


def test_another_stream_gives_the_same(gpu):
    g = torch.Generator().manual_seed(8)
    x, w = torch.randn(300, 200, generator=g).cuda(), torch.rand(200, generator=g).cuda() + 0.5
    ln = ops.LayerNorm(200)

    def step(stream):
        out = [torch.empty_like(x), torch.empty(300, device="cuda"), torch.empty(300, device="cuda"),
               torch.empty_like(x), torch.empty(200, device="cuda"), torch.empty(200, device="cuda")]
        torch.cuda.synchronize()
        y, mean, rstd, dx, dw, db = out
        ln.forward(x, w, None, y, mean, rstd, stream=stream)
        ln.backward(y, x, w, mean, rstd, dx, dw, db, stream=stream)
        stream.synchronize() if stream else torch.cuda.synchronize()
        return out

    with Stream() as s:
        assert all(torch.equal(a, b) for a, b in zip(step(None), step(s)))
