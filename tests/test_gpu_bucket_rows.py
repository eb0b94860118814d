"""Rows by bucket and back on the GPU.  Places are whole numbers and gathered rows copies:
equal, as are products, rounded in f32 and then to the type.  Sums are f32, a choice or a column
after the other."""
import numpy as np
import pytest
import torch

from tatara_amd import ops

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}
TINY = {"f32": 0.0, "f16": 2.0**-25, "bf16": 0.0}
EPS32 = 2.0**-24
# (positions, top_k, buckets): one workgroup and many, one bucket and the most, sixteen choices
PLACES = [(0, 1, 9), (1, 1, 1), (1, 2, 8), (63, 1, 9), (64, 3, 9), (65, 4, 64), (1000, 16, 1024), (8192, 1, 9),
          (8193, 1, 9), (16381, 4, 64), (65536, 1, 9), (70001, 2, 1024), (40000, 16, 300), (300000, 1, 1)]


def choices(g, n, k, e, masked=0.1):
    """Distinct buckets a position would be a gate's; here any, with some that are none."""
    b = torch.randint(0, e, (n, k), generator=g, dtype=torch.int32)
    none = torch.rand(n, k, generator=g) < masked
    b[none] = torch.tensor([-1, e, 2**31 - 1, -2**31], dtype=torch.int32)[torch.randint(0, 4, (int(none.sum()),), generator=g)]
    return b


def placed(bucket, e, capacity):
    """slot, source and offset in numpy."""
    b = bucket.numpy().reshape(-1).astype(np.int64)
    rows = len(b) if capacity is None else e * capacity
    slot, source = np.full(len(b), -1, np.int32), np.full(rows, -1, np.int32)
    order = np.argsort(b, kind="stable")
    order = order[(b[order] >= 0) & (b[order] < e)]
    offset = np.concatenate([[0], np.bincount(b[order], minlength=e).cumsum()])
    rank = np.arange(len(order)) - offset[b[order]]
    fits = np.full(len(order), True) if capacity is None else rank < capacity
    row = np.arange(len(order)) if capacity is None else b[order] * capacity + rank
    slot[order[fits]], source[row[fits]] = row[fits], order[fits]
    return torch.from_numpy(slot.reshape(bucket.shape)), torch.from_numpy(source), torch.from_numpy(offset.astype(np.int32))


def whole(*shape):
    return torch.full(shape, 77, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("capacity", [None, 1, "less", "more"])
@pytest.mark.parametrize("n,k,e", PLACES)
def test_sort(gpu, n, k, e, capacity):
    g = torch.Generator().manual_seed(n + k)
    room = dict(less=max(1, n * k // (2 * e)), more=n * k // e + 37).get(capacity, capacity)
    bucket = choices(g, n, k, e)
    op = ops.BucketRows(e, 8, k, capacity=room)
    slot, source, offset = whole(n, k), whole(op.rows(n)), whole(e + 1)
    for _ in range(2):
        op.sort(bucket.cuda(), slot, source, offset)
        for got, want in zip((slot, source, offset), placed(bucket, e, room)):
            assert torch.equal(got.cpu(), want)


def test_sort_of_few_and_no_choices(gpu):
    for b in (torch.full((20000, 1), -1, dtype=torch.int32), torch.full((20000, 1), 5, dtype=torch.int32)):
        op = ops.BucketRows(9, 8)
        slot, source, offset = whole(20000, 1), whole(20000), whole(10)
        op.sort(b.cuda(), slot, source, offset)
        for got, want in zip((slot, source, offset), placed(b, 9, None)):
            assert torch.equal(got.cpu(), want)


def rows_of(g, rows, cols, pad, dtype):
    return torch.randn(rows, cols + pad, generator=g).to(TYPES[dtype]).cuda()[:, pad // 2:pad // 2 + cols]


MOVES = [(1, 1, 1, 1), (1, 2, 8, 1536), (7, 3, 5, 3), (65, 4, 9, 7), (130, 1, 9, 64), (257, 2, 9, 100),
         (100, 5, 9, 257), (33, 16, 20, 1031), (1200, 1, 9, 1536), (20, 2, 4, 4100), (3, 3, 3, 32768), (900, 4, 64, 16)]


@pytest.mark.parametrize("capacity", [None, "less"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,k,e,cols", MOVES)
def test_moves(gpu, n, k, e, cols, dtype, capacity):
    g = torch.Generator().manual_seed(n * 3 + cols)
    pad = (0, 1, 6)[(n + cols) % 3]
    room = None if capacity is None else max(1, n * k * 2 // (3 * e))
    slot, source, _ = placed(choices(g, n, k, e), e, room)
    op = ops.BucketRows(e, cols, k, dtype, room)
    m = op.rows(n)
    S, R = slot.cuda(), source.cuda()
    # out
    x = rows_of(g, n, cols, pad, dtype)
    wide = torch.full((m, cols + 3), 7.0, dtype=TYPES[dtype], device="cuda")
    out = wide[:, 1:cols + 1]
    op.gather(x, S, R, out)
    want = torch.where(R[:, None] >= 0, x[(R.clamp(min=0) // k).long()], 0.0).to(x.dtype)
    assert torch.equal(out, want)
    assert (wide[:, 0] == 7.0).all() and (wide[:, cols + 1:] == 7.0).all()
    # back, in f64
    rows, gate = rows_of(g, m, cols, pad, dtype), torch.rand(n, k, generator=g).cuda()
    at = torch.where(S[:, :, None] >= 0, rows[S.clamp(min=0).long()].double(), 0.0)
    wide = torch.full((n, cols + 2), 7.0, dtype=TYPES[dtype], device="cuda")
    y = wide[:, 1:cols + 1]
    for w in (gate, None):
        if w is None:
            op.gather_backward(rows, S, y)
        else:
            op.combine(rows, S, w, y)
        terms = at if w is None else at * w.double()[:, :, None]
        tol = UNIT[dtype] * terms.sum(1).abs() + TINY[dtype] + 2 * k * EPS32 * terms.abs().sum(1)
        assert ((y.double() - terms.sum(1)).abs() <= tol).all()
    assert (wide[:, 0] == 7.0).all() and (wide[:, -1] == 7.0).all()
    # the gradient of that
    dy = rows_of(g, n, cols, pad, dtype)
    wide = torch.full((m, cols + 3), 7.0, dtype=TYPES[dtype], device="cuda")
    drows, dgate, only = wide[:, 1:cols + 1], torch.full_like(gate, 7.0), torch.empty(m, cols, dtype=x.dtype, device="cuda")
    op.combine_backward(dy, rows, S, R, gate, drows, dgate)
    flat = R.clamp(min=0).long()
    want = torch.where(R[:, None] >= 0, gate.view(-1)[flat][:, None] * dy[flat // k].float(), 0.0).to(x.dtype)
    assert torch.equal(drows, want)
    assert (wide[:, 0] == 7.0).all() and (wide[:, cols + 1:] == 7.0).all()
    terms = at * dy.double()[:, None, :]
    # a lane's values of a row, then the lanes
    assert ((dgate.double() - terms.sum(2)).abs() <= (-(-cols // 64) + 14) * EPS32 * terms.abs().sum(2)).all()
    op.combine_backward(dy, None, S, R, gate, only)
    assert torch.equal(only, drows)


def test_choices_without_a_row_add_nothing_whatever_they_hold(gpu):
    op = ops.BucketRows(2, 20, 2)
    slot = torch.tensor([[0, -1], [-1, -1], [3, 1]], dtype=torch.int32, device="cuda")
    source = torch.tensor([0, 5, -1, 4, -1, -1], dtype=torch.int32, device="cuda")
    nan = float("nan")
    rows = torch.full((6, 20), nan, device="cuda")
    rows[0], rows[1], rows[3] = 1.0, 2.0, 3.0
    gate = torch.tensor([[0.5, nan], [nan, nan], [0.25, 2.0]], device="cuda")
    y, dgate, drows = torch.empty(3, 20, device="cuda"), torch.empty(3, 2, device="cuda"), torch.full_like(rows, nan)
    op.combine(rows, slot, gate, y)
    assert torch.equal(y[:, 0].cpu(), torch.tensor([0.5, 0.0, 4.75]))
    dy = torch.ones(3, 20, device="cuda")
    dy[1] = nan
    op.combine_backward(dy, rows, slot, source, gate, drows, dgate)
    assert torch.equal(dgate.cpu(), torch.tensor([[20.0, 0.0], [0.0, 0.0], [60.0, 40.0]]))
    assert torch.equal(drows[:, 0].cpu(), torch.tensor([0.5, 2.0, 0.0, 0.25, 0.0, 0.0]))


def test_slots_and_sources_out_of_range_are_none(gpu):
    """What a program's mistake may put there is neither read nor written at."""
    op = ops.BucketRows(3, 40, 1)
    big = 2**31 - 1
    slot = torch.tensor([[0], [4], [big], [-2**31]], dtype=torch.int32, device="cuda")
    source = torch.tensor([0, 4, big, -5], dtype=torch.int32, device="cuda")
    x, y, out = torch.ones(4, 40, device="cuda"), torch.empty(4, 40, device="cuda"), torch.full((4, 40), 7.0, device="cuda")
    op.gather(x, slot, source, out)
    assert out[:, 0].tolist() == [1.0, 0.0, 0.0, 0.0]
    op.gather_backward(x, slot, y)
    assert y[:, 0].tolist() == [1.0, 0.0, 0.0, 0.0]


def test_no_positions(gpu):
    op = ops.BucketRows(3, 16, 2, capacity=4)
    none, z = torch.empty(0, 16, device="cuda"), torch.empty(0, 2, device="cuda")
    slot, source, offset = whole(0, 2), whole(12), whole(4)
    op.sort(slot, slot, source, offset)
    assert (source == -1).all() and not offset.any()
    rows = torch.full((12, 16), 7.0, device="cuda")
    op.gather(none, slot, source, rows)
    assert not rows.any()
    rows.fill_(7.0)
    op.combine_backward(none, rows, slot, source, z, rows, z)
    assert not rows.any()
    op.combine(rows, slot, z, none)
    packed = ops.BucketRows(3, 16, 2)
    packed.sort(slot, slot, whole(0), offset)
    packed.gather(none, slot, whole(0), none)
    packed.combine_backward(none, none, slot, whole(0), z, none, z)


def test_offsets_beyond_32_bits(gpu):
    """Rows of more than 2^32 bytes and 2^31 values, there and back."""
    n, cols = 70000, 32768
    op = ops.BucketRows(2, cols, 1, "bf16")
    bucket = (torch.arange(n, dtype=torch.int32) % 2).view(n, 1).cuda()
    slot, source, offset = whole(n, 1), whole(n), whole(3)
    op.sort(bucket, slot, source, offset)
    x = (torch.arange(n, device="cuda") % 251).to(torch.bfloat16).view(n, 1).expand(n, cols).contiguous()
    out, back = torch.empty_like(x), torch.empty_like(x)
    op.gather(x, slot, source, out)
    assert torch.equal(out[:, 7], x[source.long(), 7]) and torch.equal(out[:, -1], x[source.long(), -1])
    op.gather_backward(out, slot, back)
    assert torch.equal(back, x)
