"""Bucket rows and embedding where a wave looks after many rows without a choice, and where
a launch takes more than one turn.  Moves are copies: equal."""
import pytest
import torch

from tatara_amd import ops
from test_gpu_bucket_rows import TYPES, choices, placed

pytestmark = pytest.mark.gpu

# from 4097 rows on a wave looks at two of them, above 262144 at 64: positions, choices, buckets, room
SPARSE = [(9001, 2, 9, None), (5000, 1, 9, 2222), (20003, 3, 64, 1500), (131, 2, 1000, 301), (300001, 1, 9, None),
          (70001, 4, 7, 60007)]


@pytest.mark.parametrize("dtype,cols", [("f32", 1), ("f32", 100), ("f16", 16), ("bf16", 257), ("bf16", 3)])
@pytest.mark.parametrize("n,k,e,room", SPARSE)
def test_rows_without_a_choice_are_zeros(gpu, n, k, e, room, dtype, cols):
    g = torch.Generator().manual_seed(n + cols)
    bucket = choices(g, n, k, e, 0.5)
    bucket[n // 2:n // 2 + 500] = -1  # and a stretch of positions that have none at all
    slot, source, _ = (t.cuda() for t in placed(bucket, e, room))
    op = ops.BucketRows(e, cols, k, dtype, room)
    m = op.rows(n)
    assert m > 4096 and (source < 0).any()
    x = torch.randn(n, cols, generator=g).to(TYPES[dtype]).cuda()
    wide = torch.full((m, cols + 3), 7.0, dtype=TYPES[dtype], device="cuda")
    op.gather(x, slot, source, wide[:, 1:cols + 1])
    want = torch.where(source[:, None] >= 0, x[(source.clamp(min=0) // k).long()], 0.0).to(x.dtype)
    assert torch.equal(wide[:, 1:cols + 1], want)
    assert (wide[:, 0] == 7.0).all() and (wide[:, cols + 1:] == 7.0).all()
    gate, dgate = torch.rand(n, k, generator=g).cuda(), torch.empty(n, k, device="cuda")
    by = gate.view(-1)[source.clamp(min=0).long()][:, None]
    want = torch.where(source[:, None] >= 0, by * x[(source.clamp(min=0) // k).long()].float(), 0.0).to(x.dtype)
    wide.fill_(7.0)
    op.combine_backward(x, want, slot, source, gate, wide[:, 1:cols + 1], dgate)
    assert torch.equal(wide[:, 1:cols + 1], want)
    assert (wide[:, 0] == 7.0).all() and (wide[:, cols + 1:] == 7.0).all()
    assert not dgate[slot < 0].any()


def test_more_positions_than_a_grid_holds(gpu):
    """2^20 workgroups of 256 positions, and some, there and back."""
    n = (1 << 28) + 12345
    bucket = (torch.arange(n, dtype=torch.int32, device="cuda") % 5 - 1).view(n, 1)  # every fifth has none
    op = ops.BucketRows(4, 1, 1, "bf16")
    slot, source, offset = (torch.full(s, 77, dtype=torch.int32, device="cuda") for s in ((n, 1), (n,), (5,)))
    op.sort(bucket, slot, source, offset)
    none = (n + 4) // 5
    count = [(n + 4 - e - 1) // 5 for e in range(4)]
    assert offset.tolist() == [sum(count[:e]) for e in range(5)] and sum(count) == n - none
    assert (source[n - none:] == -1).all() and (slot[bucket < 0] == -1).all()
    for e in range(4):  # bucket e's positions in order
        at = source[int(offset[e]):int(offset[e + 1])]
        assert (at == torch.arange(e + 1, n, 5, dtype=torch.int32, device="cuda")).all()
    x = (torch.arange(n, device="cuda", dtype=torch.int32) % 251 + 1).to(torch.bfloat16).view(n, 1)
    rows, back = torch.full_like(x, 7.0), torch.full_like(x, 7.0)
    op.gather(x, slot, source, rows)
    assert (rows[n - none:] == 0).all()
    op.gather_backward(rows, slot, back)
    assert torch.equal(back, torch.where(bucket < 0, 0.0, x).to(x.dtype))


@pytest.mark.parametrize("n", [200, 5000])
def test_more_rows_of_a_table_than_a_grid_clears(gpu, n):
    """2^20 workgroups of 128 rows, twice: with the sort and without it."""
    v = 1 << 28
    g = torch.Generator().manual_seed(n)
    token = torch.randint(0, v, (n,), generator=g, dtype=torch.int32)
    token[:4] = torch.tensor([0, v - 1, v, v // 2])
    token[-1] = v - 1
    dy = torch.randn(n, 1, generator=g)
    d = torch.full((v, 1), 7.0, device="cuda")
    ops.Embedding(v, 1, n).backward(dy.cuda(), token.cuda(), d)
    at, inverse = token[token < v].long().unique(return_inverse=True)
    want = torch.zeros(len(at), dtype=torch.float64).index_add_(0, inverse, dy[token < v, 0].double())
    size = torch.zeros(len(at), dtype=torch.float64).index_add_(0, inverse, dy[token < v, 0].double().abs())
    times = torch.bincount(inverse)
    got = d[at.cuda(), 0].double().cpu()
    assert ((got - want).abs() <= (times + 1) * 2.0**-24 * size).all()
    d[at.cuda()] = 0.0
    assert not d.any()
