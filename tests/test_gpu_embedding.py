"""Embedding rows and the table's gradient on the GPU.  A row is one product, rounded once:
equal.  A gradient is an f32 sum in the positions' order, within its roundings of 64 bits."""
import pytest
import torch

from tatara_amd import ops

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS32 = 2.0**-24
# (positions, vocab, cols): one digit of the sort, two and three, one chunk and many
SHAPES = [(0, 5, 16), (1, 1, 1), (1, 73305, 64), (7, 3, 3), (9, 81, 7), (65, 9, 256), (300, 1023, 33),
          (500, 1024, 100), (3000, 1022, 770), (8192, 2, 16), (8193, 300, 30), (20000, 81, 64), (4099, 40000, 257),
          (30000, 1, 130), (50000, 2000000, 4), (2000, 9, 4100), (100000, 5, 5), (257, 81, 32768),
          (20000, 600000, 4), (40000, 200, 128), (128, 9, 100), (256, 5, 300), (255, 2, 16), (200, 30000, 1000)]


def rows_of(g, rows, cols, pad, dtype):
    return torch.randn(rows, cols + pad, generator=g).to(TYPES[dtype]).cuda()[:, pad // 2:pad // 2 + cols]


def tokens(g, n, v, kind):
    t = torch.randint(0, v, (n,), generator=g)
    if kind == "hot":  # half of the positions have one of them
        t[torch.rand(n, generator=g) < 0.5] = v // 2
    elif kind == "falling":
        t = (v ** torch.rand(n, generator=g, dtype=torch.float64)).long().clamp(max=v) - 1
    none = torch.rand(n, generator=g) < 0.02
    t[none] = torch.tensor([-1, v, 2**31 - 1, -2**31])[torch.randint(0, 4, (int(none.sum()),), generator=g)]
    return t.int()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,v,cols", SHAPES)
def test_forward(gpu, n, v, cols, dtype):
    g = torch.Generator().manual_seed(n + cols)
    pad = (0, 1, 6)[(n + cols) % 3]
    t, table = tokens(g, n, v, "any").cuda(), rows_of(g, v, cols, pad, dtype)
    wide = torch.full((n, cols + 3), 7.0, dtype=TYPES[dtype], device="cuda")
    y = wide[:, 1:cols + 1]
    known = (t >= 0) & (t < v)
    for scale in (5.25, 768.0**0.5):
        ops.Embedding(v, cols, n, dtype, scale).forward(t, table, y)
        want = table[torch.where(known, t, 0).long()].float() * scale
        assert torch.equal(y, torch.where(known[:, None], want, 0.0).to(TYPES[dtype]))
    assert (wide[:, :1] == 7.0).all() and (wide[:, cols + 1:] == 7.0).all()


@pytest.mark.parametrize("kind", ["any", "hot", "falling"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,v,cols", SHAPES)
def test_backward(gpu, n, v, cols, dtype, kind):
    g = torch.Generator().manual_seed(n + 3 * cols)
    pad = (1, 0, 6)[(n + cols) % 3]
    t, dy = tokens(g, n, v, kind), rows_of(g, n, cols, pad, dtype)
    op = ops.Embedding(v, cols, n + 5, dtype, 0.75)
    dtable = torch.full((v, cols), 7.0, device="cuda")
    op.backward(dy, t.cuda(), dtable)
    known = (t >= 0) & (t < v)
    at, d = t[known].long().cuda(), dy[known.cuda()].double()
    want = torch.zeros(v, cols, dtype=torch.float64, device="cuda").index_add_(0, at, 0.75 * d)
    size = torch.zeros(v, cols, dtype=torch.float64, device="cuda").index_add_(0, at, 0.75 * d.abs())
    count = torch.bincount(at, minlength=v)[:, None]
    # every addition of a token's rows and of its partial sums, and the product
    assert ((dtable.double() - want).abs() <= (count + 1) * EPS32 * size).all()
    again = torch.full((v, cols), 7.0, device="cuda")
    op.backward(dy, t.cuda(), again)
    assert torch.equal(again, dtable)


def test_gradient_is_the_forward_calls_transpose(gpu):
    """<E(table), dy> = <table, E'(dy)>, by the kernels alone: the look-up is linear."""
    g = torch.Generator().manual_seed(4)
    n, v, cols = 3000, 50, 40
    t, dy, table = tokens(g, n, v, "hot").cuda(), rows_of(g, n, cols, 0, "f32"), rows_of(g, v, cols, 0, "f32")
    op, y, d = ops.Embedding(v, cols, n, scale=3.0), torch.empty(n, cols, device="cuda"), torch.empty(v, cols, device="cuda")
    op.forward(t, table, y)
    op.backward(dy, t, d)
    a, b = float((y.double() * dy.double()).sum()), float((table.double() * d.double()).sum())
    assert abs(a - b) <= (n + 4) * EPS32 * float((y.double() * dy.double()).abs().sum())


def test_fewer_positions_than_it_is_made_for(gpu):
    g = torch.Generator().manual_seed(6)
    op = ops.Embedding(700, 48, 70000)
    for n in (70000, 8, 0, 9001, 70000):
        t, dy = tokens(g, n, 700, "any").cuda(), rows_of(g, n, 48, 0, "f32")
        d, e = torch.full((700, 48), 7.0, device="cuda"), torch.full((700, 48), 7.0, device="cuda")
        op.backward(dy, t, d)
        ops.Embedding(700, 48, n).backward(dy, t, e)
        assert torch.equal(d, e)
    with pytest.raises(ValueError, match="up to 70000"):
        op.backward(torch.empty(70001, 48, device="cuda"), torch.empty(70001, dtype=torch.int32, device="cuda"), d)


def test_special_values_stay_with_their_token(gpu):
    t = torch.tensor([3, 1, 3, 0, 1, -1], dtype=torch.int32, device="cuda")
    dy = torch.ones(6, 20, device="cuda")
    dy[1] = float("inf")
    dy[3] = float("nan")
    dy[5] = float("nan")
    d = torch.empty(5, 20, device="cuda")
    ops.Embedding(5, 20, 6).backward(dy, t, d)
    assert torch.isnan(d[0]).all() and torch.isinf(d[1]).all() and not d[2].any() and (d[3] == 2).all() and not d[4].any()


def test_offsets_beyond_32_bits(gpu):
    """A table's gradient of more than 2^31 values, a lookup in its last rows."""
    v, cols, n = 600000, 4096, 1000
    t = torch.arange(v - n, v, dtype=torch.int32, device="cuda").flip(0)
    dy = torch.arange(n, device="cuda").float().view(n, 1).expand(n, cols).contiguous()
    d = torch.full((v, cols), 7.0, device="cuda")
    op = ops.Embedding(v, cols, n)
    op.backward(dy, t, d)
    assert torch.equal(d[-n:], dy.flip(0)) and not d[:-n].any()
    y = torch.empty(n, cols, device="cuda")
    op.forward(t, d, y)
    assert torch.equal(y, dy)
