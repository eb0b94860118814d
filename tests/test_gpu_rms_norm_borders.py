"""RMS norm where the squares leave f32's range, without an eps: what the header says of both
borders."""
import pytest
import torch

from tatara_amd import ops
from test_gpu_rms_norm import NORM

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [3, 40, 700, 9000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("out8", ["e4m3", "i8"])
def test_squares_at_the_ends_of_the_range(gpu, cols, dtype, out8):
    """2^-74 is the last power of two whose square f32 holds, as 2 units of its smallest; half a
    unit, 2^-150, rounds to 0.  (2^64)^2 passes the range at the other end."""
    sign = torch.where(torch.arange(cols, device="cuda") % 3 == 1, -1.0, 1.0)
    x = (sign * torch.tensor([2.0**-60, 2.0**-74, 2.0**-75, 2.0**-100, 2.0**50, 2.0**64], device="cuda")[:, None]).to(dtype)
    x = torch.cat([x, x[2:3]])
    x[-1, 0] = 0.0
    y, rstd = torch.empty_like(x), torch.empty(len(x), device="cuda")
    name = {torch.float32: "f32", torch.bfloat16: "bf16"}[dtype]
    op = ops.RMSNorm(cols, name, 0.0, out8, 64)
    op.forward(x, None, y, rstd)
    for r in (0, 1, 4):  # every sum of equal powers is one, or as near as one of other values
        assert ((y[r].float() * sign - 1.0).abs() <= NORM + (2.0**-24 if name == "f32" else 2.0**-8)).all()
    for r in (2, 3):
        assert torch.equal(y[r].float(), sign * float("inf"))
    assert torch.isinf(rstd[[2, 3, 6]]).all() and rstd[5] == 0
    assert not y[5].any()
    assert torch.isnan(y[6, 0]) and torch.equal(y[6, 1:].float(), sign[1:] * float("inf"))
    q = torch.full((len(x), cols), 3, device="cuda").to(torch.float8_e4m3fn if out8 == "e4m3" else torch.int8)
    scale = torch.empty(len(x), op.groups, device="cuda")
    op.forward_8bit(x, None, q, scale)
    q = q.float()
    assert torch.isnan(scale[[2, 3, 6]]).all() and not q[[2, 3, 5, 6]].any()
    most = 448.0 if out8 == "e4m3" else 127.0
    for r in (0, 1, 4):
        assert torch.equal(q[r], sign * most) and ((scale[r] * most - 1.0).abs() <= NORM + 2.0**-23).all()
    # the largest value of a row of zeros is taken as 2^-100
    assert ((scale[5] * most / 2.0**-100 - 1.0).abs() <= 2.0**-23).all()
