"""A loss's gradient that has overflowed, as under a loss scale that is too large, reaches the
positions that count and no others."""
import math

import pytest
import torch

from tatara_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("share", [False, True])
@pytest.mark.parametrize("n,e,k", [(7, 9, 2), (300, 64, 4), (5, 1024, 1)])
def test_positions_that_do_not_count_get_zero(gpu, n, e, k, share):
    g = torch.Generator().manual_seed(n)
    l = torch.randn(n, e, generator=g)
    valid = (torch.arange(n) % 3 > 0).to(torch.uint8)
    l[1] = -math.inf  # counts as little as valid = 0
    l[3] = math.nan  # at a position that is left out
    op = ops.BucketGate(e, k, renormalise=share)
    o = (torch.empty(n, k, dtype=torch.int32, device="cuda"), torch.empty(n, k, device="cuda"),
         torch.empty(e, dtype=torch.int32, device="cuda"), torch.empty(e, device="cuda"),
         torch.empty(1, dtype=torch.int32, device="cuda"), torch.empty(1, device="cuda"))
    lg, vg = l.cuda(), valid.cuda()
    op.forward(lg, *o, valid=vg)
    out = valid == 0
    out[1] = True
    for dloss, dgate in ((math.inf, 1.0), (1.0, math.inf), (math.nan, math.nan)):
        d = torch.full((n, e), 7.0, device="cuda")
        op.backward(lg, o[0], o[2], o[4], d, torch.full((n, k), dgate, device="cuda"), dloss, valid=vg)
        d = d.cpu()
        assert (d[out] == 0.0).all(), (dloss, dgate)
        assert not torch.isfinite(d[~out]).all()
