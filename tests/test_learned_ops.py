"""Refusals of the learned-choice and orthogonalisation operators: wrong shapes,
types, sizes and pointers are errors before any device call.  CPU only."""
import ctypes as C

import numpy as np
import pytest

from tatara_amd import _lib, ops

FAKE = 4096  # an address that a refused call never reads


class Fake:
    """Stands for a device tensor."""

    def __init__(self, shape, dtype="float32"):
        self.shape, self.dtype, self.ptr = tuple(shape), np.dtype(dtype), FAKE


def refused(status, part):
    assert status == -3 and part in _lib.load().tatara_last_error(), _lib.load().tatara_last_error()


def norm_forward(**k):
    a = dict(x=FAKE, xs=16, w=FAKE, b=FAKE, y=2 * FAKE, ys=16, mean=FAKE, rstd=FAKE, rows=4, cols=16, eps=1e-5, t=0)
    a.update(k)
    return _lib.load().tatara_op_layer_norm_forward(*a.values(), None)


def norm_backward(**k):
    a = dict(dy=FAKE, dys=16, x=FAKE, xs=16, w=FAKE, mean=FAKE, rstd=FAKE, dx=FAKE, dxs=16, dw=FAKE, db=FAKE, rows=4,
             cols=16, t=0, ws=FAKE, n=1 << 30)
    a.update(k)
    return _lib.load().tatara_op_layer_norm_backward(*a.values(), None)


def test_layer_norm_refuses():
    refused(norm_forward(t=3), b"element type")
    refused(norm_forward(cols=0), b"columns")
    refused(norm_forward(cols=32769, xs=40000, ys=40000), b"columns")
    refused(norm_forward(rows=1 << 31), b"rows")
    refused(norm_forward(eps=-1.0), b"eps")
    refused(norm_forward(eps=float("nan")), b"eps")
    refused(norm_forward(x=None), b"null")
    refused(norm_forward(xs=15), b"stride")
    refused(norm_forward(ys=-16), b"stride")
    refused(norm_forward(x=FAKE + 2), b"aligned")
    refused(norm_forward(y=FAKE + 1, t=1), b"aligned")
    refused(norm_backward(ws=None), b"workspace")
    refused(norm_backward(n=4 * 512 * 2 * 16 - 1), b"workspace")
    refused(norm_backward(dx=None), b"null")
    refused(norm_backward(mean=None), b"null")
    refused(norm_backward(dxs=3), b"stride")
    refused(norm_backward(ws=FAKE + 4), b"aligned")
    refused(_lib.load().tatara_op_layer_norm_backward_workspace(16, None), b"null")
    n = C.c_uint64()
    refused(_lib.load().tatara_op_layer_norm_backward_workspace(0, C.byref(n)), b"columns")


def gate_forward(**k):
    a = dict(l=FAKE, s=9, v=None, n=4, e=9, k=2, share=0, bal=0.01, t=0, bucket=FAKE, gate=FAKE, count=FAKE,
             prob=FAKE, counted=FAKE, loss=FAKE, ws=FAKE, wn=1 << 30)
    a.update(k)
    return _lib.load().tatara_op_bucket_gate_forward(*a.values(), None)


def gate_backward(**k):
    a = dict(l=FAKE, s=9, v=None, n=4, e=9, k=2, share=0, bal=0.01, t=0, bucket=FAKE, count=FAKE, counted=FAKE,
             dgate=FAKE, dloss=1.0, d=FAKE, ds=9)
    a.update(k)
    return _lib.load().tatara_op_bucket_gate_backward(*a.values(), None)


def test_bucket_gate_refuses():
    for call in (gate_forward, gate_backward):
        refused(call(t=-1), b"element type")
        refused(call(e=0), b"buckets")
        refused(call(e=1025, s=1025), b"buckets")
        refused(call(k=0), b"top_k")
        refused(call(k=10), b"top_k")
        refused(call(k=17, e=20, s=20), b"top_k")
        refused(call(n=1 << 30), b"positions")
        refused(call(l=None), b"null")
        refused(call(bucket=None), b"null")
        refused(call(s=8), b"stride")
        refused(call(l=FAKE + 1, t=2), b"aligned")
    refused(gate_forward(loss=None), b"null")
    refused(gate_forward(ws=None), b"workspace")
    refused(gate_forward(wn=100), b"workspace")
    refused(gate_backward(d=None), b"null")
    refused(gate_backward(ds=8), b"stride")


def ortho(**k):
    a = dict(x=FAKE, xr=6, xb=24, out=FAKE, orow=6, ob=24, batch=2, rows=4, cols=6, t=0, steps=5, ws=FAKE, n=1 << 40)
    a.update(k)
    return _lib.load().tatara_op_orthogonalise(*a.values(), None)


def muon(**k):
    a = dict(w=FAKE, m=FAKE, g=FAKE, batch=2, rows=4, cols=6, t=0, beta=0.9, nesterov=1, lr=0.1, decay=0.0, scale=1.0,
             lo=-1.0, hi=1.0, steps=5, ws=FAKE, n=1 << 40)
    a.update(k)
    return _lib.load().tatara_op_muon_step(*a.values(), None)


def test_orthogonalise_and_muon_refuse():
    for call in (ortho, muon):
        refused(call(t=9), b"element type")
        refused(call(rows=0), b"sides")
        refused(call(cols=32769), b"sides")
        refused(call(batch=65536), b"matrices")
        refused(call(steps=0), b"steps")
        refused(call(steps=33), b"steps")
        refused(call(ws=None), b"workspace")
        refused(call(n=64), b"workspace")
    refused(ortho(x=None), b"null")
    refused(ortho(xr=5), b"stride")
    refused(ortho(ob=23), b"stride")
    refused(ortho(xb=-1), b"stride")
    refused(ortho(out=FAKE + 1, t=1), b"aligned")
    refused(muon(w=None), b"null")
    refused(muon(beta=1.0), b"beta")
    refused(muon(beta=float("nan")), b"beta")
    refused(muon(lo=2.0), b"min_w")
    refused(muon(g=FAKE + 2), b"aligned")


def test_python_side_refuses():
    with pytest.raises(ValueError, match="dtype"):
        ops.LayerNorm(8, "f64")
    with pytest.raises(ValueError, match="cols"):
        ops.LayerNorm(0)
    with pytest.raises(ValueError, match="eps"):
        ops.LayerNorm(8, eps=float("nan"))
    ln = ops.LayerNorm(8)
    x = Fake((3, 8))
    with pytest.raises(ValueError, match="y must"):
        ln.forward(x, None, None, Fake((3, 9)))
    with pytest.raises(ValueError, match="x must"):
        ln.forward(Fake((3, 8), "float16"), None, None, x)
    with pytest.raises(ValueError, match="weight"):
        ln.forward(x, Fake((9,)), None, x)
    with pytest.raises(ValueError, match="mean"):
        ln.forward(x, None, None, x, mean=Fake((2,)))
    for k in (dict(buckets=0), dict(buckets=9, top_k=10), dict(buckets=30, top_k=17), dict(buckets=2000)):
        with pytest.raises(ValueError):
            ops.BucketGate(**k)
    for k in (dict(batch=0, rows=2, cols=2), dict(batch=1, rows=0, cols=2), dict(batch=1, rows=2, cols=2, steps=0)):
        with pytest.raises(ValueError):
            ops.Orthogonaliser(**k)
    with pytest.raises(ValueError, match="beta"):
        ops.Muon(1, 2, 2, beta=1.0)
    with pytest.raises(ValueError, match="min_w"):
        ops.Muon(1, 2, 2, min_w=1.0, max_w=0.0)


def test_host_tensors_are_refused():
    torch = pytest.importorskip("torch")
    ln = ops.LayerNorm(8)
    with pytest.raises(ValueError, match="on the device"):
        ln.forward(torch.zeros(2, 8), None, None, torch.zeros(2, 8))
