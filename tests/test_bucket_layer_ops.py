"""Refusals of the operators around a learned choice's bucket layers: wrong shapes, types,
sizes, pointers and devices are errors before any device call.  CPU only."""
import ctypes as C

import numpy as np
import pytest

from tatara_amd import _lib, ops

FAKE = 4096  # an address that a refused call never reads


class Fake:
    """Stands for a device array."""

    def __init__(self, *shape, dtype="float32"):
        self.shape, self.dtype, self.ptr = shape, np.dtype(dtype), FAKE


class Elsewhere(Fake):
    """Stands for a tensor on the second GPU."""

    is_cuda, device = True, "cuda:1"

    def get_device(self):
        return 1

    def data_ptr(self):
        return FAKE

    def stride(self):
        return tuple(int(np.prod(self.shape[i + 1:])) for i in range(len(self.shape)))

    def is_contiguous(self):
        return True


def caller(name, **usual):
    def call(**k):
        assert set(k) <= set(usual), k
        return getattr(_lib.load(), name)(*{**usual, **k}.values(), None)
    return call


def refused(status, part):
    assert status == -3 and part in _lib.load().tatara_last_error(), _lib.load().tatara_last_error()


rms = caller("tatara_op_rms_norm_forward", x=FAKE, xs=16, res=FAKE, rs=16, w=FAKE, total=FAKE, ts=16, y=FAKE, ys=16,
             rstd=FAKE, rows=4, cols=16, eps=1e-6, t=0)
rms8 = caller("tatara_op_rms_norm_forward_8bit", x=FAKE, xs=16, res=FAKE, rs=16, w=FAKE, total=FAKE, ts=16, y=FAKE,
              ys=16, scale=FAKE, rstd=FAKE, rows=4, cols=16, group=0, eps=1e-6, t=0, format=0)
rms_back = caller("tatara_op_rms_norm_backward", dy=FAKE, dys=16, total=FAKE, ts=16, w=FAKE, rstd=FAKE, dt=FAKE, dts=16,
                  dx=FAKE, dxs=16, dw=FAKE, rows=4, cols=16, t=0, ws=FAKE, n=1 << 30)
dropout = caller("tatara_op_dropout", x=FAKE, xs=16, res=FAKE, rs=16, y=FAKE, ys=16, rows=4, cols=16, p=0.1, seed=1,
                 step=2, more=FAKE, first=0, t=0)
sort = caller("tatara_op_bucket_rows_sort", bucket=FAKE, n=4, e=9, k=2, capacity=0, slot=FAKE, source=FAKE, offset=FAKE,
              ws=FAKE, wn=1 << 30)
gather = caller("tatara_op_bucket_rows_gather", x=FAKE, xs=16, slot=FAKE, source=FAKE, n=4, k=2, rows=FAKE, rs=16, m=8,
                cols=16, t=0)
combine = caller("tatara_op_bucket_rows_combine", rows=FAKE, rs=16, m=8, slot=FAKE, gate=FAKE, n=4, k=2, y=FAKE, ys=16,
                 cols=16, t=0)
combine_back = caller("tatara_op_bucket_rows_combine_backward", dy=FAKE, dys=16, rows=FAKE, rs=16, m=8, slot=FAKE,
                      source=FAKE, gate=FAKE, n=4, k=2, drows=FAKE, drs=16, dgate=FAKE, cols=16, t=0)
embed = caller("tatara_op_embedding_forward", token=FAKE, n=4, table=FAKE, ts=16, v=9, cols=16, scale=1.0, y=FAKE,
               ys=16, t=0)
embed_back = caller("tatara_op_embedding_backward", dy=FAKE, dys=16, token=FAKE, n=4, v=9, cols=16, scale=1.0, d=FAKE,
                    t=0, ws=FAKE, wn=1 << 30)


def test_rms_norm_refuses():
    for call in (rms, rms8):
        refused(call(t=3), b"element type")
        refused(call(cols=0), b"columns")
        refused(call(cols=32769), b"columns")
        refused(call(rows=1 << 31), b"rows")
        refused(call(eps=-1.0), b"eps")
        refused(call(eps=float("nan")), b"eps")
        refused(call(res=None), b"residual")
        refused(call(x=None), b"null")
        refused(call(y=None), b"null")
        for stride in ("xs", "rs", "ts", "ys"):
            refused(call(**{stride: 15}), b"stride")
        for p in ("x", "res", "total"):
            refused(call(**{p: FAKE + 2}), b"aligned")
        refused(call(ts=17), b"in place")
        refused(call(x=2 * FAKE, ts=17), b"in place")
    refused(rms_back(dxs=17), b"in place")
    refused(rms(y=FAKE + 1, t=2), b"aligned")
    refused(rms8(format=2), b"format")
    refused(rms8(group=16), b"scale")
    refused(rms8(scale=None), b"null")
    refused(rms_back(ws=None), b"workspace")
    refused(rms_back(n=4 * 512 * 16 - 1), b"workspace")
    refused(rms_back(ws=FAKE + 8), b"aligned")
    for p in ("dy", "total", "rstd", "dx"):
        refused(rms_back(**{p: None}), b"null")
    for stride in ("dys", "ts", "dts", "dxs"):
        refused(rms_back(**{stride: 3}), b"stride")
    for p in ("dy", "total", "dt", "dx"):
        refused(rms_back(**{p: FAKE + 2}), b"aligned")
    refused(rms_back(t=-1), b"element type")
    refused(_lib.load().tatara_op_rms_norm_backward_workspace(16, None), b"null")
    n = C.c_uint64()
    refused(_lib.load().tatara_op_rms_norm_backward_workspace(0, C.byref(n)), b"columns")


def test_dropout_refuses():
    refused(dropout(t=3), b"element type")
    refused(dropout(cols=0), b"columns")
    refused(dropout(cols=(1 << 24) + 1), b"columns")
    refused(dropout(rows=1 << 31), b"rows")
    refused(dropout(first=(1 << 32) - 1, rows=2), b"rows")
    for p in (-0.1, 1.0, float("nan")):
        refused(dropout(p=p), b"p must")
    refused(dropout(x=None), b"null")
    refused(dropout(y=None), b"null")
    for stride in ("xs", "rs", "ys"):
        refused(dropout(**{stride: 15}), b"stride")
    for p in ("x", "res", "y", "more"):
        refused(dropout(**{p: FAKE + 2}), b"aligned")
    refused(dropout(ys=17), b"in place")
    refused(dropout(x=2 * FAKE, ys=17), b"in place")


def test_bucket_rows_refuse():
    for e in (0, 1025):
        refused(sort(e=e), b"buckets")
    for call in (sort, gather, combine, combine_back):
        refused(call(k=0), b"top_k")
        refused(call(k=17), b"top_k")
        refused(call(n=1 << 30), b"positions")
        refused(call(n=1 << 31, k=1), b"positions")
        refused(call(slot=None), b"null")
    refused(sort(capacity=1 << 30), b"rows")
    for p in ("bucket", "source", "offset"):
        refused(sort(**{p: None}), b"null")
    refused(sort(ws=None), b"workspace")
    refused(sort(wn=100), b"workspace")
    refused(sort(ws=FAKE + 4), b"aligned")
    n = C.c_uint64()
    refused(_lib.load().tatara_op_bucket_rows_workspace(9, None), b"null")
    refused(_lib.load().tatara_op_bucket_rows_workspace(0, C.byref(n)), b"buckets")
    for call, pointers, strides, aligned in (
            (gather, ("x", "source", "rows"), ("xs", "rs"), ("x", "rows")),
            (combine, ("rows", "y"), ("rs", "ys"), ("rows", "y")),
            (combine_back, ("dy", "rows", "source", "gate", "drows"), ("dys", "rs", "drs"), ("dy", "rows", "drows"))):
        refused(call(t=5), b"element type")
        refused(call(cols=0), b"columns")
        refused(call(cols=32769), b"columns")
        refused(call(m=1 << 31), b"rows")
        for p in pointers:
            refused(call(**{p: None}), b"null")
        for s in strides:
            refused(call(**{s: 15}), b"stride")
        for p in aligned:
            refused(call(**{p: FAKE + 2}), b"aligned")
    refused(combine(m=0), b"without rows")
    refused(combine_back(m=0), b"without rows")


def test_embedding_refuses():
    for call in (embed, embed_back):
        refused(call(t=-2), b"element type")
        refused(call(v=0), b"table")
        refused(call(v=(1 << 28) + 1), b"table")
        refused(call(cols=0), b"columns")
        refused(call(cols=32769), b"columns")
        refused(call(n=1 << 31), b"positions")
        refused(call(token=None), b"null")
    for p in ("table", "y"):
        refused(embed(**{p: None}), b"null")
        refused(embed(**{p: FAKE + 2}), b"aligned")
    for s in ("ts", "ys"):
        refused(embed(**{s: 15}), b"stride")
    for p in ("dy", "d"):
        refused(embed_back(**{p: None}), b"null")
    refused(embed_back(dys=15), b"stride")
    refused(embed_back(dy=FAKE + 2), b"aligned")
    refused(embed_back(ws=None), b"workspace")
    refused(embed_back(wn=64), b"workspace")
    refused(embed_back(ws=FAKE + 8), b"aligned")
    refused(_lib.load().tatara_op_embedding_backward_workspace(4, 9, 16, 0, None), b"null")


@pytest.mark.parametrize("make,match", [
    (lambda: ops.RMSNorm(8, "f64"), "dtype"), (lambda: ops.RMSNorm(0), "cols"),
    (lambda: ops.RMSNorm(8, eps=float("nan")), "eps"), (lambda: ops.RMSNorm(8, out8="e5m2"), "out8"),
    (lambda: ops.RMSNorm(8, group=16), "group"), (lambda: ops.Dropout(0, 0.1), "cols"),
    (lambda: ops.Dropout(8, 1.0), "p must"), (lambda: ops.Dropout(8, float("nan")), "p must"),
    (lambda: ops.Dropout(8, 0.1, seed=-1), "seed"), (lambda: ops.BucketRows(0, 8), "buckets"),
    (lambda: ops.BucketRows(1025, 8), "buckets"), (lambda: ops.BucketRows(9, 0), "cols"),
    (lambda: ops.BucketRows(9, 8, 17), "top_k"), (lambda: ops.BucketRows(9, 8, capacity=0), "capacity"),
    (lambda: ops.BucketRows(1024, 8, capacity=1 << 21), "capacity"), (lambda: ops.Embedding(0, 8, 4), "vocab"),
    (lambda: ops.Embedding(9, 40000, 4), "cols"), (lambda: ops.Embedding(9, 8, -1), "positions")])
def test_operators_that_cannot_be_made(make, match):
    with pytest.raises(ValueError, match=match):
        make()


def calls(T):
    """Every call, on 3 positions of 8 columns (9 buckets, 2 choices), by the name of the
    tensor that stands in another shape or type."""
    i32 = dict(dtype="int32")
    right = dict(x=T(3, 8), residual=T(3, 8), total=T(3, 8), y=T(3, 8), weight=T(8), rstd=T(3), dy=T(3, 8), dx=T(3, 8),
                 dtotal=T(3, 8), dweight=T(8), q=T(3, 8, dtype="uint8"), scale=T(3, 1), more_steps=T(1, dtype="int64"),
                 bucket=T(3, 2, **i32), slot=T(3, 2, **i32), source=T(6, **i32), offset=T(10, **i32), rows=T(6, 8),
                 drows=T(6, 8), gate=T(3, 2), dgate=T(3, 2), token=T(3, **i32), table=T(9, 8), dtable=T(9, 8))
    norm, drop = ops.RMSNorm(8), ops.Dropout(8, 0.1)
    rows, embedding = ops.BucketRows(9, 8, 2), ops.Embedding(9, 8, 100)
    for op in (norm, rows, embedding):
        op._ws = {d: Fake(1) for d in (-2, -1, 0, 1)}
        for w in op._ws.values():
            w.nbytes = 1 << 30
    return right, {
        norm.forward: ("x", "weight", "y", "rstd", "residual", "total"),
        norm.forward_8bit: ("x", "weight", "q", "scale", "rstd", "residual", "total"),
        norm.backward: ("dy", "total", "weight", "rstd", "dx", "dweight", "dtotal"),
        drop.backward: ("dy", "dx", "more_steps"), drop.forward: ("x", "y", "residual", "more_steps"),
        rows.sort: ("bucket", "slot", "source", "offset"), rows.gather: ("x", "slot", "source", "rows"),
        rows.gather_backward: ("drows", "slot", "dx"), rows.combine: ("rows", "slot", "gate", "y"),
        rows.combine_backward: ("dy", "rows", "slot", "source", "gate", "drows", "dgate"),
        embedding.forward: ("token", "table", "y"), embedding.backward: ("dy", "token", "dtable")}


def make(call, names, tensors):
    keywords = dict(residual="residual", total="total", more_steps="more_steps", dtotal="dtotal")
    own = [n for n in names if n not in keywords or (n == "total" and call.__name__ == "backward")]
    return lambda: call(*(tensors[n] for n in own), **{n: tensors[n] for n in names if n not in own})


def test_tensors_of_another_shape_or_type_are_refused():
    right, every = calls(Fake)
    for call, names in every.items():
        for name in names:
            t = right[name]
            for wrong in (Fake(*t.shape[:-1], t.shape[-1] + 1, dtype=t.dtype), Fake(*t.shape, 1, dtype=t.dtype),
                          Fake(*t.shape, dtype="float64"), None if name in ("x", "y", "slot", "token") else 3.0):
                with pytest.raises(ValueError, match="must be a"):
                    make(call, names, {**right, name: wrong})()


def test_tensors_of_another_device_are_refused():
    right, every = calls(Elsewhere)
    for call, names in every.items():
        with pytest.raises(ValueError, match="on device 1"):
            make(call, names, right)()


def test_arguments_that_say_nothing_together():
    right, _ = calls(Fake)
    with pytest.raises(ValueError, match="residual"):
        ops.RMSNorm(8).forward(right["x"], None, right["y"], total=right["total"])
    for k in (dict(step=-1), dict(step=1 << 64), dict(first_row=-1), dict(first_row=1 << 32)):
        with pytest.raises(ValueError, match="must be 0"):
            ops.Dropout(8, 0.1).forward(right["x"], right["y"], **k)
    with pytest.raises(ValueError, match="up to 2"):
        ops.Embedding(9, 8, 2).backward(right["dy"], right["token"], right["dtable"])


def test_rows_of_so_many_positions():
    assert ops.BucketRows(9, 8, 2).rows(5) == 10 and ops.BucketRows(9, 8, 2, capacity=4).rows(5) == 36


@pytest.mark.parametrize("name", ["norm", "rows", "embedding"])
def test_prepare_makes_one_workspace_a_device(name, monkeypatch):
    made, device = [], [0]
    monkeypatch.setattr(ops, "_Workspace", lambda nbytes: made.append((device[0], nbytes)) or object())
    monkeypatch.setattr(ops, "_here", lambda: device[0])
    op = dict(norm=ops.RMSNorm, rows=ops.BucketRows, embedding=ops.Embedding)[name](
        *dict(norm=(64,), rows=(9, 8), embedding=(9, 8, 100))[name])
    op.prepare()
    op.prepare()
    assert len(made) == 1 and made[0][1] > 0
    device[0] = 1
    op.prepare()
    assert [d for d, _ in made] == [0, 1]
