"""Operators for a learned bucket choice and for orthogonalised updates.

A LayerStack's bucket follows a fixed rule and its optimizers work element by
element, as in the reference, which has no counterpart of these operators: layer
norm (`LayerNorm`), a gate that chooses buckets by learned scores and keeps them
balanced (`BucketGate`), and Newton-Schulz orthogonalised updates of weight
matrices (`Orthogonaliser`, `Muon`), over the C ABI (tatara_op_layer_norm_*,
tatara_op_bucket_gate_*, tatara_op_orthogonalise, tatara_op_muon_step).

Around the layers that are chosen stand an embedding of a position's discrete values
(`Embedding`), dropout (`Dropout`), a root-mean-square norm with the residual's addition
and an output in 8 bits (`RMSNorm`), and the rows of each bucket side by side and
back (`BucketRows`): tatara_op_embedding_*, tatara_op_dropout, tatara_op_rms_norm_*,
tatara_op_bucket_rows_*.

An operator is made once for a layer's shape and holds its workspace.  Tensors
are device memory: a `DeviceArray`, or any object with data_ptr(), shape,
stride(), dtype, get_device() and is_contiguous() (a torch tensor on the GPU; torch is
imported before the library is loaded, so that both run on one HIP runtime).  The last
dimension is contiguous; rows may lie inside wider ones.  An operator's element
type is "f32", "f16" or "bf16"; a DeviceArray holds bf16 as uint16 (and e4m3 as uint8).  Calls queue
their work on `stream` (a runtime.Stream or a torch.cuda.Stream; None is torch's
current stream where the call's first tensor is torch's, else the null stream) and return;
one operator's calls belong on one stream at a time, since they share the
workspace.  All tensors of a call lie on the thread's current device, and what it
writes overlaps nothing else of it unless its description says so.  The first call
there that needs the workspace makes it, which waits for the device and cannot be
recorded into a graph; prepare() makes it ahead.  Wrong shapes, types and devices raise
ValueError, device errors TataraError.
"""
from __future__ import annotations

import ctypes as C
import sys

from . import _lib
from ._lib import check

DTYPES = {"f32": 0, "f16": 1, "bf16": 2}
# names of array types -> the element type that they hold
_HOLDS = {"float32": "f32", "torch.float32": "f32", "float16": "f16", "torch.float16": "f16", "uint16": "bf16",
          "torch.bfloat16": "bf16", "int32": "i32", "torch.int32": "i32", "uint8": "u8", "torch.uint8": "u8",
          "int8": "i8", "torch.int8": "i8", "torch.float8_e4m3fn": "e4m3", "uint64": "u64", "torch.uint64": "u64",
          "int64": "u64", "torch.int64": "u64"}
# DeviceArray types that stand in for one that numpy lacks
_STANDS_FOR = {"u8": "e4m3"}


class _TypeNames(dict):
    """Array type -> element type (None: no operator's), filled as types are met."""

    def __missing__(self, array_type):
        self[array_type] = name = _HOLDS.get(str(array_type))
        return name


_TYPE = _TypeNames()


# torch.cuda.current_device and the hipStream_t of its current stream on a device, once
# torch has met the GPU
_torch_device = _torch_stream = None


def _one_runtime() -> bool:
    """Whether this library and torch run on one HIP runtime.  torch brings its own and
    the library takes the one that is loaded, or the system's if none is: loaded ahead
    of torch they have two, whose streams know nothing of each other."""
    with open("/proc/self/maps") as maps:
        return len({line.split()[-1] for line in maps if "/libamdhip64.so" in line}) < 2


def _two_runtimes():
    raise RuntimeError("torch and tatara_amd's library run on two HIP runtimes, which cannot order each other's work: "
                       "import torch before the library is loaded")


def _here() -> int:
    """The thread's current device, which every tensor of a call lies on.  Below zero
    where no torch tensor can be taken, one number a device."""
    global _torch_device, _torch_stream
    if _torch_device is not None:
        return _torch_device()
    device = C.c_int32()
    if _lib.load().tatara_get_device(C.byref(device)):
        return -2  # no GPU, as the call will say; -1 is what a host tensor gives
    torch = sys.modules.get("torch")
    if torch is not None and torch.cuda.is_initialized():  # else no tensor of its lies on a GPU
        if not _one_runtime():
            return -3 - device.value
        # what torch.cuda.current_stream and current_device ask, without a Stream object for
        # the answer: 0.6 us less of a call's 7
        _torch_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                                lambda device: torch.cuda.current_stream(device).cuda_stream)
        _torch_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
        return _torch_device()
    return device.value


class _Handles(dict):
    """(device, hipStream_t) -> the library's handle of that stream of torch's."""

    def __missing__(self, key) -> int:
        h = C.c_void_p()
        check(_lib.load().tatara_stream_wrap(*key, C.byref(h)))
        self[key] = h.value  # 16 bytes, for as long as the process
        return h.value


_HANDLES = _Handles()


def _place(x, stream):
    """The current device, as _here() gives it, and the handle of the stream that a call
    goes to whose first tensor is x."""
    here = _here() if _torch_device is None else _torch_device()
    if stream is None:
        if here < 0 or not hasattr(x, "get_device"):
            return here, None
        native = _torch_stream(here)
        return here, _HANDLES[here, native] if native else None  # the default one is the null stream
    if hasattr(stream, "cuda_stream"):
        if here < -2:
            _two_runtimes()
        return here, _HANDLES[stream.device_index, stream.cuda_stream]
    if not stream.handle:
        raise ValueError("the stream is closed")
    return here, stream.handle


class _Workspaces(dict):
    """Device memory that an operator keeps for its calls, by device."""

    def __init__(self, nbytes: int):
        super().__init__()
        self.nbytes = nbytes

    def __missing__(self, device: int):  # the current one
        self[device] = w = _Workspace(self.nbytes)
        return w


class _Workspace:
    """Memory of the current device."""

    def __init__(self, nbytes: int):
        p = C.c_void_p()
        check(_lib.load().tatara_malloc(C.byref(p), nbytes))
        self.ptr, self.nbytes = p.value, nbytes
        check(_lib.load().tatara_memset(self.ptr, 0, min(nbytes, 4096)))  # counts that begin at zero
        check(_lib.load().tatara_synchronize())  # before any stream's work

    def __del__(self):
        try:
            if self.ptr:
                _lib.load().tatara_free(self.ptr)  # waits for the device's work
                self.ptr = None
        except Exception:
            pass


class _Operator:
    _ws: _Workspaces

    def prepare(self) -> None:
        """Makes the workspace on the current device, if it has none yet."""
        self._ws[_here()]


def _dtype(dtype: str) -> int:
    if dtype not in DTYPES:
        raise ValueError(f"dtype must be one of {', '.join(DTYPES)}, not {dtype!r}")
    return DTYPES[dtype]


def _wrong(name: str, x, shape, dtype: str):
    if getattr(x, "is_cuda", False) and x.get_device() != _here():
        if _here() < -2:
            _two_runtimes()
        raise ValueError(f"{name} is on device {x.get_device()}, the current device is {_here()}")
    raise ValueError(f"{name} must be a {dtype} tensor of shape {tuple(shape)} on the device with a contiguous last "
                     f"dimension, not {getattr(x, 'dtype', type(x).__name__)} {tuple(getattr(x, 'shape', ()))}")


def _count(name: str, x, cols: int, dtype: str) -> int:
    """The rows of a [rows, cols] tensor."""
    try:
        rows, _ = x.shape
        return rows
    except (AttributeError, TypeError, ValueError):
        _wrong(name, x, ("rows", cols), dtype)


def _owned(name: str, x, shape: tuple, dtype: str) -> int:
    """The address of a DeviceArray of this shape."""
    if hasattr(x, "data_ptr") or not hasattr(x, "ptr") or tuple(x.shape) != shape or not (
            _TYPE[x.dtype] == dtype or _STANDS_FOR.get(_TYPE[x.dtype]) == dtype):
        _wrong(name, x, shape, dtype)
    return x.ptr


# The checks below are most of a small call's time on the host: each reads a
# tensor's attributes once, and everything that is not a right tensor goes on to
# _owned, which takes a DeviceArray and refuses the rest.

def _dense(name: str, x, shape: tuple, dtype: str, here: int) -> int:
    """The address of a contiguous tensor of this shape."""
    try:
        if x.shape == shape and _TYPE[x.dtype] == dtype and x.get_device() == here and x.is_contiguous():
            return x.data_ptr()
    except AttributeError:
        pass
    return _owned(name, x, shape, dtype)


def _rows(name: str, x, shape: tuple, dtype: str, here: int):
    """Address and row stride of a [rows, cols] tensor."""
    try:
        if x.shape == shape and _TYPE[x.dtype] == dtype and x.get_device() == here:
            stride, one = x.stride()
            if one == 1 or shape[1] == 1:
                return x.data_ptr(), stride if shape[0] > 1 else shape[1]  # one row's stride says nothing
    except AttributeError:
        pass
    return _owned(name, x, shape, dtype), shape[1]


def _matrices(name: str, x, shape: tuple, dtype: str, here: int):
    """Address, row stride and matrix stride of a [batch, rows, cols] tensor."""
    try:
        if x.shape == shape and _TYPE[x.dtype] == dtype and x.get_device() == here:
            batch, stride, one = x.stride()
            if one == 1 or shape[2] == 1:
                return x.data_ptr(), stride if shape[1] > 1 else shape[2], batch
    except AttributeError:
        pass
    return _owned(name, x, shape, dtype), shape[2], shape[1] * shape[2]


class LayerNorm(_Operator):
    """y = (x - mean) * rstd * weight + bias over rows of `cols` values.

    x, y, dy and dx are [rows, cols] of `dtype`; weight, bias, mean, rstd and the
    weight's and bias's gradients are f32.  weight and bias may be None."""

    def __init__(self, cols: int, dtype: str = "f32", eps: float = 1e-5):
        self.cols, self.dtype, self.eps = int(cols), dtype, float(eps)
        self._code = _dtype(dtype)
        if not 1 <= self.cols <= 32768:
            raise ValueError(f"cols must be 1 to 32768, not {cols}")
        if not self.eps >= 0.0:
            raise ValueError(f"eps must not be negative, not {eps}")
        self._lib = _lib.load()
        n = C.c_uint64()
        check(self._lib.tatara_op_layer_norm_backward_workspace(self.cols, C.byref(n)))
        self._ws = _Workspaces(n.value)

    def forward(self, x, weight, bias, y, mean=None, rstd=None, stream=None) -> None:
        """Writes y, and mean and rstd [rows] for the backward pass if given."""
        cols, dtype = self.cols, self.dtype
        here, queue = _place(x, stream)
        rows = _count("x", x, cols, dtype)
        shape, vec, param = (rows, cols), (rows,), (cols,)
        xp, xs = _rows("x", x, shape, dtype, here)
        yp, ys = _rows("y", y, shape, dtype, here)
        status = self._lib.tatara_op_layer_norm_forward(
            xp, xs, None if weight is None else _dense("weight", weight, param, "f32", here),
            None if bias is None else _dense("bias", bias, param, "f32", here), yp, ys,
            None if mean is None else _dense("mean", mean, vec, "f32", here),
            None if rstd is None else _dense("rstd", rstd, vec, "f32", here), rows, cols, self.eps, self._code,
            queue)
        if status:
            check(status)

    def backward(self, dy, x, weight, mean, rstd, dx, dweight=None, dbias=None, stream=None) -> None:
        """Writes dx, and the weight's and bias's gradients [cols] if given (overwritten)."""
        cols, dtype = self.cols, self.dtype
        here, queue = _place(dy, stream)
        rows = _count("x", x, cols, dtype)
        shape, vec, param = (rows, cols), (rows,), (cols,)
        dyp, dys = _rows("dy", dy, shape, dtype, here)
        xp, xs = _rows("x", x, shape, dtype, here)
        dxp, dxs = _rows("dx", dx, shape, dtype, here)
        status = self._lib.tatara_op_layer_norm_backward(
            dyp, dys, xp, xs, None if weight is None else _dense("weight", weight, param, "f32", here),
            _dense("mean", mean, vec, "f32", here), _dense("rstd", rstd, vec, "f32", here), dxp, dxs,
            None if dweight is None else _dense("dweight", dweight, param, "f32", here),
            None if dbias is None else _dense("dbias", dbias, param, "f32", here), rows, cols, self._code,
            (ws := self._ws[here]).ptr, ws.nbytes, queue)
        if status:
            check(status)


class BucketGate(_Operator):
    """The best top_k of `buckets` for each position by its logits, with the loss
    that keeps them balanced: balance * buckets / (top_k * counted^2) *
    sum_e count[e] * prob_sum[e], which is `balance` when all are taken alike.

    Logits are [positions, buckets] of `dtype`; a logit of -infinity masks the
    bucket for the position, and valid [positions] (uint8) of 0 leaves the position out."""

    def __init__(self, buckets: int, top_k: int = 1, dtype: str = "f32", renormalise: bool = False,
                 balance: float = 0.01):
        self.buckets, self.top_k, self.dtype = int(buckets), int(top_k), dtype
        self.renormalise, self.balance = int(bool(renormalise)), float(balance)
        self._code = _dtype(dtype)
        if not 1 <= self.buckets <= 1024:
            raise ValueError(f"buckets must be 1 to 1024, not {buckets}")
        if not 1 <= self.top_k <= min(16, self.buckets):
            raise ValueError(f"top_k must be 1 to 16 and no more than buckets, not {top_k}")
        self._lib = _lib.load()
        n = C.c_uint64()
        check(self._lib.tatara_op_bucket_gate_workspace(self.buckets, C.byref(n)))
        self._ws = _Workspaces(n.value)

    def forward(self, logits, bucket, gate, count, prob_sum, counted, loss, valid=None, stream=None) -> None:
        """Writes bucket (int32) and gate (f32) [positions, top_k], count (int32)
        and prob_sum (f32) [buckets], counted (int32) and loss (f32) [1]."""
        here, queue = _place(logits, stream)
        n = _count("logits", logits, self.buckets, self.dtype)
        lp, ls = _rows("logits", logits, (n, self.buckets), self.dtype, here)
        chosen = (n, self.top_k)
        check(self._lib.tatara_op_bucket_gate_forward(
            lp, ls, None if valid is None else _dense("valid", valid, (n,), "u8", here), n, self.buckets, self.top_k,
            self.renormalise, self.balance, self._code, _dense("bucket", bucket, chosen, "i32", here),
            _dense("gate", gate, chosen, "f32", here), _dense("count", count, (self.buckets,), "i32", here),
            _dense("prob_sum", prob_sum, (self.buckets,), "f32", here), _dense("counted", counted, (1,), "i32", here),
            _dense("loss", loss, (1,), "f32", here), (ws := self._ws[here]).ptr, ws.nbytes,
            queue))

    def backward(self, logits, bucket, count, counted, dlogits, dgate=None, dloss: float = 1.0, valid=None,
                 stream=None) -> None:
        """Writes dlogits from dgate (f32 [positions, top_k], None: no gradient) and
        dloss; bucket, count and counted are the forward call's."""
        here, queue = _place(logits, stream)
        n = _count("logits", logits, self.buckets, self.dtype)
        lp, ls = _rows("logits", logits, (n, self.buckets), self.dtype, here)
        dp, ds = _rows("dlogits", dlogits, (n, self.buckets), self.dtype, here)
        chosen = (n, self.top_k)
        check(self._lib.tatara_op_bucket_gate_backward(
            lp, ls, None if valid is None else _dense("valid", valid, (n,), "u8", here), n, self.buckets, self.top_k,
            self.renormalise, self.balance, self._code, _dense("bucket", bucket, chosen, "i32", here),
            _dense("count", count, (self.buckets,), "i32", here), _dense("counted", counted, (1,), "i32", here),
            None if dgate is None else _dense("dgate", dgate, chosen, "f32", here), dloss, dp, ds,
            queue))


class Orthogonaliser(_Operator):
    """Newton-Schulz orthogonalisation of `batch` matrices [rows, cols]: called
    with input and output [batch, rows, cols] of `dtype` (out may be the input).

    Products take operands of 22 bits and sum in f32, whatever the type; the result is
    rounded to it once."""

    def __init__(self, batch: int, rows: int, cols: int, dtype: str = "f32", steps: int = 5):
        self.batch, self.rows, self.cols = int(batch), int(rows), int(cols)
        self.shape, self.dtype, self.steps = (self.batch, self.rows, self.cols), dtype, int(steps)
        self._code = _dtype(dtype)
        if self.batch < 1:
            raise ValueError(f"batch must be at least 1, not {batch}")
        if not 1 <= self.steps <= 32:
            raise ValueError(f"steps must be 1 to 32, not {steps}")
        if not (1 <= self.rows <= 32768 and 1 <= self.cols <= 32768):
            raise ValueError(f"a matrix has sides of 1 to 32768, not {rows} x {cols}")
        self._lib = _lib.load()
        n = C.c_uint64()
        check(self._lib.tatara_op_orthogonalise_workspace(self.batch, self.rows, self.cols, self._code, C.byref(n)))
        self._ws = _Workspaces(n.value)

    def __call__(self, x, out, stream=None) -> None:
        here, queue = _place(x, stream)
        xp, xr, xb = _matrices("x", x, self.shape, self.dtype, here)
        op, orow, ob = _matrices("out", out, self.shape, self.dtype, here)
        check(self._lib.tatara_op_orthogonalise(xp, xr, xb, op, orow, ob, self.batch, self.rows, self.cols,
                                                self._code, self.steps, (ws := self._ws[here]).ptr, ws.nbytes,
                                                queue))


class Muon(_Operator):
    """Muon updates of `batch` weight matrices [rows, cols]: momentum of the
    gradient, orthogonalised, subtracted from the weights.

    weights and momentum are f32 [batch, rows, cols], updated in place; the
    gradient is of `grad_dtype`.  step's scale multiplies lr in the update
    (sqrt(max(1, rows / cols)) keeps an update's size alike over shapes);
    weights are clamped to [min_w, max_w]."""

    def __init__(self, batch: int, rows: int, cols: int, beta: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0, grad_dtype: str = "f32", steps: int = 5, min_w: float = -1e30,
                 max_w: float = 1e30):
        if not 0.0 <= beta < 1.0:
            raise ValueError(f"beta must be in [0, 1), not {beta}")
        if not min_w <= max_w:
            raise ValueError(f"min_w {min_w} exceeds max_w {max_w}")
        self.grad_dtype, self._grad_code = grad_dtype, _dtype(grad_dtype)
        self._ortho = Orthogonaliser(batch, rows, cols, "f32", steps)
        self._ws = self._ortho._ws
        self.shape, self.beta, self.nesterov = self._ortho.shape, float(beta), int(bool(nesterov))
        self.weight_decay, self.min_w, self.max_w = float(weight_decay), float(min_w), float(max_w)

    def step(self, weights, momentum, grad, lr: float, scale: float = 1.0, stream=None) -> None:
        o, shape = self._ortho, self.shape
        here, queue = _place(weights, stream)
        check(o._lib.tatara_op_muon_step(
            _dense("weights", weights, shape, "f32", here), _dense("momentum", momentum, shape, "f32", here),
            _dense("grad", grad, shape, self.grad_dtype, here), o.batch, o.rows, o.cols, self._grad_code, self.beta,
            self.nesterov, lr, self.weight_decay, scale, self.min_w, self.max_w, o.steps,
            (ws := self._ws[here]).ptr, ws.nbytes, queue))


class RMSNorm(_Operator):
    """y = s * rstd * weight over rows of `cols` values, with s = x + residual.

    x, residual, total (s as it is stored, which is what is normalised), y, dy,
    dtotal and dx are [rows, cols] of `dtype`; weight, rstd and dweight are f32, and
    weight may be None.  forward_8bit writes y as q [rows, cols] of `out8` ("e4m3" or
    "i8") and scale f32 [rows, groups], y being about q * scale; a scale stands for
    `group` columns (32, 64 or 128), or for the row (0)."""

    def __init__(self, cols: int, dtype: str = "f32", eps: float = 1e-6, out8: str = "e4m3", group: int = 0):
        self.cols, self.dtype, self.eps, self.out8, self.group = int(cols), dtype, float(eps), out8, int(group)
        self._code = _dtype(dtype)
        if not 1 <= self.cols <= 32768:
            raise ValueError(f"cols must be 1 to 32768, not {cols}")
        if not self.eps >= 0.0:
            raise ValueError(f"eps must not be negative, not {eps}")
        if out8 not in ("e4m3", "i8"):
            raise ValueError(f"out8 must be e4m3 or i8, not {out8!r}")
        if self.group not in (0, 32, 64, 128):
            raise ValueError(f"group must be 0, 32, 64 or 128, not {group}")
        self.groups = -(-self.cols // self.group) if self.group else 1
        self._format = ("e4m3", "i8").index(out8)
        self._lib = _lib.load()
        n = C.c_uint64()
        check(self._lib.tatara_op_rms_norm_backward_workspace(self.cols, C.byref(n)))
        self._ws = _Workspaces(n.value)

    def _sum(self, shape, residual, total, here):
        """Addresses and strides of residual and total."""
        if residual is None:
            if total is not None:
                raise ValueError("total needs a residual")
            return None, 0, None, 0
        rp, rs = _rows("residual", residual, shape, self.dtype, here)
        return (rp, rs, None, 0) if total is None else (rp, rs, *_rows("total", total, shape, self.dtype, here))

    def forward(self, x, weight, y, rstd=None, residual=None, total=None, stream=None) -> None:
        """Writes y, rstd [rows] for the backward pass if given, and the sum of x and
        residual into total if given (which may be x or residual)."""
        cols = self.cols
        here, queue = _place(x, stream)
        rows = _count("x", x, cols, self.dtype)
        shape = (rows, cols)
        xp, xs = _rows("x", x, shape, self.dtype, here)
        yp, ys = _rows("y", y, shape, self.dtype, here)
        rp, rs, tp, ts = self._sum(shape, residual, total, here)
        status = self._lib.tatara_op_rms_norm_forward(
            xp, xs, rp, rs, None if weight is None else _dense("weight", weight, (cols,), "f32", here), tp, ts, yp, ys,
            None if rstd is None else _dense("rstd", rstd, (rows,), "f32", here), rows, cols, self.eps, self._code,
            queue)
        if status:
            check(status)

    def forward_8bit(self, x, weight, q, scale, rstd=None, residual=None, total=None, stream=None) -> None:
        """forward() with y as q and scale."""
        cols = self.cols
        here, queue = _place(x, stream)
        rows = _count("x", x, cols, self.dtype)
        shape = (rows, cols)
        xp, xs = _rows("x", x, shape, self.dtype, here)
        qp, qs = _rows("q", q, shape, self.out8, here)
        rp, rs, tp, ts = self._sum(shape, residual, total, here)
        status = self._lib.tatara_op_rms_norm_forward_8bit(
            xp, xs, rp, rs, None if weight is None else _dense("weight", weight, (cols,), "f32", here), tp, ts, qp, qs,
            _dense("scale", scale, (rows, self.groups), "f32", here),
            None if rstd is None else _dense("rstd", rstd, (rows,), "f32", here), rows, cols, self.group, self.eps,
            self._code, self._format, queue)
        if status:
            check(status)

    def backward(self, dy, total, weight, rstd, dx, dweight=None, dtotal=None, stream=None) -> None:
        """Writes dx, the gradient of x and residual alike, from dy and, if given, the
        gradient dtotal that reaches the sum by itself (dx may be dtotal, not dy or total),
        and the weight's gradient [cols] if given (overwritten)."""
        cols, dtype = self.cols, self.dtype
        here, queue = _place(dy, stream)
        rows = _count("total", total, cols, dtype)
        shape = (rows, cols)
        dyp, dys = _rows("dy", dy, shape, dtype, here)
        tp, ts = _rows("total", total, shape, dtype, here)
        dxp, dxs = _rows("dx", dx, shape, dtype, here)
        dtp, dts = (None, 0) if dtotal is None else _rows("dtotal", dtotal, shape, dtype, here)
        status = self._lib.tatara_op_rms_norm_backward(
            dyp, dys, tp, ts, None if weight is None else _dense("weight", weight, (cols,), "f32", here),
            _dense("rstd", rstd, (rows,), "f32", here), dtp, dts, dxp, dxs,
            None if dweight is None else _dense("dweight", dweight, (cols,), "f32", here), rows, cols, self._code,
            (ws := self._ws[here]).ptr, ws.nbytes, queue)
        if status:
            check(status)


class Dropout:
    """y = x / (1 - p) where a number of the counter-based generator says so, else 0,
    plus a residual: [rows, cols] of `dtype`.

    The number of a value goes by `seed`, the call's step, its row (from first_row on, for
    a part of a batch) and its column alone, so backward() makes the mask again.  A layer
    has a seed of its own, and a training step a step of its own."""

    def __init__(self, cols: int, p: float, dtype: str = "f32", seed: int = 0):
        self.cols, self.p, self.dtype, self.seed = int(cols), float(p), dtype, int(seed)
        self._code = _dtype(dtype)
        if not 1 <= self.cols <= 1 << 24:
            raise ValueError(f"cols must be 1 to 2^24, not {cols}")
        if not 0.0 <= self.p < 1.0:
            raise ValueError(f"p must be in [0, 1), not {p}")
        if not 0 <= self.seed < 1 << 64:
            raise ValueError(f"seed must be 0 to 2^64 - 1, not {seed}")
        self._lib = _lib.load()

    def forward(self, x, y, step: int = 0, residual=None, more_steps=None, first_row: int = 0, stream=None) -> None:
        """Writes y, which may be x or residual.  The step is `step` plus more_steps ([1],
        int64) if that is given, which is read when the call runs."""
        here, queue = _place(x, stream)
        rows = _count("x", x, self.cols, self.dtype)
        shape = (rows, self.cols)
        if not 0 <= step < 1 << 64:
            raise ValueError(f"step must be 0 to 2^64 - 1, not {step}")
        if not 0 <= first_row <= (1 << 32) - 1:
            raise ValueError(f"first_row must be 0 to 2^32 - 1, not {first_row}")
        xp, xs = _rows("x", x, shape, self.dtype, here)
        yp, ys = _rows("y", y, shape, self.dtype, here)
        rp, rs = (None, 0) if residual is None else _rows("residual", residual, shape, self.dtype, here)
        status = self._lib.tatara_op_dropout(
            xp, xs, rp, rs, yp, ys, rows, self.cols, self.p, self.seed, step,
            None if more_steps is None else _dense("more_steps", more_steps, (1,), "u64", here), first_row,
            self._code, queue)
        if status:
            check(status)

    def backward(self, dy, dx, step: int = 0, more_steps=None, first_row: int = 0, stream=None) -> None:
        """Writes dx, which may be dy, of the forward call with the same step (the
        residual's gradient is dy itself)."""
        self.forward(dy, dx, step, None, more_steps, first_row, stream)


class BucketRows(_Operator):
    """The rows of each of `buckets` side by side, for its layers, and back in the
    positions' order.

    sort() takes a gate's choices, bucket [positions, top_k], and gives each a row:
    slot [positions, top_k], source [rows(positions)] (position * top_k + choice) and
    offset [buckets + 1] (choices of buckets below), all int32.  Packed (capacity None), bucket e
    has rows offset[e] to offset[e + 1] - 1; with a capacity it has rows e * capacity
    to (e + 1) * capacity - 1, and choices that do not fit have none.  -1 stands in slot for
    a choice without a row (a bucket of -1 is none) and in source for a row without a
    choice.  Rows and positions are [.., cols] of `dtype`; gate and dgate are f32."""

    def __init__(self, buckets: int, cols: int, top_k: int = 1, dtype: str = "f32", capacity: int | None = None):
        self.buckets, self.cols, self.top_k, self.dtype = int(buckets), int(cols), int(top_k), dtype
        self.capacity = None if capacity is None else int(capacity)
        self._code = _dtype(dtype)
        if not 1 <= self.buckets <= 1024:
            raise ValueError(f"buckets must be 1 to 1024, not {buckets}")
        if not 1 <= self.cols <= 32768:
            raise ValueError(f"cols must be 1 to 32768, not {cols}")
        if not 1 <= self.top_k <= 16:
            raise ValueError(f"top_k must be 1 to 16, not {top_k}")
        if self.capacity is not None and not 1 <= self.capacity * self.buckets < 1 << 31:
            raise ValueError(f"capacity must be at least 1 and buckets * capacity below 2^31, not {capacity}")
        self._lib = _lib.load()
        n = C.c_uint64()
        check(self._lib.tatara_op_bucket_rows_workspace(self.buckets, C.byref(n)))
        self._ws = _Workspaces(n.value)

    def rows(self, positions: int) -> int:
        """The rows of so many positions, those without a choice among them."""
        return positions * self.top_k if self.capacity is None else self.buckets * self.capacity

    def sort(self, bucket, slot, source, offset, stream=None) -> None:
        """Writes slot, source and offset."""
        here, queue = _place(bucket, stream)
        n = _count("bucket", bucket, self.top_k, "i32")
        chosen = (n, self.top_k)
        ws = self._ws[here]
        status = self._lib.tatara_op_bucket_rows_sort(
            _dense("bucket", bucket, chosen, "i32", here), n, self.buckets, self.top_k, self.capacity or 0,
            _dense("slot", slot, chosen, "i32", here), _dense("source", source, (self.rows(n),), "i32", here),
            _dense("offset", offset, (self.buckets + 1,), "i32", here), ws.ptr, ws.nbytes, queue)
        if status:
            check(status)

    def gather(self, x, slot, source, rows, stream=None) -> None:
        """Writes rows: x at its positions' slots, zeros without a choice."""
        here, queue = _place(x, stream)
        n = _count("x", x, self.cols, self.dtype)
        m = self.rows(n)
        xp, xs = _rows("x", x, (n, self.cols), self.dtype, here)
        rp, rs = _rows("rows", rows, (m, self.cols), self.dtype, here)
        status = self._lib.tatara_op_bucket_rows_gather(
            xp, xs, _dense("slot", slot, (n, self.top_k), "i32", here), _dense("source", source, (m,), "i32", here), n,
            self.top_k, rp, rs, m, self.cols, self._code, queue)
        if status:
            check(status)

    def gather_backward(self, drows, slot, dx, stream=None) -> None:
        """Writes dx: the sum of drows at each position's slots."""
        self.combine(drows, slot, None, dx, stream)

    def combine(self, rows, slot, gate, y, stream=None) -> None:
        """Writes y: the sum of rows at each position's slots, times gate
        [positions, top_k] unless that is None."""
        here, queue = _place(rows, stream)
        n = _count("y", y, self.cols, self.dtype)
        m = self.rows(n)
        rp, rs = _rows("rows", rows, (m, self.cols), self.dtype, here)
        yp, ys = _rows("y", y, (n, self.cols), self.dtype, here)
        chosen = (n, self.top_k)
        status = self._lib.tatara_op_bucket_rows_combine(
            rp, rs, m, _dense("slot", slot, chosen, "i32", here),
            None if gate is None else _dense("gate", gate, chosen, "f32", here), n, self.top_k, yp, ys, self.cols,
            self._code, queue)
        if status:
            check(status)

    def combine_backward(self, dy, rows, slot, source, gate, drows, dgate=None, stream=None) -> None:
        """Writes drows, and the gate's gradient if given; rows (the forward call's) may
        be None without it."""
        here, queue = _place(dy, stream)
        n = _count("dy", dy, self.cols, self.dtype)
        m = self.rows(n)
        dyp, dys = _rows("dy", dy, (n, self.cols), self.dtype, here)
        rp, rs = (None, 0) if rows is None and dgate is None else _rows("rows", rows, (m, self.cols), self.dtype, here)
        drp, drs = _rows("drows", drows, (m, self.cols), self.dtype, here)
        chosen = (n, self.top_k)
        status = self._lib.tatara_op_bucket_rows_combine_backward(
            dyp, dys, rp, rs, m, _dense("slot", slot, chosen, "i32", here),
            _dense("source", source, (m,), "i32", here), _dense("gate", gate, chosen, "f32", here), n, self.top_k, drp,
            drs, None if dgate is None else _dense("dgate", dgate, chosen, "f32", here), self.cols, self._code, queue)
        if status:
            check(status)


class Embedding(_Operator):
    """y = scale * table[token]: rows of a table [vocab, cols] by a position's token.

    token is int32 [positions]; one outside 0..vocab - 1, such as -1, stands for none: its
    row is zeros, and it has no gradient.  table, y and dy are of `dtype`, dtable is f32.
    `positions` is the most that a backward call takes."""

    def __init__(self, vocab: int, cols: int, positions: int, dtype: str = "f32", scale: float = 1.0):
        self.vocab, self.cols, self.positions, self.dtype = int(vocab), int(cols), int(positions), dtype
        self.scale = float(scale)
        self._code = _dtype(dtype)
        if not 1 <= self.vocab <= 1 << 28:
            raise ValueError(f"vocab must be 1 to 2^28, not {vocab}")
        if not 1 <= self.cols <= 32768:
            raise ValueError(f"cols must be 1 to 32768, not {cols}")
        if not 0 <= self.positions < 1 << 31:
            raise ValueError(f"positions must be 0 to 2^31 - 1, not {positions}")
        self._lib = _lib.load()
        n = C.c_uint64()
        check(self._lib.tatara_op_embedding_backward_workspace(self.positions, self.vocab, self.cols, self._code,
                                                               C.byref(n)))
        self._ws = _Workspaces(n.value)

    def _tokens(self, token) -> int:
        try:
            n, = token.shape
            return n
        except (AttributeError, TypeError, ValueError):
            _wrong("token", token, ("positions",), "i32")

    def forward(self, token, table, y, stream=None) -> None:
        """Writes y [positions, cols]."""
        here, queue = _place(token, stream)
        n = self._tokens(token)
        tp, ts = _rows("table", table, (self.vocab, self.cols), self.dtype, here)
        yp, ys = _rows("y", y, (n, self.cols), self.dtype, here)
        status = self._lib.tatara_op_embedding_forward(
            _dense("token", token, (n,), "i32", here), n, tp, ts, self.vocab, self.cols, self.scale, yp, ys,
            self._code, queue)
        if status:
            check(status)

    def backward(self, dy, token, dtable, stream=None) -> None:
        """Writes dtable [vocab, cols] (overwritten)."""
        here, queue = _place(dy, stream)
        n = self._tokens(token)
        if n > self.positions:
            raise ValueError(f"a backward call takes up to {self.positions} positions, not {n}")
        dp, ds = _rows("dy", dy, (n, self.cols), self.dtype, here)
        ws = self._ws[here]
        status = self._lib.tatara_op_embedding_backward(
            dp, ds, _dense("token", token, (n,), "i32", here), n, self.vocab, self.cols, self.scale,
            _dense("dtable", dtable, (self.vocab, self.cols), "f32", here), self._code, ws.ptr, ws.nbytes, queue)
        if status:
            check(status)
