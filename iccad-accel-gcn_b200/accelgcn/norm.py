"""Layer norm of features, with the ReLU and the dropout that follow it in a GCN layer, and its gradients: the Python face
of agcn_layer_norm / agcn_layer_norm_backward.

    stats = torch.empty((rows, 2), device=y.device)
    h = norm.layer_norm(y, weight, bias, relu=True, p=0.5, seed=seed, offset=step, stats=stats)       # y = A @ Z
    ...
    dy, dweight, dbias = norm.layer_norm_backward(dh, y, stats, weight, bias, relu=True, p=0.5, seed=seed, offset=step)

One pass over the rows each.  The dropout mask is made from (seed, offset, the element's number) in both and never stored:
give every layer and step another offset, and both passes of one the same.  These are plain functions on tensors: autograd does not see them.
"""
from __future__ import annotations

import ctypes
import functools
from operator import index

import torch

from . import _lib, _rows

_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream
_forward = _backward = None


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, relu: bool = False, p: float = 0.0, seed: int = 0, offset: int = 0,
               row0: int = 0, step=None, out=None, stats=None, stream=None):
    """dropout(relu(layer_norm(x) * weight + bias)) of x [rows, cols] (float32, bfloat16 or float16 CUDA, any row stride, at
    most 8192 columns); weight and bias float32 [cols] or None.  relu and dropout (p > 0) are optional; eps is 1e-30 to 1e30.  `stats`, float32
    [rows, 2], receives mean and 1 / sqrt(variance + eps) of the rows: what the backward pass needs.  row0: where this
    rank's rows begin in the whole.  step: an int64 on the device that is added to `offset` when the kernel runs (a captured
    graph counts it up to have new masks).  out may be x.  Asynchronous on the current stream (or `stream`)."""
    global _forward
    rows, cols, ldx, code, dtype, dev = _rows.features("x", x)
    if _current_device() != dev:
        with torch.cuda.device(dev):
            return layer_norm(x, weight, bias, eps, relu, p, seed, offset, row0, step, out, stats, stream)
    if _forward is None:
        _forward = _rows.function("agcn_layer_norm")
    if out is None:
        out, ldy = _rows.empty(rows, cols, dtype, dev, stream), cols
    else:
        ldy = _rows.more_features("out", out, rows, cols, dtype, dev)
    rc = _forward(x.data_ptr(), ldx, None if weight is None else _rows.array("weight", weight, cols, dev),
                  None if bias is None else _rows.array("bias", bias, cols, dev), float(eps), out.data_ptr(), ldy,
                  None if stats is None else _rows.stats("stats", stats, rows, dev), rows, cols, code, 1 if relu else 0, float(p), index(seed),
                  index(offset), None if step is None else _rows.step_address(step, dev), index(row0),
                  _raw_stream(dev) if stream is None else stream.cuda_stream)
    if rc != 0:
        _lib.check(rc)
    return out


@functools.lru_cache(maxsize=4096)
def _work_floats(dev: int, rows: int, cols: int, dtype: int) -> int:
    n = ctypes.c_int64()
    _lib.check(_lib.load().agcn_layer_norm_backward_work(rows, cols, dtype, ctypes.byref(n)))      # of the current device: `dev`
    return n.value // 4


def layer_norm_backward(dy, x, stats, weight=None, bias=None, relu: bool = False, p: float = 0.0, seed: int = 0, offset: int = 0,
                        row0: int = 0, step=None, dx=None, dweight=None, dbias=None, stream=None):
    """Gradients of `layer_norm`: (dx, dweight, dbias) from dy, and the x, stats, weight, bias and mask numbers of the forward
    pass.  dweight and dbias are float32 [cols], overwritten, the same bits from run to run; None where there was no weight (bias)
    and no array is given for it.  dx may be dy or x.  Asynchronous on the current stream (or `stream`)."""
    global _backward
    rows, cols, ldx, code, dtype, dev = _rows.features("x", x)
    if _current_device() != dev:
        with torch.cuda.device(dev):
            return layer_norm_backward(dy, x, stats, weight, bias, relu, p, seed, offset, row0, step, dx, dweight, dbias, stream)
    if _backward is None:
        _backward = _rows.function("agcn_layer_norm_backward")
    lddy = _rows.more_features("dy", dy, rows, cols, dtype, dev)
    if stats is None:
        raise TypeError("layer_norm_backward needs the stats of the forward pass")
    if dx is None:
        dx, lddx = _rows.empty(rows, cols, dtype, dev, stream), cols
    else:
        lddx = _rows.more_features("dx", dx, rows, cols, dtype, dev)
    if (dweight is None and weight is not None) or (dbias is None and bias is not None):
        with _rows.allocating_on(stream):
            if dweight is None and weight is not None:
                dweight = torch.empty(cols, dtype=_rows.F32, device=x.device)
            if dbias is None and bias is not None:
                dbias = torch.empty(cols, dtype=_rows.F32, device=x.device)
    work, n = None, 0
    if dweight is not None or dbias is not None:
        n = _work_floats(dev, rows, cols, code)
        if n:
            # of this call alone: calls on other streams, and captured graphs, have their own
            with _rows.allocating_on(stream):
                work = torch.empty(n, dtype=_rows.F32, device=x.device)
    rc = _backward(dy.data_ptr(), lddy, x.data_ptr(), ldx, _rows.stats("stats", stats, rows, dev),
                   None if weight is None else _rows.array("weight", weight, cols, dev), None if bias is None else _rows.array("bias", bias, cols, dev),
                   dx.data_ptr(), lddx, None if dweight is None else _rows.array("dweight", dweight, cols, dev),
                   None if dbias is None else _rows.array("dbias", dbias, cols, dev), None if work is None else work.data_ptr(), 4 * n, rows, cols, code,
                   1 if relu else 0, float(p), index(seed), index(offset), None if step is None else _rows.step_address(step, dev), index(row0),
                   _raw_stream(dev) if stream is None else stream.cuda_stream)
    if rc != 0:
        _lib.check(rc)
    return dx, dweight, dbias
