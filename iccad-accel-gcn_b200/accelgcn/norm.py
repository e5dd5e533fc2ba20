"""Layer norm of features, with the ReLU and the dropout that follow it in a GCN layer, and its gradients: the Python face
of agcn_layer_norm / agcn_layer_norm_backward.

    stats = torch.empty((rows, 2), device=y.device)
    h = norm.layer_norm(y, weight, bias, relu=True, p=0.5, seed=seed, offset=step, stats=stats)       # y = A @ Z
    ...
    dy, dweight, dbias = norm.layer_norm_backward(dh, y, stats, weight, bias, relu=True, p=0.5, seed=seed, offset=step)

One pass over the rows each.  The dropout mask is made from (seed, offset, the element's number) in both and never stored:
give every layer and step another offset, and both passes of one the same.
"""
from __future__ import annotations

import ctypes
import functools
from operator import index

import torch

from . import _lib, _rows


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, relu: bool = False, p: float = 0.0, seed: int = 0, offset: int = 0,
               row0: int = 0, step=None, out=None, stats=None, stream=None):
    """dropout(relu(layer_norm(x) * weight + bias)) of x [rows, cols] (float32, bfloat16 or float16 CUDA, any row stride, at
    most 8192 columns); weight and bias float32 [cols] or None.  relu and dropout (p > 0) are optional.  `stats`, float32
    [rows, 2], receives mean and 1 / sqrt(variance + eps) of the rows: what the backward pass needs.  row0: where this
    rank's rows begin in the whole.  step: an int64 on the device that is added to `offset` when the kernel runs (a captured
    graph counts it up to have new masks).  out may be x.  Asynchronous on the current stream (or `stream`)."""
    rows, cols, ldx, code, dtype, dev = _rows.features("x", x)
    if out is None:
        out, ldy = _rows.empty(rows, cols, dtype, dev, stream), cols
    else:
        ldy = _rows.more_features("out", out, rows, cols, dtype, dev)
    vector = (cols,)
    _rows.run("agcn_layer_norm", dev, stream, x.data_ptr(), ldx, _rows.array("weight", weight, vector, dev), _rows.array("bias", bias, vector, dev),
              float(eps), out.data_ptr(), ldy, None if stats is None else _rows.array("stats", stats, (rows, 2), dev), rows, cols, code,
              1 if relu else 0, float(p), index(seed), index(offset), None if step is None else _rows.step_address(step, dev), index(row0))
    return out


@functools.lru_cache(maxsize=4096)
def _work_floats(dev: int, rows: int, cols: int, dtype: int) -> int:
    n = ctypes.c_int64()
    with _lib.on_device(dev):
        _lib.check(_lib.load().agcn_layer_norm_backward_work(rows, cols, dtype, ctypes.byref(n)))
    return n.value // 4


def layer_norm_backward(dy, x, stats, weight=None, bias=None, relu: bool = False, p: float = 0.0, seed: int = 0, offset: int = 0,
                        row0: int = 0, step=None, dx=None, dweight=None, dbias=None, stream=None):
    """Gradients of `layer_norm`: (dx, dweight, dbias) from dy, and the x, stats, weight, bias and mask numbers of the forward
    pass.  dweight and dbias are float32 [cols], overwritten, the same bits from run to run; None where there was no weight (bias)
    and no array is given for it.  dx may be dy or x.  Asynchronous on the current stream (or `stream`)."""
    rows, cols, ldx, code, dtype, dev = _rows.features("x", x)
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
    vector = (cols,)
    _rows.run("agcn_layer_norm_backward", dev, stream, dy.data_ptr(), lddy, x.data_ptr(), ldx, _rows.array("stats", stats, (rows, 2), dev),
              _rows.array("weight", weight, vector, dev), _rows.array("bias", bias, vector, dev), dx.data_ptr(), lddx,
              _rows.array("dweight", dweight, vector, dev), _rows.array("dbias", dbias, vector, dev), None if work is None else work.data_ptr(), 4 * n,
              rows, cols, code, 1 if relu else 0, float(p), index(seed), index(offset), None if step is None else _rows.step_address(step, dev),
              index(row0))
    return dx, dweight, dbias
