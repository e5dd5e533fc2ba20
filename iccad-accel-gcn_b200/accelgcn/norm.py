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

import torch

from . import _lib, _rows


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, relu: bool = False, p: float = 0.0, seed: int = 0, offset: int = 0,
               row0: int = 0, step=None, out=None, stats=None, stream=None):
    """dropout(relu(layer_norm(x) * weight + bias)) of x [rows, cols] (float32, bfloat16 or float16 CUDA, any row stride, at
    most 8192 columns); weight and bias float32 [cols] or None.  relu and dropout (p > 0) are optional.  `stats`, float32
    [rows, 2], receives mean and 1 / sqrt(variance + eps) of the rows: what the backward pass needs.  row0: where this
    rank's rows begin in the whole.  step: an int64 on the device that is added to `offset` when the kernel runs (a captured
    graph counts it up to have new masks).  out may be x.  Asynchronous on the current stream (or `stream`)."""
    ldx = _rows.features("x", x)
    with _rows.allocating_on(stream):
        y = out if out is not None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    ldy = _rows.features("out", y, x)
    rows, cols = x.shape
    dev = _lib.device_index(x.device)
    p, seed, offset, row0 = _rows.mask_numbers(p, seed, offset, row0)
    args = (x.data_ptr(), ldx, _rows.array("weight", weight, torch.float32, (cols,), x), _rows.array("bias", bias, torch.float32, (cols,), x),
            float(eps), y.data_ptr(), ldy, _rows.array("stats", stats, torch.float32, (rows, 2), x), rows, cols, _rows.DTYPES[x.dtype],
            1 if relu else 0, p, seed, offset, _rows.step_address(step, x), row0, _rows.stream_of(stream, dev))
    with _lib.on_device(dev):
        rc = _lib.call()(_lib.address("agcn_layer_norm"), *args)
    if rc != 0:
        _lib.check(rc)
    return y


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
    lddy = _rows.features("dy", dy)
    ldx = _rows.features("x", x, dy)
    rows, cols = x.shape
    dev, dtype = _lib.device_index(x.device), _rows.DTYPES[x.dtype]
    if stats is None:
        raise TypeError("layer_norm_backward needs the stats of the forward pass")
    with _rows.allocating_on(stream):
        if dx is None:
            dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if dweight is None and weight is not None:
            dweight = torch.empty(cols, dtype=torch.float32, device=x.device)
        if dbias is None and bias is not None:
            dbias = torch.empty(cols, dtype=torch.float32, device=x.device)
        # of this call alone: calls on other streams, and captured graphs, have their own
        n = _work_floats(dev, rows, cols, dtype) if dweight is not None or dbias is not None else 0
        work = torch.empty(n, dtype=torch.float32, device=x.device) if n else None
    lddx = _rows.features("dx", dx, x)
    p, seed, offset, row0 = _rows.mask_numbers(p, seed, offset, row0)
    args = (dy.data_ptr(), lddy, x.data_ptr(), ldx, _rows.array("stats", stats, torch.float32, (rows, 2), x),
            _rows.array("weight", weight, torch.float32, (cols,), x), _rows.array("bias", bias, torch.float32, (cols,), x), dx.data_ptr(), lddx,
            _rows.array("dweight", dweight, torch.float32, (cols,), x), _rows.array("dbias", dbias, torch.float32, (cols,), x),
            work.data_ptr() if n else None, 4 * n, rows, cols, dtype, 1 if relu else 0, p, seed, offset, _rows.step_address(step, x), row0,
            _rows.stream_of(stream, dev))
    with _lib.on_device(dev):
        rc = _lib.call()(_lib.address("agcn_layer_norm_backward"), *args)
    if rc != 0:
        _lib.check(rc)
    return dx, dweight, dbias
