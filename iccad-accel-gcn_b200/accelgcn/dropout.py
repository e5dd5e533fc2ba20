"""Dropout of features from a counter-based generator, with the ReLU before it, and its gradient: the Python face of
agcn_dropout / agcn_dropout_backward.

    h = dropout.dropout(y, p=0.5, seed=seed, offset=step)                 # behind a product with its fused ReLU
    dy = dropout.dropout_backward(dh, p=0.5, seed=seed, offset=step, relu=True, x=y)      # x: what went in, or relu of it

The mask is made from (seed, offset, the element's number) in both passes and never stored: give every layer and step another
offset, and both passes of one the same.  These are plain functions on tensors: autograd does not see them.
"""
from __future__ import annotations

from operator import index

import torch

from . import _lib, _rows

_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream
_forward = _backward = None


def dropout(x, p: float, seed: int, offset: int = 0, row0: int = 0, step=None, relu: bool = False, out=None, stream=None):
    """dropout(relu(x)) (relu optional) of x [rows, cols] (float32, bfloat16 or float16 CUDA, any row stride): elements are 0 with
    probability p and multiplied by 1 / (1 - p) otherwise.  row0, step: as for norm.layer_norm.  out may be x.  Asynchronous on the
    current stream (or `stream`)."""
    global _forward
    rows, cols, ldx, code, dtype, dev = _rows.features("x", x)
    if _current_device() != dev:
        with torch.cuda.device(dev):
            return dropout(x, p, seed, offset, row0, step, relu, out, stream)
    if _forward is None:
        _forward = _rows.function("agcn_dropout")
    if out is None:
        out, ldy = _rows.empty(rows, cols, dtype, dev, stream), cols
    else:
        ldy = _rows.more_features("out", out, rows, cols, dtype, dev)
    rc = _forward(x.data_ptr(), ldx, out.data_ptr(), ldy, rows, cols, code, 1 if relu else 0, float(p), index(seed), index(offset),
                  None if step is None else _rows.step_address(step, dev), index(row0), _raw_stream(dev) if stream is None else stream.cuda_stream)
    if rc != 0:
        _lib.check(rc)
    return out


def dropout_backward(dy, p: float, seed: int, offset: int = 0, row0: int = 0, step=None, relu: bool = False, x=None, out=None, stream=None):
    """Gradient of `dropout` from dy and the same mask numbers; with relu also from the x that went in (or relu(x)).  out may be dy or
    x.  Asynchronous on the current stream (or `stream`)."""
    global _backward
    rows, cols, lddy, code, dtype, dev = _rows.features("dy", dy)
    if _current_device() != dev:
        with torch.cuda.device(dev):
            return dropout_backward(dy, p, seed, offset, row0, step, relu, x, out, stream)
    if _backward is None:
        _backward = _rows.function("agcn_dropout_backward")
    if not relu:
        x_address, ldx = None, 0
    elif x is None:
        raise TypeError("dropout_backward with relu needs the x of the forward pass")
    else:
        x_address, ldx = x.data_ptr(), _rows.more_features("x", x, rows, cols, dtype, dev)
    if out is None:
        out, lddx = _rows.empty(rows, cols, dtype, dev, stream), cols
    else:
        lddx = _rows.more_features("out", out, rows, cols, dtype, dev)
    rc = _backward(dy.data_ptr(), lddy, x_address, ldx, out.data_ptr(), lddx, rows, cols, code, 1 if relu else 0, float(p), index(seed), index(offset),
                   None if step is None else _rows.step_address(step, dev), index(row0), _raw_stream(dev) if stream is None else stream.cuda_stream)
    if rc != 0:
        _lib.check(rc)
    return out
