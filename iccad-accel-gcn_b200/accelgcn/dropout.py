"""Dropout of features from a counter-based generator, with the ReLU before it, and its gradient: the Python face of
agcn_dropout / agcn_dropout_backward.

    h = dropout.dropout(y, p=0.5, seed=seed, offset=step)                 # behind a product with its fused ReLU
    dy = dropout.dropout_backward(dh, p=0.5, seed=seed, offset=step, relu=True, x=y)      # x: what went in, or relu of it

The mask is made from (seed, offset, the element's number) in both passes and never stored: give every layer and step another
offset, and both passes of one the same.
"""
from __future__ import annotations

import torch

from . import _lib, _rows


def dropout(x, p: float, seed: int, offset: int = 0, row0: int = 0, step=None, relu: bool = False, out=None, stream=None):
    """dropout(relu(x)) (relu optional) of x [rows, cols] (float32, bfloat16 or float16 CUDA, any row stride): elements are 0 with
    probability p and multiplied by 1 / (1 - p) otherwise.  row0, step: as for norm.layer_norm.  out may be x.  Asynchronous on the
    current stream (or `stream`)."""
    ldx = _rows.features("x", x)
    with _rows.allocating_on(stream):
        y = out if out is not None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    ldy = _rows.features("out", y, x)
    rows, cols = x.shape
    dev = _lib.device_index(x.device)
    p, seed, offset, row0 = _rows.mask_numbers(p, seed, offset, row0)
    args = (x.data_ptr(), ldx, y.data_ptr(), ldy, rows, cols, _rows.DTYPES[x.dtype], 1 if relu else 0, p, seed, offset,
            _rows.step_address(step, x), row0, _rows.stream_of(stream, dev))
    with _lib.on_device(dev):
        rc = _lib.call()(_lib.address("agcn_dropout"), *args)
    if rc != 0:
        _lib.check(rc)
    return y


def dropout_backward(dy, p: float, seed: int, offset: int = 0, row0: int = 0, step=None, relu: bool = False, x=None, out=None, stream=None):
    """Gradient of `dropout` from dy and the same mask numbers; with relu also from the x that went in (or relu(x)).  out may be dy or
    x.  Asynchronous on the current stream (or `stream`)."""
    lddy = _rows.features("dy", dy)
    if relu and x is None:
        raise TypeError("dropout_backward with relu needs the x of the forward pass")
    ldx = _rows.features("x", x, dy) if relu else 0
    with _rows.allocating_on(stream):
        dx = out if out is not None else torch.empty(dy.shape, dtype=dy.dtype, device=dy.device)
    lddx = _rows.features("out", dx, dy)
    rows, cols = dy.shape
    dev = _lib.device_index(dy.device)
    p, seed, offset, row0 = _rows.mask_numbers(p, seed, offset, row0)
    args = (dy.data_ptr(), lddy, x.data_ptr() if relu else None, ldx, dx.data_ptr(), lddx, rows, cols, _rows.DTYPES[dy.dtype],
            1 if relu else 0, p, seed, offset, _rows.step_address(step, dy), row0, _rows.stream_of(stream, dev))
    with _lib.on_device(dev):
        rc = _lib.call()(_lib.address("agcn_dropout_backward"), *args)
    if rc != 0:
        _lib.check(rc)
    return dx
