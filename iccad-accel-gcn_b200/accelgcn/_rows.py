"""What the row-wise operators (norm, dropout) ask of their tensors before the library sees a pointer.

A call on a graph of a few thousand nodes takes 3 us on the GPU; every attribute of a tensor that Python asks for is 50 to
100 ns, so each is asked for once and compared in the cheapest way."""
from __future__ import annotations

import contextlib
import functools

import torch

from . import _lib

F32 = torch.float32
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}        # AGCN_F32, AGCN_BF16, AGCN_F16


def features(name, t):
    """(rows, cols, row stride, type code, type, device index) of [rows, cols] features with unit column stride."""
    dtype, dev = t.dtype, t.get_device()
    code = DTYPES.get(dtype)
    if dev < 0 or code is None:
        raise TypeError(f"{name} must be a float32, bfloat16 or float16 CUDA tensor")
    shape = t.shape
    if len(shape) != 2:
        raise ValueError(f"{name} must be [rows, cols]")
    rows, cols = shape
    ld, inner = t.stride()
    if rows <= 1:
        ld = cols
    if (inner != 1 and cols > 1) or ld < cols:
        raise ValueError(f"{name} must have unit column stride and rows that do not overlap (strides {ld}, {inner}): copy it first")
    return rows, cols, ld, code, dtype, dev


def more_features(name, t, rows, cols, dtype, dev):
    """The row stride of features that must be like others."""
    if t.dtype is not dtype or t.get_device() != dev:
        raise ValueError(f"{name} must have the type and device of the other features")
    shape = t.shape
    if len(shape) != 2 or shape[0] != rows or shape[1] != cols:
        raise ValueError(f"{name} must be [{rows}, {cols}] like the other features")
    ld, inner = t.stride()
    if rows <= 1:
        ld = cols
    if (inner != 1 and cols > 1) or ld < cols:
        raise ValueError(f"{name} must have unit column stride and rows that do not overlap (strides {ld}, {inner}): copy it first")
    return ld


def array(name, t, count, dev):
    """Address of a contiguous float32 array of `count` elements on the features' device."""
    if t.dtype is not F32 or t.get_device() != dev:
        raise TypeError(f"{name} must be a float32 tensor on the features' device")
    if t.numel() != count or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous, of {count} elements")
    return t.data_ptr()


def stats(name, t, rows, dev):
    """Address of the rows' statistics [rows, 2]."""
    if t.shape != (rows, 2):
        raise ValueError(f"{name} must be [{rows}, 2]")
    return array(name, t, 2 * rows, dev)


def step_address(step, dev):
    """Address of the device counter that is added to a mask's offset."""
    if step.dtype is not torch.int64 or step.get_device() != dev or step.numel() != 1:
        raise TypeError("step must be one int64 on the features' device")
    return step.data_ptr()


_NO_CONTEXT = contextlib.nullcontext()


def allocating_on(stream):
    """Memory made inside belongs to `stream`, where it is used (None: the current one)."""
    return _NO_CONTEXT if stream is None else torch.cuda.stream(stream)


def empty(rows, cols, dtype, dev, stream):
    with allocating_on(stream):
        return torch.empty((rows, cols), dtype=dtype, device=f"cuda:{dev}")


def function(name):
    """The library's function: called with its arguments, it returns its status."""
    _lib.load()
    return functools.partial(_lib.call(), _lib.address(name))
