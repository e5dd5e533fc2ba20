"""What the row-wise operators (norm, dropout) ask of their tensors before the library sees a pointer."""
from __future__ import annotations

import contextlib
from operator import index

import torch

from . import _lib

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}        # AGCN_F32, AGCN_BF16, AGCN_F16


def features(name, t, like=None):
    """Checks [rows, cols] features with unit column stride (of the shape, type and device of `like`); returns the row stride."""
    if not t.is_cuda or t.dtype not in DTYPES:
        raise TypeError(f"{name} must be a float32, bfloat16 or float16 CUDA tensor")
    if t.dim() != 2:
        raise ValueError(f"{name} must be [rows, cols]")
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{name} must have the shape, type and device of the other features")
    rows, cols = t.shape
    ld, inner = t.stride()
    if cols > 1 and inner != 1:
        raise ValueError(f"{name} must have unit column stride")
    if rows <= 1:
        return cols
    if ld < cols:
        raise ValueError(f"rows of {name} overlap (stride {ld}): copy it first")
    return ld


def array(name, t, dtype, shape, like):
    """Checks a contiguous array on the features' device; returns its address (None where there is none)."""
    if t is None:
        return None
    if not t.is_cuda or t.dtype != dtype or t.device != like.device:
        raise TypeError(f"{name} must be a {dtype} tensor on the features' device")
    if tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous {list(shape)}")
    return t.data_ptr()


def step_address(step, like):
    """Address of the device counter that is added to a mask's offset."""
    if step is None:
        return None
    if not step.is_cuda or step.dtype != torch.int64 or step.device != like.device or step.numel() != 1:
        raise TypeError("step must be one int64 on the features' device")
    return step.data_ptr()


def mask_numbers(p, seed, offset, row0):
    """As the library takes them: what is no integer must not become a double on the way."""
    return float(p), index(seed), index(offset), index(row0)


_NO_CONTEXT = contextlib.nullcontext()


def allocating_on(stream):
    """Memory made inside belongs to `stream`, where it is used (None: the current one)."""
    return _NO_CONTEXT if stream is None else torch.cuda.stream(stream)


def stream_of(stream, dev):
    return stream.cuda_stream if stream is not None else _lib.raw_stream(dev)
