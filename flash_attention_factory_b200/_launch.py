"""Calling an entry point of the library on torch's current stream, with few instructions.

A decode step on a small batch runs for a few microseconds on the GPU, so the host side of a call counts:
looking up the stream through `torch.cuda.current_stream` and entering a device context take about
3 us together, the raw stream handle and a comparison of device indices 0.2 us.
"""
from __future__ import annotations

import ctypes

import torch

from . import _cabi

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def current_stream(index: int) -> int:
    """cudaStream_t of torch's current stream on device `index`."""
    if _raw_stream is not None:
        return _raw_stream(index)
    return torch.cuda.current_stream(index).cuda_stream


def call(fn, params, index: int, *more) -> None:
    """fn(&params, stream, *more) with device `index` current; raises on a status other than PA_OK."""
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            return call(fn, params, index, *more)
    rc = fn(ctypes.byref(params), current_stream(index), *more)
    if rc != _cabi.PA_OK:
        _cabi.check(rc)
