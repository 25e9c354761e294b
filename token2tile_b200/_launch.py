"""Calls into the library on a tensor's device and current stream, at the least cost to the host: the smallest calls of
the operators around the attention take less time on the GPU than their way there."""
from __future__ import annotations

import torch

from ._lib import check

DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}

# torch.cuda.current_stream builds a Python object for every call (2.2 us, these 0.1)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", None)
if _raw_stream is None or _current_device is None:
    _raw_stream = lambda index: torch.cuda.current_stream(index).cuda_stream
    _current_device = torch.cuda.current_device


def launch(dev, what, fn, *args):
    """fn(*args, stream) on the current stream of the CUDA device `dev`; raises RuntimeError for an error code."""
    index = dev.index
    if index is None:      # a tensor's CUDA device has one
        raise ValueError(f"{what}: expected tensors on a CUDA device, got {dev}")
    if _current_device() == index:
        code = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            code = fn(*args, _raw_stream(index))
    if code:
        check(code, what)
