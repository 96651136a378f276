"""Launching library calls on the device of their tensors, with little host work.

``launch(name, device, *args)`` calls an entry point whose last argument is the stream, on
``device`` (made current for the call when it is not) and its current stream.  A serving step at
small batches is bound by the host, so what does not change is looked up once.
"""
from __future__ import annotations

from functools import lru_cache

import torch

from . import _lib


@lru_cache(maxsize=None)
def sm_count(index: int) -> int:
    """Multiprocessors of a device (by its index)."""
    return torch.cuda.get_device_properties(index).multi_processor_count


def launch(name: str, device: torch.device, *args) -> None:
    index = device.index
    if torch._C._cuda_getDevice() == index:         # (a tensor is there: CUDA has been set up)
        _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))
        return
    with torch.cuda.device(device):
        _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))
