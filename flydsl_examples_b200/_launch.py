"""Host-side odds and ends of a launch: the current stream as a plain handle, switching device or stream only when needed."""
from __future__ import annotations

import contextlib
import functools
from typing import Optional

import torch

_NOTHING = contextlib.nullcontext()


def raw_stream(index: int) -> int:
    """cudaStream_t of the device's current stream, without building a torch.cuda.Stream."""
    return torch._C._cuda_getCurrentRawStream(index)


def on_device(index: int, stream: Optional[torch.cuda.Stream]):
    """A context in which `index` is the current device and `stream` (None: the device's current one) its current stream."""
    if stream is not None:
        if stream.device_index != index:
            raise ValueError(f"the stream belongs to cuda:{stream.device_index}, the tensors are on cuda:{index}")
        return torch.cuda.stream(stream)  # also makes the stream's device the current one
    return _NOTHING if is_current(index) else torch.cuda.device(index)


def is_current(index: int) -> bool:
    return torch._C._cuda_getDevice() == index


@functools.lru_cache(maxsize=None)
def device_sms(index: int) -> int:
    return torch.cuda.get_device_properties(index).multi_processor_count
