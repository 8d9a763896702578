"""The current device and stream, for calls that are made often: ``torch.cuda.device`` and
``torch.cuda.current_stream`` cost several microseconds, as much as a launch."""
import contextlib

import torch

_NO_SWITCH = contextlib.nullcontext()


def current_device(device):
    """``torch.cuda.device(device)`` where that is not the current one already."""
    return _NO_SWITCH if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def raw_stream(device):
    """The address of the device's current stream: ``current_stream(device).cuda_stream`` without the object."""
    return torch._C._cuda_getCurrentRawStream(device.index)
