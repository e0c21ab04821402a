"""What the wrappers of the attention and logits operators do around a library
call, kept short: for short sequences this is most of the call's time."""
from __future__ import annotations

import contextlib

import torch

__all__ = ["on_device", "raw_stream", "once_when_recorded", "same_as_saved"]

_HERE = contextlib.nullcontext()


def on_device(device):
    """A context in which `device` is current; nothing to enter where it is already."""
    index = device.index
    return _HERE if torch._C._cuda_getDevice() == index else torch.cuda.device(index)


def raw_stream(device) -> int:
    """cudaStream_t of the device's current stream."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def once_when_recorded(backward):
    """``once_differentiable`` for a backward that autograd records
    (create_graph=True): a second derivative raises.  Where nothing is recorded it
    costs nothing."""
    once = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return (once if torch.is_grad_enabled() else backward)(ctx, *grads)
    return staticmethod(run)


def same_as_saved(t, shape, dtype, device):
    """Checks a tensor that autograd kept for the backward.  A saved-tensor hook
    (``torch.autograd.graph.save_on_cpu``, activation offload) may give it back with
    other strides, never with another shape, type or device."""
    assert t.shape == shape and t.dtype is dtype and t.device == device, \
        "a saved tensor came back with another shape, dtype or device"
    return t
