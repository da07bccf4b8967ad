"""Device-tensor plumbing of the decoding operators: checks, strides, workspaces.

The operators take torch CUDA tensors (a cache lives on the device); only
pointers, sizes and strides cross the C ABI.  Work goes to the current stream
of the tensors' device.

A decoding loop calls these functions once a layer and step with tensors of
the same form, and a step of a small model is a few microseconds, so what
depends on the tensors' form alone (types, shapes, strides, device) is checked
and laid out once for each form (`Forms`).
"""
from __future__ import annotations

import ctypes as C

import torch

from .. import _native as N

TYPES = {torch.float32: N.TYPE_F32, torch.float16: N.TYPE_F16, torch.bfloat16: N.TYPE_BF16}


def form(t):
    """What of a tensor the checks and the C ABI's sizes and strides depend on."""
    return None if t is None else (t.dtype, t.get_device(), t.shape, t.stride())


class Forms(dict):
    """What was found for a call's form; bounded, since a form costs nothing but its checks."""

    def keep(self, key, found):
        if len(self) >= 1024:
            self.clear()
        self[key] = found
        return found


def check_dev(dev, **tensors):
    """Every tensor on the CUDA device `dev` (they are all read there)."""
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError("%s is on %s, not on %s" % (name, t.device, dev))


def check_i32(t, ndim, name):
    if t.dtype is not torch.int32 or t.dim() != ndim:
        raise ValueError("%s must be an int32 tensor of %d dimension(s)" % (name, ndim))
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError("%s must be contiguous in its last dimension" % name)


def i64s(*values):
    """The values as a host int64 array (shapes and strides of the C ABI)."""
    return (C.c_int64 * len(values))(*values)


def needed(fn, *args):
    """What a workspace query says."""
    out = C.c_int64()
    N.call(fn, *args, C.byref(out))
    return out.value


_workspaces = {}


def workspace(op, dev, stream, nbytes):
    """Scratch of one operator on one stream (its handle): calls on a stream
    follow each other, so they share it (nothing in it lasts from call to
    call).  Under stream capture every call gets its own out of the graph's
    memory."""
    if nbytes == 0:
        return None
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=dev)
    key = (op, dev.index, stream)
    buf = _workspaces.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = _workspaces[key] = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    return buf


def ptr(t):
    return None if t is None else t.data_ptr()


def stream(dev):
    """The handle of the device's current stream."""
    return torch.cuda.current_stream(dev).cuda_stream


if hasattr(torch._C, "_cuda_getCurrentRawStream"):  # the same without the objects in between
    def stream(dev):  # noqa: F811
        return torch._C._cuda_getCurrentRawStream(dev.index)


def call(name, dev, *args):
    """N.call with the tensors' device as the current one."""
    if torch.cuda.current_device() == dev.index:
        N.call(name, *args)
    else:
        with torch.cuda.device(dev):
            N.call(name, *args)
