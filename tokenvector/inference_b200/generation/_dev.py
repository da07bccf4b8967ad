"""Device-tensor plumbing of the decoding operators: checks, strides, workspaces.

The operators take torch CUDA tensors (a cache lives on the device); only
pointers, sizes and strides cross the C ABI.  Work goes to the current stream
of the tensors' device.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from .. import _native as N

TYPES = {torch.float32: N.TYPE_F32, torch.float16: N.TYPE_F16, torch.bfloat16: N.TYPE_BF16}


def check_dev(dev, **tensors):
    """Every tensor on the CUDA device `dev` (they are all read there)."""
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError("%s is on %s, not on %s" % (name, t.device, dev))


def check_i32(t, ndim, name):
    if t.dtype is not torch.int32 or t.dim() != ndim:
        raise ValueError("%s must be an int32 tensor of %d dimension(s)" % (name, ndim))
    if ndim and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError("%s must be contiguous in its last dimension" % name)


@functools.lru_cache(maxsize=512)
def i64s(*values):
    """The values as a host int64 array (shapes and strides of the C ABI)."""
    return (C.c_int64 * len(values))(*values)


@functools.lru_cache(maxsize=512)
def needed(fn, *args):
    """What a workspace query says."""
    out = C.c_int64()
    N.call(fn, *args, C.byref(out))
    return out.value


_workspaces = {}


def workspace(op, dev, nbytes):
    """Scratch of one operator on the current stream of `dev`: calls on one
    stream follow each other, so they share it (nothing in it lasts from
    call to call).  Under stream capture every call gets its own out of the
    graph's memory."""
    if nbytes == 0:
        return None
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=dev)
    key = (op, dev.index, torch.cuda.current_stream(dev).cuda_stream)
    buf = _workspaces.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = _workspaces[key] = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    return buf


def ptr(t):
    return None if t is None else t.data_ptr()


def stream(dev):
    return torch.cuda.current_stream(dev).cuda_stream
