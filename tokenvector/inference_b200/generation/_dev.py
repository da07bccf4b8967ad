"""Device-tensor plumbing of the decoding operators.

The operators take torch CUDA tensors (a cache lives on the device), check
them, and put their work on the current stream of the tensors' device;
`ops` does so natively (csrc/tvq_torch.cpp), since a decoding loop makes these
calls once a layer and step.
"""
from __future__ import annotations

import os

import torch

from .. import _native as N

try:
    from .. import _tvq_torch as ops  # noqa: F401
except ImportError as e:
    raise RuntimeError("_tvq_torch.so cannot be loaded from %s (%s); run tokenvector/inference_b200/build.py"
                       % (os.path.dirname(N.LIB_PATH), e)) from e


def ptr(t):
    return None if t is None else t.data_ptr()


def stream(dev):
    """The handle of the device's current stream."""
    return torch.cuda.current_stream(dev).cuda_stream


def call(name, dev, *args):
    """N.call with the tensors' device as the current one."""
    if torch.cuda.current_device() == dev.index:
        N.call(name, *args)
    else:
        with torch.cuda.device(dev):
            N.call(name, *args)
