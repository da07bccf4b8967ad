"""Decoding: a paged key/value cache, attention of new tokens over it, and beam search on the device.

The operators have no backward pass; a tensor that requires a gradient is
refused outside torch.no_grad().
"""
from .beam import beam_reorder, beam_select  # noqa: F401
from .gpt2 import GPT2Generator  # noqa: F401
from .paged import paged_append, paged_attention  # noqa: F401
