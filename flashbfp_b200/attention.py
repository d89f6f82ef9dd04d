"""Attention of whole prompts: causal, grouped heads, packed sequences of different lengths.

Rows of several sequences lie back to back, without padding: ``starts`` (int32 [sequences + 1], on the
device) holds where each begins, and after the last where it ends. Lengths stay on the device, so a
call reads nothing back. Forward only: results carry no gradient, whatever their inputs; ``out`` must
not require one while gradients are recorded, must not overlap the inputs, and counts as modified for autograd.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import device_errors
from .device_errors import check as check_device_errors

__all__ = ["prompt_attention", "check_device_errors"]


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor,
                     kv_starts: Optional[torch.Tensor] = None, window: int = 0, scaling: Optional[float] = None,
                     out: Optional[torch.Tensor] = None, err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(q k^T scaling) v for rows q [T, heads, D] and k, v [N, kv_heads, D], all bf16 or all fp16;
    query head h reads key/value head h // (heads // kv_heads). D is a multiple of 8 up to 256; rows and
    heads may be strided (views of fused q | k | v rows), a head's values are contiguous.

    Of a sequence with n query rows and c keys (``kv_starts``; c = n without it) row i stands at place
    c - n + i: it sees the keys up to its own place, with ``window`` > 0 the last ``window`` of them. A
    row that sees no key gives 0. Rows of ``out`` from starts[-1] on are left as they were (in a new
    ``out``: undefined). ``scaling`` is 1 / sqrt(D) by default.

    Scores, softmax statistics and sums are fp32; the weights are rounded to the inputs' type for the
    product with v (fp16: by 2^-11 of themselves, or by 2^-31 of the row's largest), the result once to it. ``err``: an int32 that records a device-side wait which gave up,
    by default one per device that ``check_device_errors`` reads."""
    return (device_errors._bind or device_errors.module()).prompt_attention(q, k, v, starts, kv_starts, window,
                                                                            scaling, out, err)
