"""Per device one word in which the kernels of ``attention`` and ``kv4`` record what they met: a
position outside a cache (2), or a bounded device-side wait that gave up (its site, 32 or more, which a
position does not replace)."""
from __future__ import annotations

import threading
from typing import Dict

import torch

from . import _lib

# never reallocated, so captured graphs may hold their addresses
_WORDS: Dict[int, torch.Tensor] = {}
_LOCK = threading.Lock()
OUTSIDE = 2


def word(index: int) -> int:
    """The address of a device's word (made at the first call)."""
    with _LOCK:                                    # synchronising lets other threads in: they wait here
        w = _WORDS.get(index)
        if w is None:
            with torch.cuda.device(index):
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("the first attention or cache call on a device must run outside a CUDA "
                                       "graph capture")
                w = torch.zeros(64, dtype=torch.int32, device=torch.device("cuda", index))
                torch.cuda.synchronize(index)      # zero before any stream uses it
            _WORDS[index] = w
    return w.data_ptr()


def check(device=None) -> None:
    """Synchronise and raise what an attention or cache call on `device` (all devices where None)
    recorded; the word is cleared."""
    for idx, w in list(_WORDS.items()):
        if device is not None and torch.device(device).index not in (None, idx):
            continue
        with torch.cuda.device(idx):
            torch.cuda.synchronize(idx)
            code = int(w[0].item())
            if code:
                w[:1].zero_()
                torch.cuda.synchronize(idx)
        if code == OUTSIDE:
            raise RuntimeError("a position outside the cache")
        if code:
            raise _lib.FlashBFPError(f"a device-side wait gave up (site {code})")


_bind = None


def module():
    """The checks and calls of csrc/attn_bind.cpp (loaded on first use)."""
    global _bind
    if _bind is None:
        from . import fp8
        m = fp8._module()
        m.attn_setup(word)
        _bind = m
    return _bind
