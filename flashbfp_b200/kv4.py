"""The key/value cache in 4 bits: rows are quantised as they are written, read back as plain rows,
or attended to as they are held.

A cached head of D values is cut into groups of 32 (the last may be shorter). A group's scale is the
bf16 nearest to max|x| / 7, and a value is held as x / scale rounded to the nearest whole number (ties to
even), plus 8, in 4 bits: 4.5 bits a value with the scales. Whole numbers end at -7 and 7 (only a scale among
bf16's lowest subnormals, below 2^-130, lies so far from max|x| / 7 that a quotient passes them). A group with an infinity or a NaN reads
back as NaN. Rows that enter are plain rows of any float type; what is already rounded stays what it
is, so a row that is read back and written again is held as it was.

``KV4Cache`` holds keys and values [sequences, kv_heads, positions, ...]. Positions are int32 tensors on
the device, and so are lengths: calls read nothing back and can be captured. A position outside the
cache is skipped and recorded (``check_device_errors`` raises it). Forward only, as ``attention``; what a
call writes must not overlap what it reads.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from . import _lib, device_errors
from .device_errors import check as check_device_errors

__all__ = ["KV4Cache", "empty_cache", "kv4_write", "kv4_append", "kv4_read", "kv4_attention", "check_device_errors"]


class KV4Cache(NamedTuple):
    k_values: torch.Tensor                # uint8 [sequences, kv_heads, positions, 16 ceil(D / 32)]
    k_scales: torch.Tensor                # bfloat16 [sequences, kv_heads, positions, ceil(D / 32)]
    v_values: torch.Tensor
    v_scales: torch.Tensor
    head_dim: int

    @property
    def positions(self) -> int:
        return self.k_values.shape[2]

    def sequence(self, b: int) -> "KV4Cache":
        """Sequence b alone (a view)."""
        return KV4Cache(*(t[b:b + 1] for t in self[:4]), self.head_dim)


def empty_cache(sequences: int, kv_heads: int, positions: int, head_dim: int, device) -> KV4Cache:
    """A cache of zeros; ``positions`` is rounded up to a multiple of 32."""
    if head_dim < 8 or head_dim > 256 or head_dim % 8:
        raise ValueError(f"head_dim {head_dim} is not a multiple of 8 up to 256")
    if min(sequences, kv_heads, positions) < 1:
        raise ValueError("a cache holds at least one sequence, head and position")
    g = -(-head_dim // 32)
    shape = (sequences, kv_heads, -(-positions // 32) * 32)
    made = [torch.zeros(*shape, n, dtype=t, device=device)
            for n, t in ((16 * g, torch.uint8), (g, torch.bfloat16)) * 2]
    return KV4Cache(*made, head_dim)


def _module():
    return device_errors._bind or device_errors.module()


def kv4_write(cache: KV4Cache, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor,
              starts: Optional[torch.Tensor] = None, err: Optional[torch.Tensor] = None) -> None:
    """Quantise rows k, v [T, kv_heads, D] (bf16, fp16 or fp32) into the cache: row r of sequence b goes
    to position pos[b] + r - starts[b]. ``starts`` (int32 [sequences + 1]) packs the rows of several
    sequences; without it there is one row per sequence. Rows from starts[-1] on are not written."""
    _module().kv4_write(cache, k, v, pos, starts, err)


def kv4_append(cache: KV4Cache, qkv: torch.Tensor, q_norm: torch.Tensor, k_norm: torch.Tensor, eps: float,
               cos: torch.Tensor, sin: torch.Tensor, pos: torch.Tensor, q_out: torch.Tensor,
               starts: Optional[torch.Tensor] = None, err: Optional[torch.Tensor] = None) -> None:
    """A decoder layer's step to the cache in one launch: of fused bf16 rows q | k | v [T, (heads + 2 kv_heads) D],
    RMSNorm (weights 1 + w) of every q and k head, the rotary embedding with the bf16 rows cos, sin
    [positions, D] at the row's position, q to q_out [T, heads, D], k and v into the cache as ``kv4_write``
    puts them. D is a multiple of 16."""
    _module().kv4_check(cache, q_out)
    values, d = cache.k_values, cache.head_dim
    kvh = values.shape[1]
    what = {"qkv": qkv, "q_norm": q_norm, "k_norm": k_norm, "cos": cos, "sin": sin, "q_out": q_out}
    for name, t in what.items():
        _lib.require_cuda(t, name)
        if t.dtype != torch.bfloat16 or not t.is_contiguous() or t.device != values.device:
            raise ValueError(f"{name} must be contiguous bfloat16 on {values.device}")
    rows, width = qkv.shape if qkv.dim() == 2 else (0, 0)
    heads = width // d - 2 * kvh
    if heads < 1 or width != (heads + 2 * kvh) * d or q_out.numel() != rows * heads * d:
        raise ValueError(f"qkv {tuple(qkv.shape)} and q_out {tuple(q_out.shape)} do not hold heads of {d} beside "
                         f"2 x {kvh}")
    if q_norm.numel() != d or k_norm.numel() != d or cos.shape != sin.shape or cos.dim() != 2 or cos.shape[1] != d:
        raise ValueError("norm weights and cos / sin rows must have one value per value of a head")
    if cos.shape[0] < cache.positions:
        raise ValueError(f"cos and sin hold {cos.shape[0]} positions, the cache {cache.positions}")
    for name, t, n in (("pos", pos, values.shape[0]), ("starts", starts, values.shape[0] + 1), ("err", err, 1)):
        if t is not None and (t.dtype != torch.int32 or t.numel() != n or not t.is_contiguous() or t.device != values.device):
            raise ValueError(f"{name} must be {n} contiguous int32 on {values.device}")
    if starts is None and rows != values.shape[0]:
        raise ValueError(f"{rows} rows for {values.shape[0]} sequences: pass starts")
    if rows == 0:
        return
    c = _lib.KV4CacheStruct(*(t.data_ptr() for t in cache[:4]), *values.shape[:3], d)
    P = _lib.ptr
    with torch.cuda.device(values.device):
        word = P(err) if err is not None else device_errors.word(values.device.index)
        _lib.check(_lib.lib().fbfp_kv4_append(ctypes.byref(c), P(qkv), rows, heads, P(q_norm), P(k_norm), float(eps),
                                              P(cos), P(sin), P(pos), P(starts), P(q_out), word,
                                              _lib.stream_ptr(values.device)), "fbfp_kv4_append")
    for t in (*cache[:4], q_out):
        torch.autograd.graph.increment_version(t)


def kv4_read(cache: KV4Cache, first: torch.Tensor, starts: torch.Tensor, rows: Optional[int] = None,
             dtype: torch.dtype = torch.bfloat16, out: Optional[Sequence[torch.Tensor]] = None,
             err: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows k, v [rows, kv_heads, D] of ``dtype`` from the cache: row r of sequence b comes from position
    first[b] + r - starts[b]. ``out`` gives both tensors (any strides between rows and heads), else
    ``rows`` and ``dtype`` make them; rows from starts[-1] on are left as they were. The two must not overlap."""
    if out is None:
        if rows is None:
            raise ValueError("kv4_read needs the number of rows, or out")
        shape = (rows, cache.k_values.shape[1], cache.head_dim)
        out = [torch.empty(shape, dtype=dtype, device=cache.k_values.device) for _ in range(2)]
    k, v = out
    _module().kv4_read(cache, first, starts, k, v, err)
    return k, v


def kv4_attention(q: torch.Tensor, cache: KV4Cache, pos: torch.Tensor, window: int = 0,
                  scaling: Optional[float] = None, out: Optional[torch.Tensor] = None,
                  err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the newest rows of each sequence over its cache. q is [sequences, heads, D] (one row
    each) or [sequences, rows, heads, D], bf16 or fp16; row i of sequence b stands at position pos[b] + i
    (its keys and values are in the cache already) and sees the positions up to its own, with ``window``
    > 0 the last ``window`` of them; query head h reads key/value head h // (heads // kv_heads). A row
    whose position is outside the cache gives 0. The result has q's shape and type.

    The cached whole numbers enter the products as they are; scales, scores, softmax statistics and sums
    are fp32. Two roundings come before the result's own. Queries enter as fp16 under a power of two for each
    row and head: bf16 values below 2^-29 of its largest lose bits, those below 2^-37 are 0. A softmax weight times
    its value's scale is rounded to fp16: by 2^-11 of itself, or, where it is small beside the row's others, by
    at most 2^-19 of the largest weight times the smallest scale."""
    return _module().kv4_attention(q, cache, pos, window, scaling, out, err)
