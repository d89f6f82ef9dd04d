"""Block-scaled 8-bit linears: e4m3 rows with one power-of-two scale per 128 values.

``quantize_fp8``, ``rmsnorm_fp8`` and ``geglu_fp8`` make such rows (from plain rows, from an
RMSNorm with the residual's addition, from the GeGLU activation); ``fp8_linear`` multiplies two of
them on the tensor cores' block-scaled path, with fp32 accumulation. A weight matrix is one more
``quantize_fp8``, done once at load time. Decoders take such weights as their layers' linears
(``decode.GemmaDecoder``).

An operand is an ``Fp8Rows``: ``values`` (float8_e4m3fn [m, k], rows a multiple of 16 bytes apart)
and ``scales`` (float8_e8m0fnu, one byte per row and 128 values in tiles of 128 rows x 4 blocks:
[ceil(m / 128), ceil(k / 512), 32, 4, 4], element [row / 128, block / 4, row % 32,
row % 128 / 32, block % 4]), the layout the tensor core's scale copies take as it is. A scale is
the smallest power of two (at least 2^-127) that brings its block into e4m3's range of 448. A
block with an infinity or a NaN becomes NaN, scale and values, and so does the output row (or
column) of a product that reads it. Everything runs on the GPU; the results of a call follow its
inputs' stream order on the current stream.

Forward only: results carry no gradient, whatever their inputs. What a call writes in place (the
residual, ``out``) must not require one while gradients are recorded, and counts as modified for
autograd. ``out`` must not overlap the inputs, nor the residual the other inputs, unless x is the
residual itself.
"""
from __future__ import annotations

import importlib.util
import os
import threading
from typing import Dict, NamedTuple, Optional

import torch

from . import _lib, build

_F8, _E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


class Fp8Rows(NamedTuple):
    values: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self) -> torch.Size:
        return self.values.shape

    def scale_matrix(self) -> torch.Tensor:
        """The scales as fp32 [m, ceil(k / 128)]."""
        m, k = self.values.shape
        t = self.scales.view(torch.uint8)
        codes = t.permute(0, 3, 2, 1, 4).reshape(t.shape[0] * 128, t.shape[1] * 4)[:m, :-(-k // 128)].int()
        s = torch.ldexp(torch.ones_like(codes, dtype=torch.float32), codes - 127)
        return torch.where(codes == 255, torch.full_like(s, float("nan")), s)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The rows the operand stands for: values * scale, rounded to `dtype` (exact in fp32, and in
        bf16 where the scale is at least 2^-124)."""
        k = self.values.shape[1]
        s = self.scale_matrix().repeat_interleave(128, dim=1)[:, :k]
        return (self.values.float() * s).to(dtype)


def scale_shape(m: int, k: int) -> tuple:
    return (-(-m // 128), -(-k // 512), 32, 4, 4)


def empty_rows(m: int, k: int, device) -> Fp8Rows:
    """Uninitialised rows to pass as ``out``."""
    v = torch.empty(m, -(-k // 16) * 16, dtype=_F8, device=device)
    return Fp8Rows(v[:, :k] if k % 16 else v, torch.empty(scale_shape(m, k), dtype=_E8, device=device))


# per device: the word in which a kernel records a bounded wait that gave up (never reallocated,
# so captured graphs may hold its address)
_ERROR_WORDS: Dict[int, torch.Tensor] = {}
_ERROR_WORDS_LOCK = threading.Lock()


def _error_word(index: int) -> int:
    """The address of a device's error word (made at the first call)."""
    with _ERROR_WORDS_LOCK:                        # synchronising lets other threads in: they wait here
        w = _ERROR_WORDS.get(index)
        if w is None:
            with torch.cuda.device(index):
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("the first fp8_linear on a device must run outside a CUDA graph capture")
                w = torch.zeros(64, dtype=torch.int32, device=torch.device("cuda", index))
                torch.cuda.synchronize(index)      # zero before any stream uses it
            _ERROR_WORDS[index] = w
    return w.data_ptr()


def check_device_errors(device=None) -> None:
    """Synchronise and raise if an ``fp8_linear`` on `device` gave up a bounded device-side wait."""
    for idx, w in list(_ERROR_WORDS.items()):
        if device is not None and torch.device(device).index not in (None, idx):
            continue
        with torch.cuda.device(idx):
            torch.cuda.synchronize(idx)
            _lib.check(_lib.lib().fbfp_gemv_check(_lib.ptr(w), _lib.stream_ptr(idx)), "fp8_linear")


_bind = None


def _module():
    """The checks and calls of csrc/fp8_bind.cpp (loaded on first use)."""
    global _bind
    if _bind is None:
        _lib.lib()                                 # raises if the library is not built
        if not os.path.exists(build.BIND):
            raise _lib.FlashBFPError(f"{build.BIND} is missing: build it with `python -m flashbfp_b200.build`")
        spec = importlib.util.spec_from_file_location("flashbfp_b200._fp8_bind", build.BIND)
        again = "build it again with `python -m flashbfp_b200.build`"
        try:
            m = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(m)
        except ImportError as e:                   # another torch's symbols
            raise _lib.FlashBFPError(f"{build.BIND} does not load ({e}): {again}") from e
        if m.built_for != build.bind_for():
            raise _lib.FlashBFPError(f"{build.BIND} is built for {m.built_for}, this is {build.bind_for()}: {again}")
        m.setup(Fp8Rows, _error_word)
        _bind = m
    return _bind


def quantize_fp8(x: torch.Tensor, out: Optional[Fp8Rows] = None) -> Fp8Rows:
    """Rows x [m, k] (bf16, fp16 or fp32, any row stride) as e4m3 values with their scales."""
    return (_bind or _module()).quantize(x, out)


def geglu_fp8(gate_up: torch.Tensor, out: Optional[Fp8Rows] = None) -> Fp8Rows:
    """gelu_tanh(gate) * up of rows [gate | up] as e4m3 values with their scales."""
    return (_bind or _module()).geglu(gate_up, out)


def rmsnorm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: Optional[torch.Tensor] = None,
                post_weight: Optional[torch.Tensor] = None, out: Optional[Fp8Rows] = None) -> Fp8Rows:
    """RMSNorm(h) = h * rsqrt(mean(h^2) + eps) * (1 + weight) as e4m3 values with their scales.

    h is x, with ``residual`` x + residual, with ``post_weight`` too RMSNorm(x; post_weight) +
    residual (the post-norm, residual addition and next pre-norm between a layer's halves). The
    residual is replaced by h rounded to its type; the norm reads the unrounded h. Rows of up to
    32768 values; x, weights and residual have one dtype."""
    return (_bind or _module()).rmsnorm(x, weight, eps, residual, post_weight, out)


def fp8_linear(x: Fp8Rows, w: Fp8Rows, bias: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y [m, n] = x w^T (+ bias) of rows x [m, k] and weight rows w [n, k]: fp32 accumulation of
    the scaled products, one rounding to ``out_dtype`` (bf16 by default, fp16 or fp32)."""
    return (_bind or _module()).linear(x, w, bias, out_dtype, out)
