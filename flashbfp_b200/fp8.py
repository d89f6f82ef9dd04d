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
"""
from __future__ import annotations

from typing import Dict, NamedTuple, Optional

import torch

from . import _lib

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
        """The rows the operand stands for: values * scale (exact in fp32 and in bf16)."""
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


def _error_word(index: int) -> torch.Tensor:
    w = _ERROR_WORDS.get(index)
    if w is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the first fp8_linear on a device must run outside a CUDA graph capture")
        w = torch.zeros(64, dtype=torch.int32, device=torch.device("cuda", index))
        torch.cuda.synchronize(index)              # zero before any stream uses it
        _ERROR_WORDS[index] = w
    return w


def check_device_errors(device=None) -> None:
    """Synchronise and raise if an ``fp8_linear`` on `device` gave up a bounded device-side wait."""
    for idx, w in _ERROR_WORDS.items():
        if device is not None and torch.device(device).index not in (None, idx):
            continue
        with torch.cuda.device(idx):
            torch.cuda.synchronize(idx)
            _lib.check(_lib.lib().fbfp_gemv_check(_lib.ptr(w), _lib.stream_ptr(idx)), "fp8_linear")


def _plain_rows(t, what: str, cols: Optional[int] = None) -> torch.Tensor:
    _lib.require_cuda(t, what)
    if t.dim() != 2:
        raise ValueError(f"{what} must have two dimensions, not {t.dim()}")
    if cols is not None and t.shape[1] != cols:
        raise ValueError(f"{what} has {t.shape[1]} columns, not {cols}")
    if t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError(f"{what} must have contiguous rows (stride {t.stride(1)} between columns)")
    if t.dtype not in _lib.DTYPE_CODE:
        raise NotImplementedError(f"{what}: unsupported dtype {t.dtype}")
    return t


def _row_stride(t: torch.Tensor) -> int:
    # a single row's stride is never used (views of one row may carry any)
    return t.stride(0) if t.shape[0] > 1 else -(-t.shape[1] // 16) * 16


def _check_rows(r: Fp8Rows, what: str, m: Optional[int], k: Optional[int], device) -> None:
    v, s = r
    if not (v.is_cuda and s.is_cuda):
        raise RuntimeError(f"{what} must be on a CUDA device (no CPU fallback)")
    if v.device != device or s.device != device:
        raise ValueError(f"{what} is not on {device}")
    if v.dtype != _F8 or s.dtype != _E8 or v.dim() != 2:
        raise ValueError(f"{what}: values must be 2-D float8_e4m3fn and scales float8_e8m0fnu")
    vm, vk = v.shape
    if (m is not None and vm != m) or (k is not None and vk != k):
        raise ValueError(f"{what} has shape {tuple(v.shape)}, not ({m if m is not None else '*'}, "
                         f"{k if k is not None else '*'})")
    if vk > 1 and v.stride(1) != 1 or vm > 1 and (v.stride(0) % 16 or v.stride(0) < vk):
        raise ValueError(f"{what}: rows must be contiguous and a multiple of 16 bytes apart "
                         f"(strides {v.stride()})")
    if tuple(s.shape) != scale_shape(vm, vk) or not s.is_contiguous():
        raise ValueError(f"{what}: scales must be contiguous {scale_shape(vm, vk)}, not {tuple(s.shape)}")


def _result(out: Optional[Fp8Rows], m: int, k: int, device) -> Fp8Rows:
    if k < 1:
        raise ValueError("rows must have at least one value")
    if out is None:
        return empty_rows(m, k, device)
    _check_rows(out, "out", m, k, device)
    return out


def quantize_fp8(x: torch.Tensor, out: Optional[Fp8Rows] = None) -> Fp8Rows:
    """Rows x [m, k] (bf16, fp16 or fp32, any row stride) as e4m3 values with their scales."""
    _plain_rows(x, "x")
    m, k = x.shape
    dev = x.device
    r = _result(out, m, k, dev)
    if m:
        with torch.cuda.device(dev):
            _lib.check(_lib.lib().fbfp_fp8_quantize(
                x.data_ptr(), _lib.DTYPE_CODE[x.dtype], m, k, _row_stride(x), r.values.data_ptr(),
                _row_stride(r.values), r.scales.data_ptr(), torch.cuda.current_stream(dev).cuda_stream),
                "fbfp_fp8_quantize")
    return r


def geglu_fp8(gate_up: torch.Tensor, out: Optional[Fp8Rows] = None) -> Fp8Rows:
    """gelu_tanh(gate) * up of rows [gate | up] as e4m3 values with their scales."""
    _plain_rows(gate_up, "gate_up")
    m, k2 = gate_up.shape
    if k2 % 2:
        raise ValueError(f"gate_up must hold as many gate as up columns (got {k2})")
    k, dev = k2 // 2, gate_up.device
    r = _result(out, m, k, dev)
    if m:
        with torch.cuda.device(dev):
            _lib.check(_lib.lib().fbfp_fp8_geglu(
                gate_up.data_ptr(), _lib.DTYPE_CODE[gate_up.dtype], m, k, _row_stride(gate_up),
                r.values.data_ptr(), _row_stride(r.values), r.scales.data_ptr(),
                torch.cuda.current_stream(dev).cuda_stream), "fbfp_fp8_geglu")
    return r


def rmsnorm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: Optional[torch.Tensor] = None,
                post_weight: Optional[torch.Tensor] = None, out: Optional[Fp8Rows] = None) -> Fp8Rows:
    """RMSNorm(h) = h * rsqrt(mean(h^2) + eps) * (1 + weight) as e4m3 values with their scales.

    h is x, with ``residual`` x + residual, with ``post_weight`` too RMSNorm(x; post_weight) +
    residual (the post-norm, residual addition and next pre-norm between a layer's halves). The
    residual is replaced by h rounded to its type; the norm reads the unrounded h. Rows of up to
    32768 values; x, weights and residual have one dtype."""
    _plain_rows(x, "x")
    m, k = x.shape
    dev, dt = x.device, x.dtype
    for t, what in ((weight, "weight"), (post_weight, "post_weight")):
        if t is None:
            continue
        if t.dtype != dt or t.device != dev or t.shape != (k,) or not t.is_contiguous():
            raise ValueError(f"{what} must be a contiguous {dt} vector of {k} on {dev}")
    if residual is not None:
        _plain_rows(residual, "residual", k)
        if residual.dtype != dt or residual.device != dev or residual.shape[0] != m:
            raise ValueError(f"residual must be {dt} of shape ({m}, {k}) on {dev}")
        if m > 1 and residual.stride(0) < k:
            raise ValueError("residual rows overlap: each is updated in place")
    elif post_weight is not None:
        raise ValueError("post_weight needs the residual that its output is added to")
    r = _result(out, m, k, dev)
    if m:
        with torch.cuda.device(dev):
            _lib.check(_lib.lib().fbfp_fp8_rmsnorm(
                x.data_ptr(), _lib.DTYPE_CODE[dt], m, k, _row_stride(x), weight.data_ptr(),
                post_weight.data_ptr() if post_weight is not None else None,
                residual.data_ptr() if residual is not None else None,
                _row_stride(residual) if residual is not None else 0, eps, r.values.data_ptr(),
                _row_stride(r.values), r.scales.data_ptr(), torch.cuda.current_stream(dev).cuda_stream),
                "fbfp_fp8_rmsnorm")
    return r


def fp8_linear(x: Fp8Rows, w: Fp8Rows, bias: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y [m, n] = x w^T (+ bias) of rows x [m, k] and weight rows w [n, k]: fp32 accumulation of
    the scaled products, one rounding to ``out_dtype`` (bf16 by default, fp16 or fp32)."""
    dev = x[0].device
    _check_rows(x, "x", None, None, dev)
    m, k = x[0].shape
    _check_rows(w, "w", None, k, dev)
    n = w[0].shape[0]
    if k < 1:
        raise ValueError("rows must have at least one value")
    if bias is not None:
        if bias.shape != (n,) or bias.device != dev or not bias.is_contiguous():
            raise ValueError(f"bias must be a contiguous vector of {n} on {dev}")
        bd = _lib.dtype_code(bias.dtype, "bias")
    if out is None:
        out = torch.empty(m, n, dtype=out_dtype or torch.bfloat16, device=dev)
    else:
        _plain_rows(out, "out", n)
        if out.shape[0] != m or out.device != dev or (out_dtype is not None and out.dtype != out_dtype):
            raise ValueError(f"out must have shape ({m}, {n}) on {dev}" +
                             (f" and dtype {out_dtype}" if out_dtype is not None else ""))
        if m > 1 and out.stride(0) < n:
            raise ValueError("out's rows overlap")
    yd = _lib.dtype_code(out.dtype, "out")
    if m and n:
        with torch.cuda.device(dev):
            _lib.check(_lib.lib().fbfp_fp8_linear(
                x[0].data_ptr(), m, k, _row_stride(x[0]), x[1].data_ptr(), w[0].data_ptr(), n, _row_stride(w[0]),
                w[1].data_ptr(), bias.data_ptr() if bias is not None else None, bd if bias is not None else 0,
                out.data_ptr(), yd, _row_stride(out), _error_word(dev.index).data_ptr(),
                torch.cuda.current_stream(dev).cuda_stream), "fbfp_fp8_linear")
    return out
