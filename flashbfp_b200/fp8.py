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


# The checks and the call itself are most of a small call's time (a launch is about 4 us), so they
# stay on cheap tensor queries: device indices instead of device objects, one shape and one stride
# query per tensor, and the device switched only where it is not the current one.
def _call(fn, what: str, index: int, *args) -> None:
    """fn(*args, stream) on device `index` and its current stream."""
    if torch.cuda.current_device() == index:
        status = fn(*args, _lib.raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _lib.raw_stream(index))
    if status:
        _lib.check(status, what)


def _plain_rows(t, what: str):
    """(device index, dtype code, rows, columns, row stride) of a 2-D tensor of plain values."""
    index = t.get_device() if isinstance(t, torch.Tensor) else -1
    if index < 0:
        _lib.require_cuda(t, what)
    shape = t.shape
    if len(shape) != 2:
        raise ValueError(f"{what} must have two dimensions, not {len(shape)}")
    m, k = shape
    ld, step = t.stride()
    if step != 1 and k > 1:
        raise ValueError(f"{what} must have contiguous rows (stride {step} between columns)")
    code = _lib.DTYPE_CODE.get(t.dtype)
    if code is None:
        raise NotImplementedError(f"{what}: unsupported dtype {t.dtype}")
    # a single row's stride is never used (views of one row may carry any)
    return index, code, m, k, ld if m > 1 else (k + 15) // 16 * 16


def _check_rows(r: Fp8Rows, what: str, index: int, m: int = -1, k: int = -1):
    """(rows, columns, row stride) of an operand on device `index`, of shape (m, k) where given."""
    v, s = r
    if index < 0 or v.get_device() != index or s.get_device() != index:
        if not (v.is_cuda and s.is_cuda):
            raise RuntimeError(f"{what} must be on a CUDA device (no CPU fallback)")
        raise ValueError(f"{what} is not on cuda:{index}")
    if v.dtype != _F8 or s.dtype != _E8 or v.dim() != 2:
        raise ValueError(f"{what}: values must be 2-D float8_e4m3fn and scales float8_e8m0fnu")
    vm, vk = v.shape
    if (m >= 0 and vm != m) or (k >= 0 and vk != k):
        raise ValueError(f"{what} has shape {(vm, vk)}, not ({m if m >= 0 else '*'}, {k if k >= 0 else '*'})")
    if vk < 1:
        raise ValueError("rows must have at least one value")
    ld, step = v.stride()
    if vm <= 1:
        ld = (vk + 15) // 16 * 16
    if (step != 1 and vk > 1) or ld % 16 or ld < vk:
        raise ValueError(f"{what}: rows must be contiguous and a multiple of 16 bytes apart (strides {v.stride()})")
    if s.shape != ((vm + 127) // 128, (vk + 511) // 512, 32, 4, 4) or not s.is_contiguous():
        raise ValueError(f"{what}: scales must be contiguous {scale_shape(vm, vk)}, not {tuple(s.shape)}")
    return vm, vk, ld


def _result(out: Optional[Fp8Rows], m: int, k: int, index: int):
    """The rows to write and their row stride."""
    if out is None:
        if k < 1:
            raise ValueError("rows must have at least one value")
        out = empty_rows(m, k, torch.device("cuda", index))
        return out, (k + 15) // 16 * 16
    return out, _check_rows(out, "out", index, m, k)[2]


def quantize_fp8(x: torch.Tensor, out: Optional[Fp8Rows] = None) -> Fp8Rows:
    """Rows x [m, k] (bf16, fp16 or fp32, any row stride) as e4m3 values with their scales."""
    index, code, m, k, ldx = _plain_rows(x, "x")
    r, ldv = _result(out, m, k, index)
    if m:
        _call(_lib.lib().fbfp_fp8_quantize, "fbfp_fp8_quantize", index, x.data_ptr(), code, m, k, ldx,
              r[0].data_ptr(), ldv, r[1].data_ptr())
    return r


def geglu_fp8(gate_up: torch.Tensor, out: Optional[Fp8Rows] = None) -> Fp8Rows:
    """gelu_tanh(gate) * up of rows [gate | up] as e4m3 values with their scales."""
    index, code, m, k2, ldx = _plain_rows(gate_up, "gate_up")
    if k2 % 2:
        raise ValueError(f"gate_up must hold as many gate as up columns (got {k2})")
    r, ldv = _result(out, m, k2 // 2, index)
    if m:
        _call(_lib.lib().fbfp_fp8_geglu, "fbfp_fp8_geglu", index, gate_up.data_ptr(), code, m, k2 // 2, ldx,
              r[0].data_ptr(), ldv, r[1].data_ptr())
    return r


def _norm_weight(w: torch.Tensor, what: str, x: torch.Tensor, index: int, k: int) -> int:
    if w.dtype != x.dtype or w.get_device() != index or w.shape != (k,) or not w.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {x.dtype} vector of {k} on {x.device}")
    return w.data_ptr()


def rmsnorm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: Optional[torch.Tensor] = None,
                post_weight: Optional[torch.Tensor] = None, out: Optional[Fp8Rows] = None) -> Fp8Rows:
    """RMSNorm(h) = h * rsqrt(mean(h^2) + eps) * (1 + weight) as e4m3 values with their scales.

    h is x, with ``residual`` x + residual, with ``post_weight`` too RMSNorm(x; post_weight) +
    residual (the post-norm, residual addition and next pre-norm between a layer's halves). The
    residual is replaced by h rounded to its type; the norm reads the unrounded h. Rows of up to
    32768 values; x, weights and residual have one dtype."""
    index, code, m, k, ldx = _plain_rows(x, "x")
    wp = _norm_weight(weight, "weight", x, index, k)
    pp, rp, ldr = None, None, 0
    if residual is not None:
        ri, rcode, rm, rk, ldr = _plain_rows(residual, "residual")
        if rcode != code or ri != index or rm != m or rk != k:
            raise ValueError(f"residual must be {x.dtype} of shape ({m}, {k}) on {x.device}")
        if ldr < k:
            raise ValueError("residual rows overlap: each is updated in place")
        rp = residual.data_ptr()
        if post_weight is not None:
            pp = _norm_weight(post_weight, "post_weight", x, index, k)
    elif post_weight is not None:
        raise ValueError("post_weight needs the residual that its output is added to")
    r, ldv = _result(out, m, k, index)
    if m:
        _call(_lib.lib().fbfp_fp8_rmsnorm, "fbfp_fp8_rmsnorm", index, x.data_ptr(), code, m, k, ldx, wp, pp, rp, ldr,
              eps, r[0].data_ptr(), ldv, r[1].data_ptr())
    return r


def fp8_linear(x: Fp8Rows, w: Fp8Rows, bias: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y [m, n] = x w^T (+ bias) of rows x [m, k] and weight rows w [n, k]: fp32 accumulation of
    the scaled products, one rounding to ``out_dtype`` (bf16 by default, fp16 or fp32)."""
    index = x[0].get_device()
    m, k, ldx = _check_rows(x, "x", index)
    n, _, ldw = _check_rows(w, "w", index, -1, k)
    bp, bd = None, 0
    if bias is not None:
        if bias.shape != (n,) or bias.get_device() != index or not bias.is_contiguous():
            raise ValueError(f"bias must be a contiguous vector of {n} on cuda:{index}")
        bp, bd = bias.data_ptr(), _lib.dtype_code(bias.dtype, "bias")
    if out is None:
        out = torch.empty(m, n, dtype=out_dtype or torch.bfloat16, device=x[0].device)
    oi, yd, om, on, ldy = _plain_rows(out, "out")
    if om != m or on != n or oi != index or (out_dtype is not None and out.dtype != out_dtype):
        raise ValueError(f"out must have shape ({m}, {n}) on cuda:{index}" +
                         (f" and dtype {out_dtype}" if out_dtype is not None else ""))
    if ldy < n:
        raise ValueError("out's rows overlap")
    if m and n:
        _call(_lib.lib().fbfp_fp8_linear, "fbfp_fp8_linear", index, x[0].data_ptr(), m, k, ldx, x[1].data_ptr(),
              w[0].data_ptr(), n, ldw, w[1].data_ptr(), bp, bd, out.data_ptr(), yd, ldy,
              _error_word(index).data_ptr())
    return out
