"""The block-scaled 8-bit entry points refuse bad calls before they touch a GPU, and the scale
tiles' layout agrees with the C ABI's size."""
import ctypes

import pytest
import torch

from flashbfp_b200 import _lib, build, fp8


@pytest.fixture(scope="module")
def L():
    build.build()
    return _lib.lib()


P = ctypes.c_void_p(4096)               # an aligned address that no refused call reads


@pytest.mark.parametrize("m,k", [(1, 1), (128, 512), (129, 513), (7, 3840)])
def test_scale_bytes(L, m, k):
    shape = fp8.scale_shape(m, k)
    n = 1
    for s in shape:
        n *= s
    assert L.fbfp_fp8_scale_bytes(m, k) == n
    assert L.fbfp_fp8_scale_bytes(0, k) == -1


def refused(L, status, text):
    assert status == 1
    assert text in L.fbfp_last_error().decode()


def test_row_entries_refuse(L):
    odd = ctypes.c_void_p(4100)
    for fn in (L.fbfp_fp8_quantize, L.fbfp_fp8_geglu):
        refused(L, fn(None, 1, 1, 16, 16, P, 16, P, None), "null")
        refused(L, fn(P, 1, 1, 16, 16, None, 16, P, None), "null")
        refused(L, fn(P, 7, 1, 16, 16, P, 16, P, None), "dtype")
        refused(L, fn(P, 1, 0, 16, 16, P, 16, P, None), "sizes")
        refused(L, fn(P, 1, 1, 0, 16, P, 16, P, None), "sizes")
        refused(L, fn(P, 1, 1, 17, 40, P, 16, P, None), "ldv")
        refused(L, fn(P, 1, 1, 17, 40, P, 24, P, None), "ldv")
        refused(L, fn(P, 1, 1, 16, 32, odd, 16, P, None), "aligned")
        refused(L, fn(P, 1, 1, 16, 32, P, 16, odd, None), "aligned")
        refused(L, fn(P, 1, 4, 16, -1, P, 16, P, None), "stride")
        refused(L, fn(ctypes.c_void_p(4097), 1, 1, 16, 32, P, 16, P, None), "aligned to their type")
        refused(L, fn(ctypes.c_void_p(4098), 0, 1, 16, 32, P, 16, P, None), "aligned to their type")

    def norm(x=P, dt=1, m=2, k=16, ldx=16, w=P, wp=None, r=None, ldr=0, v=P, ldv=16, s=P):
        return L.fbfp_fp8_rmsnorm(x, dt, m, k, ldx, w, wp, r, ldr, 1e-6, v, ldv, s, None)

    refused(L, norm(x=None), "null")
    refused(L, norm(w=None), "null")
    refused(L, norm(wp=P), "post-norm")
    refused(L, norm(r=P, ldr=8), "stride")
    refused(L, norm(k=32769, ldx=40000, ldv=32784), "at most 32768")
    refused(L, norm(dt=3), "dtype")
    refused(L, norm(w=ctypes.c_void_p(4097)), "aligned to their type")
    refused(L, norm(r=ctypes.c_void_p(4097), ldr=16), "aligned to their type")


def test_linear_refuses(L):
    def lin(x=P, m=2, k=16, ldx=16, xs=P, w=P, n=8, ldw=16, ws=P, b=None, bd=1, y=P, yd=1, ldy=8, err=P):
        return L.fbfp_fp8_linear(x, m, k, ldx, xs, w, n, ldw, ws, b, bd, y, yd, ldy, err, None)

    for name in ("x", "xs", "w", "ws", "y", "err"):
        refused(L, lin(**{name: None}), "null")
    refused(L, lin(m=0), "sizes")
    refused(L, lin(n=0), "sizes")
    refused(L, lin(k=0), "sizes")
    refused(L, lin(m=1 << 31), "sizes")
    refused(L, lin(ldx=24), "operands")
    refused(L, lin(ldw=8), "operands")
    refused(L, lin(x=ctypes.c_void_p(4104)), "operands")
    refused(L, lin(ws=ctypes.c_void_p(4104)), "scales")
    refused(L, lin(ldy=7), "ldy")
    refused(L, lin(yd=5), "dtype")
    refused(L, lin(b=P, bd=9), "dtype")
    refused(L, lin(y=ctypes.c_void_p(4097)), "aligned to their types")
    refused(L, lin(b=ctypes.c_void_p(4098), bd=0), "aligned to their types")


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        fp8.quantize_fp8(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        fp8.geglu_fp8(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        fp8.rmsnorm_fp8(x, torch.zeros(64), 1e-6)
    r = fp8.empty_rows(4, 64, "cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        fp8.fp8_linear(r, r)


def test_rows_on_the_cpu():
    """The container's own views need no GPU: layout of the tiles and the values they stand for."""
    m, k = 130, 700
    r = fp8.empty_rows(m, k, "cpu")
    assert r.values.stride(0) == 704 and r.shape == (m, k)
    codes = (torch.arange(m)[:, None] + torch.arange(6)[None, :]) % 200
    flat = r.scales.view(torch.uint8).view(-1)
    for row in (0, 31, 32, 127, 128, 129):
        for b in range(6):
            flat[((row // 128) * 2 + b // 4) * 512 + (row % 32) * 16 + (row % 128) // 32 * 4 + b % 4] = codes[row, b]
    s = r.scale_matrix()
    for row in (0, 31, 32, 127, 128, 129):
        assert torch.equal(s[row].double(), torch.exp2(codes[row].double() - 127))


def test_decoder_weight_kinds():
    from flashbfp_b200.decode import GemmaDecoder
    with pytest.raises(ValueError, match="'oabf' or 'fp8'"):
        GemmaDecoder.from_hf(None, max_ctx=8, weights="int4")
    with pytest.raises(ValueError, match="one GPU"):
        GemmaDecoder.from_hf(None, max_ctx=8, weights="fp8", reducer=object())
