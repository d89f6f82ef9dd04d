"""The attention and cache entry points refuse bad calls before they touch a GPU."""
import ctypes

import pytest
import torch

from flashbfp_b200 import _lib, attention, build, kv4


@pytest.fixture(scope="module")
def L():
    build.build()
    return _lib.lib()


P, ODD = ctypes.c_void_p(4096), ctypes.c_void_p(4098)        # addresses that no refused call reads


def refused(L, status, text, code=1):
    assert status == code, (status, L.fbfp_last_error())
    assert text in L.fbfp_last_error().decode(), L.fbfp_last_error()


def cache(values=P, seqs=2, heads=2, positions=64, dim=64):
    return ctypes.byref(_lib.KV4CacheStruct(values, P, P, P, seqs, heads, positions, dim))


def test_cache_refusals(L):
    def write(c, k=P, dt=1, rows=2, kr=128, pos=P, starts=None, err=P):
        return L.fbfp_kv4_write(c, k, P, dt, rows, kr, 64, 128, 64, pos, starts, err, None)

    refused(L, write(None), "null")
    refused(L, write(cache(values=None)), "null")
    refused(L, write(cache(seqs=0)), "sizes")
    refused(L, write(cache(dim=60)), "multiple of 8")
    refused(L, write(cache(dim=264)), "multiple of 8")
    refused(L, write(cache(positions=33)), "multiple of 32")
    refused(L, write(cache(positions=1 << 30)), "below 2^30")
    refused(L, write(cache(values=ODD)), "aligned", code=4)
    for fn in (write, lambda c, **a: L.fbfp_kv4_read(c, a.get("k", P), P, a.get("dt", 1), a.get("rows", 2), a.get("kr", 128),
                                                     64, 128, 64, a.get("pos", P), None, a.get("err", P), None)):
        refused(L, fn(cache(), k=None), "null")
        refused(L, fn(cache(), pos=None), "null")
        refused(L, fn(cache(), err=None), "null")
        refused(L, fn(cache(), dt=7), "dtype")
        refused(L, fn(cache(), rows=0), "row count")
        refused(L, fn(cache(), rows=3), "without starts")
        refused(L, fn(cache(), kr=-8), "stride")
        refused(L, fn(cache(), k=ODD, dt=0), "aligned to their type")

    def append(c=None, heads=4, rows=2, q=P, qkv=P):
        return L.fbfp_kv4_append(c or cache(), qkv, rows, heads, P, P, 1e-6, P, P, P, None, q, P, None)

    refused(L, append(qkv=None), "null")
    refused(L, append(cache(dim=72)), "multiple of 16")
    refused(L, append(heads=3), "heads")
    refused(L, append(rows=0), "row count")
    refused(L, append(rows=3), "without starts")
    refused(L, append(q=ODD), "aligned", code=4)


def test_cache_attention_refusals(L):
    def attend(c=None, q=P, dt=1, rows=1, heads=4, qs=256, pos=P, window=0, out=P, err=P):
        return L.fbfp_kv4_attention(c or cache(), q, dt, rows, heads, qs, 0, 64, pos, window, 0.125, out, 256, 0, 64, P,
                                    1 << 30, err, None)

    for name in ("q", "pos", "out", "err"):
        refused(L, attend(**{name: None}), "null")
    refused(L, attend(dt=0), "dtype")
    refused(L, attend(rows=0), "rows")
    refused(L, attend(heads=3), "heads")
    refused(L, attend(qs=252), "strides")
    refused(L, attend(window=-1), "window")
    refused(L, attend(q=ODD), "aligned", code=4)


def test_prompt_attention_refusals(L):
    def attend(q=P, dt=1, rows=8, kv_rows=8, seqs=1, heads=4, kv=2, dim=64, qr=256, starts=P, window=0, out=P, err=P):
        return L.fbfp_prompt_attention(q, P, P, dt, rows, kv_rows, seqs, heads, kv, dim, qr, 64, 128, 64, 128, 64, starts,
                                       None, window, 0.125, out, 256, 64, P, 1 << 30, err, None)

    for name in ("q", "starts", "out", "err"):
        refused(L, attend(**{name: None}), "null")
    refused(L, attend(dt=0), "dtype")
    for bad in (dict(rows=0), dict(kv_rows=0), dict(seqs=0), dict(rows=1 << 30)):
        refused(L, attend(**bad), "sizes")
    refused(L, attend(heads=3), "heads")
    refused(L, attend(dim=4), "multiple of 8")
    refused(L, attend(dim=512), "multiple of 8")
    refused(L, attend(qr=252), "strides")
    refused(L, attend(window=-3), "window")
    refused(L, attend(out=ODD), "aligned", code=4)


def test_cpu_tensors_are_refused():
    x, i = torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int32)
    c = kv4.empty_cache(2, 2, 40, 64, "cpu")
    assert c.positions == 64 and c.k_values.shape == (2, 2, 64, 32) and c.v_scales.shape == (2, 2, 64, 2)
    for call in (lambda: attention.prompt_attention(x, x, x, i), lambda: kv4.kv4_write(c, x, x, i),
                 lambda: kv4.kv4_read(c, i, i, rows=2), lambda: kv4.kv4_attention(x, c, i)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_empty_cache_refusals():
    for bad in (dict(head_dim=60), dict(head_dim=0), dict(head_dim=264), dict(positions=0), dict(sequences=0)):
        a = dict(sequences=1, kv_heads=1, positions=32, head_dim=64, device="cpu")
        with pytest.raises(ValueError):
            kv4.empty_cache(**{**a, **bad})
    c = kv4.empty_cache(3, 1, 32, 40, "cpu")
    assert c.sequence(1).k_values.data_ptr() == c.k_values[1].data_ptr() and c.k_scales.shape[3] == 2


def test_the_longest_window_is_none(L):
    """A window of 2^63 - 1 plans as one that no sequence fills (the workspace follows the plan)."""
    for n in ((16, 20000, 1, 16, 8, 256), (1, 9000, 1, 2, 1, 64), (4096, 4096, 3, 16, 8, 128)):
        none, *others = [L.fbfp_prompt_attention_workspace_bytes(*n, w) for w in (0, (1 << 63) - 1, (1 << 63) - 200, 1 << 40)]
        assert others == [none] * 3, (n, none, others)
    assert L.fbfp_prompt_attention_workspace_bytes(16, 20000, 1, 16, 8, 256, 0) > 0


@pytest.mark.parametrize("scaling", [float("inf"), float("-inf"), float("nan"), 3e38, -3e38])
def test_scalings_that_are_not_finite(L, scaling):
    refused(L, L.fbfp_kv4_attention(cache(), P, 1, 1, 4, 256, 0, 64, P, 0, scaling, P, 256, 0, 64, P, 1 << 30, P, None), "scaling")
    refused(L, L.fbfp_prompt_attention(P, P, P, 1, 8, 8, 1, 4, 2, 64, 256, 64, 128, 64, 128, 64, P, None, 0, scaling, P, 256,
                                       64, P, 1 << 30, P, None), "scaling")
