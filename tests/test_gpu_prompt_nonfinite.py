"""Infinities and NaN in keys and values of prompts' attention, for every way that values are looked over: what does
not see them is as without them (within attention_reference's bounds), what does is not finite."""
import math

import pytest
import torch

from attention_reference import packed, starts_of
from test_gpu_kv4_store import ints

pytestmark = pytest.mark.gpu
DEV = "cuda"
WAYS = [(64, torch.bfloat16), (64, torch.float16), (128, torch.bfloat16), (128, torch.float16), (136, torch.float16),
        (200, torch.bfloat16), (256, torch.bfloat16), (256, torch.float16)]


def normal(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def check(q, k, v, bad_k, bad_v, lens, kv_lens, window, sees):
    """bad_k, bad_v: keys and values with what is not finite in them, elsewhere as k and v; sees [T, H, D]: the results
    that it reaches."""
    from flashbfp_b200 import attention
    starts, kv_starts = starts_of(lens), starts_of(kv_lens)
    want, bound = packed(q, k, v, starts, kv_starts, window, q.shape[-1] ** -0.5, torch.finfo(q.dtype).eps / 2)
    first = None
    for _ in range(3):
        got = attention.prompt_attention(q, bad_k, bad_v, ints(starts), kv_starts=ints(kv_starts), window=window)
        attention.check_device_errors()
        g = got.double().cpu()
        assert not torch.isfinite(g[sees]).any()
        off = (g - want).abs()[~sees]
        assert (off <= bound[~sees]).all(), (off / bound[~sees]).max().item()
        assert first is None or torch.equal(got.view(torch.int16)[~sees], first.view(torch.int16)[~sees])
        first = got


@pytest.mark.parametrize("dim,dtype", WAYS)
def test_neighbours(dim, dtype):
    """A whole sequence of them between two others, whose last blocks reach into it and past the last key."""
    lens = [100, 70, 130]
    q, k, v = (normal((300, h, dim), dtype, i) for i, h in enumerate((4, 2, 2)))
    bk, bv = k.clone(), v.clone()
    bk[100:170], bv[100:170] = math.nan, math.inf
    sees = torch.zeros(300, 4, dim, dtype=torch.bool)
    sees[100:170] = True
    check(q, k, v, bk, bv, lens, lens, 0, sees)
    check(q, k, v, bk, bv, lens, lens, 40, sees)


@pytest.mark.parametrize("dim,dtype", WAYS)
def test_values_behind_a_window_and_after_a_row(dim, dtype):
    n, window = 700, 50
    q, k, v = (normal((n, h, dim), dtype, 3 + i) for i, h in enumerate((4, 2, 2)))
    bk, bv = k.clone(), v.clone()
    bk[:200], bv[:200] = math.inf, math.nan
    sees = torch.zeros(n, 4, dim, dtype=torch.bool)
    sees[:249] = True                                  # row 249's window begins at 200
    check(q, k, v, bk, bv, [n], [n], window, sees)
    bv = v.clone()
    bv[620:, :, 3] = math.nan                          # one value of each head, late in the sequence
    bv[333, 1, dim - 1] = -math.inf
    sees = torch.zeros(n, 4, dim, dtype=torch.bool)
    sees[620:, :, 3] = True
    sees[333:, 2:, dim - 1] = True
    check(q, k, v, k, bv, [n], [n], 0, sees)
    sees[333 + 320:, 2:, dim - 1] = False
    check(q, k, v, k, bv, [n], [n], 320, sees)


@pytest.mark.parametrize("dim,dtype", WAYS)
def test_split_keys(dim, dtype):
    """Few rows over a long axis, cut into parts: before a window, inside what all rows see, and after some rows."""
    rows, keys = 40, 6000
    q = normal((rows, 4, dim), dtype, 7)
    k, v = normal((keys, 2, dim), dtype, 8), normal((keys, 2, dim), dtype, 9)
    bv = v.clone()
    bv[:3000] = math.nan
    none = torch.zeros(rows, 4, dim, dtype=torch.bool)
    check(q, k, v, k, bv, [rows], [keys], 2900, none)
    bv = v.clone()
    bv[keys - 10, 0, 1] = math.inf
    sees = none.clone()
    sees[rows - 10:, :2, 1] = True
    check(q, k, v, k, bv, [rows], [keys], 0, sees)
    bv[100, 1, 2] = math.nan
    sees[:, 2:, 2] = True
    check(q, k, v, k, bv, [rows], [keys], 0, sees)


@pytest.mark.parametrize("dim,dtype", [(64, torch.bfloat16), (128, torch.float16)])
def test_two_tiles_over_one_end(dim, dtype):
    """Two tiles of a CTA whose last steps reach past the same end, where a neighbour's values are not finite: each puts
    zeros there, or sees the other's."""
    lens = [130, 255, 129, 200]
    t = sum(lens)
    q, k, v = (normal((t, h, dim), dtype, 11 + i) for i, h in enumerate((2, 2, 2)))
    for b in range(len(lens)):
        s = starts_of(lens)
        bv = torch.full_like(v, math.nan)
        bv[s[b]:s[b + 1]] = v[s[b]:s[b + 1]]
        sees = torch.ones(t, 2, dim, dtype=torch.bool)
        sees[s[b]:s[b + 1]] = False
        check(q, k, v, k, bv, lens, lens, 0, sees)
