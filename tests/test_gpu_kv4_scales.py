"""Attention over the 4-bit cache where the values' scales lie far apart: between groups of a head, between positions,
and where a position of small weight brings the largest values.

The bound, for a value d of group g: u |o| of the result's rounding, (2^-11 + 2 e_s + 2^-19) sum_j p_j |v_jd| of the weights'
(e_s the scores' error, as attention_reference derives it), and for terms p_j s_jg n_jd that are small beside the
largest p_j s_jg, which fp16 may hold as subnormals or not at all: 2^-19 of that, times 7, each."""
import math

import pytest
import torch

from test_gpu_kv4_store import ints

pytestmark = pytest.mark.gpu
DEV = "cuda"


def check(cache, q, pos, window=0):
    from flashbfp_b200 import kv4
    got = kv4.kv4_attention(q, cache, ints(pos), window=window).double().cpu()
    kv4.check_device_errors()
    d, grp = q.shape[-1], q.shape[2] // cache.k_values.shape[1]

    def held(values, scales, b, lo, n):
        x = torch.stack((values[b, :, lo:n] & 15, values[b, :, lo:n] >> 4), -1).flatten(-2).double().cpu() - 8
        s = scales[b, :, lo:n].double().cpu().repeat_interleave(32, -1)
        return (x * s)[..., :d].repeat_interleave(grp, 0), s[..., :d].repeat_interleave(grp, 0)

    worst = 0.0
    for b in range(q.shape[0]):
        for i in range(q.shape[1]):
            n = pos[b] + i + 1
            lo = max(0, n - window) if window else 0
            k, _ = held(cache.k_values, cache.k_scales, b, lo, n)
            v, s = held(cache.v_values, cache.v_scales, b, lo, n)
            x = q[b, i].double().cpu()
            score = torch.einsum("hd,hjd->hj", x, k) * d ** -0.5
            e_s = float((torch.einsum("hd,hjd->hj", x.abs(), k.abs()) * d ** -0.5).max()) * (d + 4) * 2.0 ** -24
            p = torch.softmax(score, -1)
            o = torch.einsum("hj,hjd->hd", p, v)
            u = torch.finfo(q.dtype).eps / 2
            bound = u * o.abs() + (1 + u) * (2.0 ** -11 + 2 * e_s + 2.0 ** -19) * torch.einsum("hj,hjd->hd", p, v.abs()) \
                + 7 * 2.0 ** -19 * (n - lo) * (p[..., None] * s).amax(1) + 1e-42
            if q.dtype == torch.float16:
                bound += 2.0 ** -25
            assert torch.isfinite(got[b, i]).all()
            off = (got[b, i] - o).abs() / bound
            worst = max(worst, off.max().item())
            assert off.max().item() <= 1, (b, i, off.max().item())
    return worst


def cache_of(k, v):
    """Rows [sequences, positions, heads, D] of fp32 in a cache."""
    from flashbfp_b200 import kv4
    s, n, h, d = k.shape
    cache = kv4.empty_cache(s, h, n, d, DEV)
    kv4.kv4_write(cache, k.flatten(0, 1).to(DEV), v.flatten(0, 1).to(DEV), ints([0] * s), starts=ints([n * b for b in range(s + 1)]))
    return cache


def normal(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("apart", [8, 14, 15, 20, 29, 33, 40, 60, 100])
@pytest.mark.parametrize("rows,heads,dim", [(1, 2, 64), (1, 4, 256), (4, 8, 128), (2, 16, 64), (3, 2, 96)])
def test_groups_apart(rows, heads, dim, apart):
    """Each group of a head 2^-apart as large as another, largest last or first."""
    n = 200
    k, v = normal(2, n, 2, dim, seed=1), normal(2, n, 2, dim, seed=2)
    f = torch.ones(dim)
    f[dim // 2:] = 2.0 ** -apart
    v[0] *= f
    v[1] *= f.flip(0)
    q = normal(2, rows, heads, dim, seed=3).bfloat16().to(DEV)
    check(cache_of(k, v), q, [n - rows, 150])
    check(cache_of(k, v), q, [n - rows, 150], window=70)


@pytest.mark.parametrize("dtype,apart", [(torch.float16, 10), *[(torch.bfloat16, a) for a in (10, 20, 33, 45, 70)]])
@pytest.mark.parametrize("rows,heads,dim", [(1, 2, 64), (1, 2, 256), (4, 8, 128)])
def test_positions_apart(rows, heads, dim, dtype, apart):
    """One position attended to in earnest among others whose values are far larger, their weights such that they
    vanish beside it, weigh as much, or outweigh it; early and late in the sequence."""
    n = 700
    q = torch.ones(1, rows, heads, dim).to(dtype).to(DEV)
    for at in (3, 400, n - rows - 1):
        for less in (apart + 30, apart, apart - 8, apart - 25):
            k = torch.zeros(1, n, 2, dim)
            k[:] = -less * math.log(2) / dim ** 0.5                # scores: -less ln 2, 0 at `at`
            k[0, at] = 0.0
            v = normal(1, n, 2, dim, seed=5)
            v[0, at] = normal(2, dim, seed=6) * 2.0 ** -apart
            check(cache_of(k, v), q, [n - rows])


@pytest.mark.parametrize("rows,heads", [(1, 2), (4, 8)])
def test_all_scales(rows, heads):
    """Scales anywhere in bf16's middle range, each position and group its own; the same bits every time."""
    from flashbfp_b200 import kv4
    n, dim = 500, 128
    k = normal(2, n, 2, dim, seed=7)
    v = normal(2, n, 2, dim, seed=8) * torch.exp2(60 * torch.rand(2, n, 2, dim // 32, generator=torch.Generator().manual_seed(9)) - 30).repeat_interleave(32, -1)
    cache = cache_of(k, v)
    q = normal(2, rows, heads, dim, seed=10).bfloat16().to(DEV)
    check(cache, q, [n - rows, 333])
    first = kv4.kv4_attention(q, cache, ints([n - rows, 333]))
    for _ in range(3):
        assert torch.equal(kv4.kv4_attention(q, cache, ints([n - rows, 333])), first)
