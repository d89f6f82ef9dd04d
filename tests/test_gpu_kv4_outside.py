"""Rows whose position is outside the cache: 0 whatever their queries and the cache hold."""
import math

import pytest
import torch

from test_gpu_kv4_attention import filled, queries
from test_gpu_kv4_store import ints

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("positions", [96, 640, 12800])                 # a CTA's own, and joined from parts
@pytest.mark.parametrize("what", ["nan query", "inf query", "nan cache"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_outside_rows_are_zero(positions, what, dtype):
    from flashbfp_b200 import kv4
    cache = filled(3, 2, positions, 64, 3)
    q = queries((3, 4, 4, 64), dtype, 4)
    pos = [cache.positions, cache.positions - 2, -2]
    outside = [(0, range(4)), (1, (2, 3)), (2, (0, 1))]
    clean = kv4.kv4_attention(q, cache, ints(pos), err=ints([0]))
    for b, rows in outside:
        for i in rows:
            if what != "nan cache":
                q[b, i] = math.nan if what == "nan query" else math.inf
    if what == "nan cache":
        cache.k_scales[0] = math.nan
        cache.v_scales[0] = math.inf
    err = ints([0])
    out = kv4.kv4_attention(q, cache, ints(pos), err=err)
    assert err.item() == 2
    for b, rows in outside:
        for i in rows:
            assert not out[b, i].any() and torch.isfinite(out[b, i]).all(), (b, i)
    assert torch.equal(out[1, :2], clean[1, :2]) and torch.equal(out[2, 2:], clean[2, 2:])
