"""Rows whose position is outside the cache: 0 whatever their queries and the cache hold, and an error word that does
not hide a wait that gave up."""
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


def test_a_position_outside_does_not_hide_a_wait_that_gave_up():
    """The word holds the site of a wait from another call; positions outside come after it."""
    from flashbfp_b200 import kv4
    d = 32
    cache = filled(2, 1, 64, d, 5)
    k = queries((2, 1, d), torch.bfloat16, 6)
    bf = dict(dtype=torch.bfloat16, device=DEV)
    ang, w = torch.ones(64, d, **bf), torch.zeros(d, **bf)
    calls = {
        "write": lambda e: kv4.kv4_write(cache, k, k, ints([-1, 64]), err=e),
        "read": lambda e: kv4.kv4_read(cache, ints([-1, 64]), ints([0, 1, 2]), rows=2, err=e),
        "append": lambda e: kv4.kv4_append(cache, torch.ones(2, 3 * d, **bf), w, w, 1e-6, ang, ang, ints([-1, 64]),
                                           torch.empty(2, 1, d, **bf), err=e),
        "attention": lambda e: kv4.kv4_attention(k, cache, ints([-1, 64]), err=e)}
    long = filled(2, 1, 6400, d, 7)
    calls["joined"] = lambda e: kv4.kv4_attention(k, long, ints([6400, 6399]), err=e)
    for name, call in calls.items():
        for before, after in ((0, 2), (48, 48), (33, 33)):
            err = ints([before])
            call(err)
            assert err.item() == after, (name, before, err.item())


def test_the_decoders_word_keeps_a_wait_that_gave_up():
    """GemmaDecoder: tokens outside the vocabulary and positions outside its cache after a recorded wait."""
    from test_gpu_decode_int4 import _decoder
    model, dec = _decoder(5, max_ctx=64, max_prefill=8)
    for outside in (lambda: dec.tok.fill_(10 ** 6), lambda: dec.pos.fill_(dec.cache4[0].positions)):
        for before in (0, 36):
            dec.reset(0)
            with torch.cuda.stream(dec.stream):
                dec.tok.fill_(1)
                dec.err.fill_(before)
                outside()
            dec.step()
            with pytest.raises(RuntimeError, match=f"error {before}" if before else "outside"):
                dec.check()
    dec.reset(0)
    with torch.cuda.stream(dec.stream):
        dec.err.fill_(36)
        dec.pos.fill_(50)                              # behind the decoder's back
    dec.prefill([1, 2, 3])
    with pytest.raises(RuntimeError, match="error 36"):
        dec.check()
    dec.release()
