"""Attention over the 4-bit cache against its definition in 64 bits, with the bounds that
attention_reference derives: cached whole numbers are exact in the products; the weight that meets them
(softmax weight times the value's scale) is rounded to fp16, u = 2^-11."""
import pytest
import torch

from attention_reference import cached
from test_gpu_kv4_store import garbage, ints, rows

pytestmark = pytest.mark.gpu
DEV = "cuda"
WEIGHT_U = {torch.bfloat16: 2.0 ** -11, torch.float16: 2.0 ** -11}


def filled(seqs, heads, positions, dim, seed):
    """A cache that holds rows everywhere."""
    from flashbfp_b200 import kv4
    cache = kv4.empty_cache(seqs, heads, positions, dim, DEV)
    n = cache.positions
    k, v = (rows((seqs * n, heads, dim), torch.bfloat16, seed + i).to(DEV).clamp(-30, 30) for i in range(2))
    kv4.kv4_write(cache, k, v, ints([0] * seqs), starts=ints([n * b for b in range(seqs + 1)]))
    return cache


def check(q, cache, pos, window=0, scaling=None, out=None):
    from flashbfp_b200 import kv4
    got = kv4.kv4_attention(q, cache, ints(pos), window=window, scaling=scaling, out=out)
    q4 = q if q.dim() == 4 else q[:, None]
    s = q.shape[-1] ** -0.5 if scaling is None else scaling
    want, bound = cached(q4, cache, pos, window, s, WEIGHT_U[q.dtype])
    g = got.double().cpu().view(want.shape)
    assert torch.isfinite(g).all()
    excess = ((g - want).abs() - bound).max().item()
    assert excess <= 0, (excess, ((g - want).abs() / bound).max().item())
    return got


def queries(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 1, 64), (16, 8, 256), (8, 1, 128), (3, 3, 40), (12, 1, 96),
                                                (40, 2, 256), (7, 1, 8), (6, 2, 192)])
def test_one_token(dtype, heads, kv_heads, dim):
    from flashbfp_b200 import kv4
    pos = [0, 1, 31, 32, 33, 63, 64, 200, 255, 500]
    cache = filled(len(pos), kv_heads, 512, dim, 1)
    q = queries((len(pos), heads, dim), dtype, 3)
    check(q, cache, pos)
    for window in (1, 2, 32, 100):
        check(q, cache, pos, window=window)
    kv4.check_device_errors()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows_,heads,kv_heads,dim", [(4, 64, 8, 128), (3, 6, 2, 80), (7, 4, 2, 256), (2, 16, 1, 64),
                                                      (33, 5, 1, 32)])
def test_several_rows(dtype, rows_, heads, kv_heads, dim):
    pos = [0, 30, 127, 290]
    cache = filled(len(pos), kv_heads, 352, dim, 5)
    q = queries((len(pos), rows_, heads, dim), dtype, 6)
    check(q, cache, pos)
    check(q, cache, pos, window=3)
    check(q, cache, pos, window=rows_ + 60)


@pytest.mark.parametrize("seqs,n", [(1, 20000), (2, 4999), (5, 3000)])
def test_long(seqs, n):
    """The work of a sequence split over CTAs and joined."""
    cache = filled(seqs, 2, n, 128, 7)
    pos = [max(0, n - 1 - 700 * b) for b in range(seqs)]
    q = queries((seqs, 4, 128), torch.bfloat16, 8)
    check(q, cache, pos)
    check(q, cache, pos, window=1024)
    check(queries((seqs, 2, 4, 128), torch.float16, 9), cache, [p - 1 for p in pos])


def test_mixed_lengths_and_repeats():
    """One long sequence among short ones; the same bits every time."""
    pos = [12000, 0, 5, 3, 700, 1, 0, 64]
    cache = filled(len(pos), 4, 12032, 64, 9)
    q = queries((len(pos), 8, 64), torch.bfloat16, 10)
    first = check(q, cache, pos)
    from flashbfp_b200 import kv4
    for _ in range(5):
        assert torch.equal(kv4.kv4_attention(q, cache, ints(pos)), first)


def test_unseen_positions_may_hold_anything():
    """NaN scales and random bytes before the window and after the newest position."""
    from flashbfp_b200 import kv4
    cache = filled(2, 2, 256, 96, 11)
    keep = [t.clone() for t in cache[:4]]
    garbage(cache, 12)
    cache.k_scales.fill_(float("nan"))
    cache.v_scales.fill_(float("inf"))
    pos, window = [100, 237], 70
    for t, k in zip(cache[:4], keep):
        for b, p in enumerate(pos):
            t[b, :, p + 1 - window:p + 1] = k[b, :, p + 1 - window:p + 1]
    q = queries((2, 4, 96), torch.bfloat16, 13)
    check(q, cache, pos, window=window)
    kv4.check_device_errors()


def test_sharp_and_flat_softmax():
    """Scores far apart (one key takes all, the maximum last or first) and all equal."""
    from flashbfp_b200 import kv4
    cache = filled(1, 1, 640, 64, 15)
    q = queries((1, 2, 64), torch.bfloat16, 16)
    for scaling in (0.0, 1e-4, 3.0, 40.0, -3.0):
        check(q, cache, [600], scaling=scaling)
    # scores that grow along the axis, so that the running maximum moves at every step
    k = torch.arange(640, device=DEV).float()[:, None, None].expand(640, 1, 64) / 64 + 1
    v = rows((640, 1, 64), torch.bfloat16, 17).to(DEV).float()
    kv4.kv4_write(cache, k.contiguous(), v, ints([0]), starts=ints([0, 640]))
    check(torch.ones(1, 2, 64, dtype=torch.bfloat16, device=DEV), cache, [639], scaling=1.0)
    check(-torch.ones(1, 2, 64, dtype=torch.bfloat16, device=DEV), cache, [639], scaling=1.0)


def test_strided_queries_and_outputs():
    cache = filled(3, 2, 96, 72, 18)
    qkv = queries((3, 4 + 4, 72), torch.bfloat16, 19)                  # fused q | k | v rows
    out = torch.full((3, 6, 80), 7.0, dtype=torch.bfloat16, device=DEV)
    check(qkv[:, :4], cache, [95, 3, 40], out=out[:, 1:5, :72])
    assert bool((out[:, 0] == 7).all()) and bool((out[:, 5] == 7).all()) and bool((out[:, :, 72:] == 7).all())
    q = queries((4, 3, 2, 72), torch.float16, 20).permute(1, 2, 0, 3)  # [3 sequences, 2 rows, 4 heads, 72]
    check(q, cache, [94, 0, 31])


def test_rows_outside_give_zero_and_are_recorded():
    from flashbfp_b200 import kv4
    cache = filled(3, 1, 64, 32, 21)
    q = queries((3, 2, 2, 32), torch.bfloat16, 22)
    err = ints([0])
    pos = [-1, 63, 64]
    out = kv4.kv4_attention(q, cache, ints(pos), err=err)
    assert err.item() == 2
    want, bound = cached(q, cache, pos, 0, 32 ** -0.5, WEIGHT_U[q.dtype])
    assert ((out.double().cpu() - want).abs() <= bound).all()
    assert not out[0, 0].any() and not out[1, 1].any() and not out[2].any()
    kv4.check_device_errors()
    kv4.kv4_attention(q, cache, ints(pos))
    with pytest.raises(RuntimeError, match="outside the cache"):
        kv4.check_device_errors()


def test_captured_and_replayed_with_moving_positions():
    """A graph of write and attention replayed as the positions advance; two graphs in turn on two
    streams give what eager calls give."""
    from flashbfp_b200 import kv4
    seqs, kvh, h, d = 4, 2, 4, 64
    cache = filled(seqs, kvh, 384, d, 23)
    eager = kv4.KV4Cache(*[t.clone() for t in cache[:4]], d)
    pos = ints([5, 60, 200, 0])
    k, v = queries((seqs, kvh, d), torch.bfloat16, 24), queries((seqs, kvh, d), torch.bfloat16, 25)
    q = queries((seqs, h, d), torch.bfloat16, 26)
    q2, out, out2 = queries((seqs, h, d), torch.bfloat16, 27), torch.empty_like(q), torch.empty_like(q)

    def step():
        kv4.kv4_write(cache, k, v, pos)
        kv4.kv4_attention(q, cache, pos, out=out)

    step()
    torch.cuda.synchronize()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        step()
        pos.add_(1)
    with torch.cuda.graph(gb):
        kv4.kv4_attention(q2, cache, pos, window=40, out=out2)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(6):
        at = pos.clone()
        k.normal_()
        v.normal_()
        q.normal_()
        kv4.kv4_write(eager, k, v, at)
        want, want2 = kv4.kv4_attention(q, eager, at), None
        torch.cuda.synchronize()
        with torch.cuda.stream(sa):
            ga.replay()
        torch.cuda.synchronize()
        want2 = kv4.kv4_attention(q2, eager, pos, window=40)
        torch.cuda.synchronize()
        with torch.cuda.stream(sb):                                     # both at once: each has a workspace of its own
            gb.replay()
        other = kv4.kv4_attention(q, cache, at)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(out2, want2) and torch.equal(other, want)
    kv4.check_device_errors()


def test_offsets_beyond_32_bits():
    """A cache of over 2^32 bytes of keys, its last positions in a window."""
    from flashbfp_b200 import kv4
    n = 34_000_000 // 32 * 32
    cache = kv4.KV4Cache(*[torch.zeros(1, 1, n, w, dtype=t, device=DEV)
                           for w, t in ((128, torch.uint8), (8, torch.bfloat16)) * 2], 256)
    k, v = (rows((300, 1, 256), torch.bfloat16, 30 + i).to(DEV).clamp(-30, 30) for i in range(2))
    kv4.kv4_write(cache, k, v, ints([n - 300]), starts=ints([0, 300]))
    check(queries((1, 2, 256), torch.bfloat16, 32), cache, [n - 1], window=290)


def test_many_sequences():
    """More sequences than a warp looks through at once."""
    seqs = 150
    cache = filled(seqs, 2, 96, 64, 40)
    pos = [(37 * b) % 96 for b in range(seqs)]
    check(queries((seqs, 4, 64), torch.bfloat16, 42), cache, pos)
    check(queries((seqs, 2, 4, 64), torch.bfloat16, 43), cache, [max(0, p - 1) for p in pos], window=33)


def test_two_streams_at_once():
    """Calls whose sequences are joined from parts, each with a workspace of its own."""
    from flashbfp_b200 import kv4
    cache = filled(2, 2, 6016, 128, 44)
    qs = [queries((2, 4, 128), torch.bfloat16, 46 + i) for i in range(2)]
    pos = ints([6000, 5000])
    want = [kv4.kv4_attention(q, cache, pos) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for q, st in zip(qs, streams):
            with torch.cuda.stream(st):
                got.append(kv4.kv4_attention(q, cache, pos))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    kv4.check_device_errors()
