"""Writing rows into the 4-bit cache and reading them back: bytes, scales and values exactly those of the
definition in 64 bits, and nothing else of the cache or of the output touched."""
import math

import pytest
import torch

from attention_reference import starts_of, stored

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def rows(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(2 * torch.randn(shape[:-1], generator=g))[..., None]
    x[..., ::7] *= 10
    return x.to(dtype)


def garbage(cache, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    for t in cache[:4]:
        raw = t.view(torch.uint8)
        raw.copy_(torch.randint(0, 256, raw.shape, generator=g, device=DEV, dtype=torch.uint8))
    return [t.clone() for t in cache[:4]]


def expect(before, cache, k, v, pos, starts):
    """The cache's four tensors after the write, from its contents before (CPU)."""
    want = [t.cpu() for t in before]
    for x, values, scales in ((k, want[0], want[1]), (v, want[2], want[3])):
        packed, s, _ = stored(x)
        for b in range(len(starts) - 1):
            for r in range(starts[b], starts[b + 1]):
                p = pos[b] + r - starts[b]
                if 0 <= p < values.shape[2]:
                    values[b, :, p], scales[b, :, p] = packed[r], s[r].to(torch.bfloat16)
    return want


def same(a, b):
    return torch.equal(a.cpu().view(torch.uint8), b.cpu().view(torch.uint8))


def same_nan(a, b):                       # NaN scales: any NaN
    a, b = a.cpu(), b.cpu()
    if a.dtype == torch.uint8:
        return torch.equal(a, b)
    nan = torch.isnan(a) & torch.isnan(b)
    return torch.equal(torch.where(nan, 0, a.view(torch.int16)), torch.where(nan, 0, b.view(torch.int16)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim,heads", [(8, 1), (40, 3), (64, 2), (96, 1), (128, 5), (256, 8)])
def test_write_and_read(dtype, dim, heads):
    from flashbfp_b200 import kv4
    lens, pos = [3, 0, 37, 1], [29, 5, 60, 0]
    starts = starts_of(lens)
    t = starts[-1]
    k, v = rows((t + 2, heads, dim), dtype, 1).to(DEV), rows((t + 2, heads, dim), dtype, 2).to(DEV)
    cache = kv4.empty_cache(4, heads, 97, dim, DEV)
    assert cache.positions == 128
    before = garbage(cache, 3)
    kv4.kv4_write(cache, k, v, ints(pos), starts=ints(starts))
    kv4.check_device_errors()
    want = expect(before, cache, k.cpu(), v.cpu(), pos, starts)
    for got, w in zip(cache, want):
        assert same_nan(got, w)
    # read back, older rows (whose scales may be anything) and what was written among them
    first, lens2 = [29, 0, 58, 0], [3, 7, 39, 0]
    s2 = starts_of(lens2)
    for out_dtype in (torch.float32, torch.bfloat16, torch.float16):
        out = [torch.full((s2[-1] + 1, heads, dim), 5.0, dtype=out_dtype, device=DEV) for _ in range(2)]
        got = kv4.kv4_read(cache, ints(first), ints(s2), out=out)
        kv4.check_device_errors()
        for x, values, scales in ((got[0], want[0], want[1]), (got[1], want[2], want[3])):
            n = torch.stack((values & 15, values >> 4), -1).flatten(-2).double() - 8
            held = (n * scales.double().repeat_interleave(32, -1))[..., :dim]
            ref = torch.cat([held[b, :, first[b]:first[b] + lens2[b]].transpose(0, 1) for b in range(4)]).to(out_dtype)
            assert torch.equal(torch.nan_to_num(x[:-1].cpu()), torch.nan_to_num(ref))
            assert torch.equal(torch.isnan(x[:-1].cpu()), torch.isnan(ref))
            assert bool((x[-1] == 5).all())
    k2, v2 = kv4.kv4_read(cache, ints(first), ints(s2), rows=s2[-1], dtype=torch.float32)
    assert k2.shape == (s2[-1], heads, dim) and v2.dtype == torch.float32


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_special_values(dtype):
    """Infinities, NaN, zeros, subnormals, ties and the largest numbers, each alone in its group."""
    from flashbfp_b200 import kv4
    tiny, big = torch.finfo(dtype).tiny, torch.finfo(dtype).max
    groups = [[0.0], [-0.0], [math.inf, 1.0], [-math.inf], [math.nan, 2.0], [tiny, tiny / 4], [tiny * 7, tiny],
              [big, -big, big / 2, big / 14], [7.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 6.5, -6.5],
              [14.0, 1.0, 3.0, 5.0, -7.0], [1.0, 1e-6, -1e-6], [tiny / 64, -tiny / 64]]
    x = torch.zeros(1, 1, 32 * len(groups[:8]), dtype=dtype)
    y = torch.zeros(1, 1, 32 * len(groups[:8]), dtype=dtype)
    for i, g in enumerate(groups):
        z = x if i < 8 else y
        z[0, 0, 32 * (i % 8):32 * (i % 8) + len(g)] = torch.tensor(g, dtype=torch.float64).to(dtype)
    cache = kv4.empty_cache(1, 1, 32, 256, DEV)
    before = garbage(cache, 5)
    kv4.kv4_write(cache, x.to(DEV), y.to(DEV), ints([4]))
    want = expect(before, cache, x, y, [4], [0, 1])
    for got, w in zip(cache, want):
        assert same_nan(got, w)
    k, v = kv4.kv4_read(cache, ints([4]), ints([0, 1]), rows=1, dtype=torch.float32)
    for got, z in ((k, x), (v, y)):
        ref = stored(z)[2].float()
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(ref))
        assert torch.equal(torch.nan_to_num(got.cpu()), torch.nan_to_num(ref))


def test_fp32_scales_and_values_next_to_borders():
    """fp32 rows whose quotients fall onto, or a last place beside, the middle of two scales or values."""
    from flashbfp_b200 import kv4
    g = torch.Generator().manual_seed(7)
    n = 4096
    mid = (torch.randint(128, 256, (n,), generator=g).double() + 0.5) * 7 * torch.exp2(torch.randint(-9, 9, (n,), generator=g).double())
    top = mid.float()
    top = (top.view(torch.int32) + torch.randint(-1, 2, (n,), generator=g, dtype=torch.int32)).view(torch.float32)
    s = stored(top[:, None, None].expand(n, 1, 32).contiguous())[1][:, 0, 0]
    x = torch.zeros(n, 1, 32)
    x[:, 0, 0] = top
    h = (torch.randint(-7, 7, (n, 31), generator=g).double() + 0.5) * s[:, None]
    h = h.float()
    x[:, 0, 1:] = (h.view(torch.int32) + torch.randint(-1, 2, (n, 31), generator=g, dtype=torch.int32)).view(torch.float32)
    cache = kv4.empty_cache(1, 1, n, 32, DEV)
    before = [t.clone() for t in cache[:4]]
    kv4.kv4_write(cache, x.to(DEV), -x.to(DEV), ints([0]), starts=ints([0, n]))
    want = expect(before, cache, x, -x, [0], [0, n])
    for got, w in zip(cache, want):
        assert same(got, w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_alignment(dtype):
    """Views of fused rows, heads before rows, rows that start off 16 bytes."""
    from flashbfp_b200 import kv4
    t, h, d = 33, 2, 72
    base = rows((t, 3 * h, d + 1), dtype, 11).to(DEV)
    fused = base[:, :, :d]                                             # odd strides
    heads_first = rows((h, t, d), dtype, 12).to(DEV).transpose(0, 1)
    off = rows((t * h * d + 3,), dtype, 13).to(DEV)[3:].view(t, h, d)  # unaligned start
    starts = [0, t]
    for k, v in ((fused[:, h:2 * h], fused[:, 2 * h:]), (heads_first, off)):
        cache = kv4.empty_cache(1, h, 64, d, DEV)
        before = garbage(cache, 14)
        kv4.kv4_write(cache, k, v, ints([7]), starts=ints(starts))
        want = expect(before, cache, k.cpu(), v.cpu(), [7], starts)
        for got, w in zip(cache, want):
            assert same_nan(got, w)
        out = [torch.zeros(h, t, d, dtype=dtype, device=DEV).transpose(0, 1),
               torch.zeros(t * h * d + 1, dtype=dtype, device=DEV)[1:].view(t, h, d)]
        kv4.kv4_read(cache, ints([7]), ints(starts), out=out)
        for x, z in zip(out, (k, v)):
            assert torch.equal(x.cpu(), stored(z)[2].to(dtype))


def test_positions_outside_are_recorded_and_skipped():
    from flashbfp_b200 import kv4
    k = rows((6, 2, 64), torch.bfloat16, 1).to(DEV)
    cache = kv4.empty_cache(3, 2, 32, 64, DEV)
    before = garbage(cache, 2)
    pos, starts = [-1, 31, 30], [0, 2, 4, 6]                          # outside at the front, at the end, inside
    kv4.kv4_write(cache, k, k, ints(pos), starts=ints(starts))
    with pytest.raises(RuntimeError, match="outside the cache"):
        kv4.check_device_errors()
    kv4.check_device_errors()                                          # cleared
    for got, w in zip(cache, expect(before, cache, k.cpu(), k.cpu(), pos, starts)):
        assert same_nan(got, w)
    err = ints([0])
    out = [torch.full((6, 2, 64), 3.0, device=DEV) for _ in range(2)]
    kv4.kv4_read(cache, ints(pos), ints(starts), out=out, err=err)
    assert err.item() == 2 and bool((out[0][0] == 3).all()) and bool((out[0][3] == 3).all())
    kv4.check_device_errors()                                          # the caller's word, not the device's


def test_starts_of_any_contents_stay_inside():
    """Descending, negative and too large starts write no row but those that some sequence holds."""
    from flashbfp_b200 import kv4
    k = rows((8, 1, 32), torch.bfloat16, 1).to(DEV)
    for starts in ([5, 3, 1], [-4, 100, 2], [2, 2, 2], [9, 9, 9]):
        cache = kv4.empty_cache(2, 1, 32, 32, DEV)
        before = garbage(cache, 2)
        kv4.kv4_write(cache, k, k, ints([0, 0]), starts=ints(starts))
        torch.cuda.synchronize()
        changed = (cache.k_values != before[0]).any(-1).sum().item()
        assert changed <= 8
        try:
            kv4.check_device_errors()
        except RuntimeError:
            pass


def test_last_position_beyond_32_bits():
    """A cache whose byte offsets pass 2^32."""
    from flashbfp_b200 import kv4
    n = 34_000_000 // 32 * 32
    cache = kv4.KV4Cache(*[torch.zeros(1, 1, n, w, dtype=t, device=DEV)
                           for w, t in ((128, torch.uint8), (8, torch.bfloat16)) * 2], 256)
    k, v = rows((2, 1, 256), torch.bfloat16, 1).to(DEV), rows((2, 1, 256), torch.bfloat16, 2).to(DEV)
    kv4.kv4_write(cache, k, v, ints([n - 2]), starts=ints([0, 2]))
    got = kv4.kv4_read(cache, ints([n - 2]), ints([0, 2]), rows=2)
    kv4.check_device_errors()
    for x, z in zip(got, (k, v)):
        assert torch.equal(x.cpu(), stored(z)[2].to(torch.bfloat16))
    assert not cache.k_values[0, 0, :n - 2].any() and not cache.v_scales[0, 0, :n - 2].any()


def test_a_row_read_back_and_written_again_is_held_as_it_was():
    """What fp32 holds exactly: n s with max|n| = 7 quantises to the same scale and whole numbers."""
    from flashbfp_b200 import kv4
    k, v = rows((64, 4, 128), torch.bfloat16, 21).to(DEV), rows((64, 4, 128), torch.bfloat16, 22).to(DEV)
    a, b = kv4.empty_cache(1, 4, 64, 128, DEV), kv4.empty_cache(1, 4, 64, 128, DEV)
    kv4.kv4_write(a, k, v, ints([0]), starts=ints([0, 64]))
    kv4.kv4_write(b, *kv4.kv4_read(a, ints([0]), ints([0, 64]), rows=64, dtype=torch.float32), ints([0]),
                  starts=ints([0, 64]))
    for x, y in zip(a[:4], b[:4]):
        assert same(x, y)
