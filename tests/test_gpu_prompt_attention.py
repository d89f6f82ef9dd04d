"""Attention of packed prompts against its definition in 64 bits, with the bounds that
attention_reference derives; the weights are rounded to the inputs' type (u = eps / 2)."""
import math

import pytest
import torch

from attention_reference import packed, starts_of
from test_gpu_kv4_store import ints

pytestmark = pytest.mark.gpu
DEV = "cuda"


def normal(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def check(q, k, v, lens, kv_lens=None, window=0, scaling=None, out=None):
    from flashbfp_b200 import attention
    starts = starts_of(lens)
    kv_starts = starts if kv_lens is None else starts_of(kv_lens)
    got = attention.prompt_attention(q, k, v, ints(starts), kv_starts=None if kv_lens is None else ints(kv_starts),
                                     window=window, scaling=scaling, out=out)
    attention.check_device_errors()
    s = q.shape[-1] ** -0.5 if scaling is None else scaling
    n = starts[-1]
    want, bound = packed(q, k, v, starts, kv_starts, window, s, torch.finfo(q.dtype).eps / 2)
    g = got[:n].double().cpu()
    assert torch.isfinite(g).all()
    off = (g - want[:n]).abs()
    assert (off <= bound[:n]).all(), (off / bound[:n]).max().item()
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (16, 8, 256), (8, 1, 128), (3, 1, 40), (6, 2, 96),
                                                (12, 1, 8), (5, 5, 136), (40, 2, 80)])
def test_packed(dtype, heads, kv_heads, dim):
    lens = [1, 0, 130, 17, 128, 2, 257]
    t = sum(lens)
    q, k, v = (normal((t, h, dim), dtype, i) for i, h in enumerate((heads, kv_heads, kv_heads)))
    check(q, k, v, lens)
    for window in (1, 5, 128, 200):
        check(q, k, v, lens, window=window)


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257, 500])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_lengths(n, dim):
    q, k, v = (normal((n, h, dim), torch.bfloat16, i) for i, h in enumerate((4, 2, 2)))
    check(q, k, v, [n])
    check(q, k, v, [n], window=70)


@pytest.mark.parametrize("dim,dtype", [(64, torch.bfloat16), (128, torch.float16), (256, torch.bfloat16),
                                       (72, torch.float16)])
def test_context_before_the_rows(dim, dtype):
    """More keys than rows (a chunk late in a prompt), and as the limit one row over many keys."""
    lens, kv_lens = [1, 40, 130, 0, 3], [700, 41, 300, 9, 3]
    q = normal((sum(lens), 4, dim), dtype, 1)
    k, v = normal((sum(kv_lens), 2, dim), dtype, 2), normal((sum(kv_lens), 2, dim), dtype, 3)
    check(q, k, v, lens, kv_lens)
    check(q, k, v, lens, kv_lens, window=150)
    check(q, k, v, lens, kv_lens, window=3)


@pytest.mark.parametrize("rows_,keys,heads,kv_heads,dim", [(1, 9000, 2, 1, 128), (16, 5001, 16, 8, 256),
                                                           (100, 3333, 4, 1, 64)])
def test_few_rows_over_a_long_axis(rows_, keys, heads, kv_heads, dim):
    """The keys of a tile split over CTAs and joined."""
    q = normal((rows_, heads, dim), torch.bfloat16, 1)
    k, v = normal((keys, kv_heads, dim), torch.bfloat16, 2), normal((keys, kv_heads, dim), torch.bfloat16, 3)
    a = check(q, k, v, [rows_], [keys])
    assert torch.equal(check(q, k, v, [rows_], [keys]), a)              # the same bits every time
    check(q, k, v, [rows_], [keys], window=2000)


def test_rows_that_see_nothing_give_zero():
    """Fewer keys than rows: the first rows stand before the first key. Sequences without keys."""
    lens, kv_lens = [5, 3, 200], [3, 0, 150]
    q = normal((208, 2, 64), torch.bfloat16, 1)
    k, v = normal((153, 1, 64), torch.bfloat16, 2), normal((153, 1, 64), torch.bfloat16, 3)
    for window in (0, 2):
        got = check(q, k, v, lens, kv_lens, window=window)
        assert not got[:2].any() and not got[5:8].any() and not got[8:58].any()


def test_rows_behind_the_last_sequence_stay():
    q, k, v = (normal((150, h, 128), torch.bfloat16, i) for i, h in enumerate((4, 2, 2)))
    k[90:], v[90:], q[90:] = math.nan, math.inf, math.nan
    out = torch.full_like(q, 7.0)
    check(q, k, v, [60, 30], out=out)
    assert bool((out[90:] == 7).all())


def test_neighbours_do_not_leak():
    """NaN and infinities in one sequence, in the unseen part of its own keys and outside a window."""
    lens = [100, 100, 100]
    q, k, v = (normal((300, h, 64), torch.bfloat16, i) for i, h in enumerate((2, 1, 1)))
    clean = check(q, k, v, lens)
    k[100:200], v[100:200] = math.nan, math.inf
    from flashbfp_b200 import attention
    got = attention.prompt_attention(q, k, v, ints([0, 100, 200, 300]))
    assert torch.equal(got[:100], clean[:100]) and torch.equal(got[200:], clean[200:])
    q, k, v = (normal((400, h, 64), torch.bfloat16, i) for i, h in enumerate((2, 1, 1)))
    late = check(q, k, v, [400], window=50)
    k[:200], v[:200] = math.inf, math.nan
    got = attention.prompt_attention(q, k, v, ints([0, 400]), window=50)
    assert torch.equal(got[250:], late[250:])
    # values after a row's place: earlier rows are not touched by them
    k2, v2 = normal((400, 1, 64), torch.bfloat16, 5), normal((400, 1, 64), torch.bfloat16, 6)
    a = attention.prompt_attention(q, k2, v2, ints([0, 400]))
    k2[300:], v2[300:] = math.nan, math.nan
    assert torch.equal(attention.prompt_attention(q, k2, v2, ints([0, 400]))[:300], a[:300])


def test_views_of_fused_rows_and_heads_first():
    t, h, kvh, d = 200, 4, 2, 128
    rows = normal((t, h + 2 * kvh, d), torch.bfloat16, 1)
    check(rows[:, :h], rows[:, h:h + kvh], rows[:, h + kvh:], [120, 80])
    q = normal((h, t, d), torch.float16, 2).transpose(0, 1)
    k, v = normal((kvh, t, d), torch.float16, 3).transpose(0, 1), normal((t, kvh, d + 8), torch.float16, 4)[..., :d]
    out = torch.full((t, 2 * h, d + 8), 3.0, dtype=torch.float16, device=DEV)
    check(q, k, v, [t], out=out[:, ::2, :d])
    assert bool((out[:, 1::2] == 3).all()) and bool((out[:, :, d:] == 3).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sharp_and_flat_softmax(dtype):
    q, k, v = (normal((300, h, 64), dtype, i) for i, h in enumerate((2, 1, 1)))
    for scaling in (0.0, 1e-3, 2.0, 20.0, -2.0):
        check(q, k, v, [300], scaling=scaling)
    # scores that grow or fall along the axis: the running maximum moves at every step, or never
    ramp = (torch.arange(300, device=DEV).float() / 16)[:, None, None].expand(300, 1, 64).to(dtype).contiguous()
    one = torch.ones(300, 2, 64, dtype=dtype, device=DEV)
    check(one, ramp, v, [300], scaling=0.5)
    check(-one, ramp, v, [300], scaling=0.5)


def test_long_prompt():
    q, k, v = (normal((5000, h, 128), torch.bfloat16, i) for i, h in enumerate((2, 1, 1)))
    check(q, k, v, [4000, 1000])
    check(q, k, v, [5000], window=1024)


def test_captured_and_replayed_with_other_lengths():
    from flashbfp_b200 import attention
    q, k, v = (normal((300, h, 128), torch.bfloat16, i) for i, h in enumerate((4, 2, 2)))
    starts = ints([0, 100, 300])
    out = torch.zeros_like(q)
    attention.prompt_attention(q, k, v, starts, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        attention.prompt_attention(q, k, v, starts, out=out)
    for lens in ([100, 200], [1, 0], [299, 1], [0, 300], [150, 20]):
        starts.copy_(ints(starts_of(lens)))
        out.fill_(5.0)
        g.replay()
        torch.cuda.synchronize()
        n = sum(lens)
        want = attention.prompt_attention(q, k, v, starts)
        assert torch.equal(out[:n], want[:n]) and bool((out[n:] == 5).all())
    attention.check_device_errors()


def test_two_streams_at_once():
    from flashbfp_b200 import attention
    sets = [[normal((400, h, 256), torch.bfloat16, 10 * j + i) for i, h in enumerate((4, 2, 2))] for j in range(2)]
    want = [attention.prompt_attention(*s, ints([0, 400])) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(attention.prompt_attention(*s, ints([0, 400])))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_starts_of_any_contents_stay_inside():
    """Descending, negative and too large starts: nothing is read or written outside the tensors."""
    from flashbfp_b200 import attention
    q, k, v = (normal((200, h, 64), torch.bfloat16, i) for i, h in enumerate((2, 1, 1)))
    for starts, kv_starts in (([5, 3, 1], [0, 100, 200]), ([-50, 100, 900], [-20, 400, 90]), ([0, 100, 200], [300, 200, -5]),
                              ([500, 600, 700], [0, 1, 2])):
        attention.prompt_attention(q, k, v, ints(starts), kv_starts=ints(kv_starts))
    attention.check_device_errors()


def test_many_sequences():
    """More sequences than a warp looks through at once, a third of them empty."""
    lens = [(0, 3, 1)[i % 3] for i in range(700)]
    kv_lens = [n + 7 * (i % 5) for i, n in enumerate(lens)]
    q = normal((sum(lens), 4, 64), torch.bfloat16, 1)
    k, v = (normal((sum(kv_lens), 2, 64), torch.bfloat16, i) for i in (2, 3))
    check(q, k, v, lens, kv_lens=kv_lens)
    check(q, k, v, lens, kv_lens=kv_lens, window=4)


def test_broadcast_keys():
    """Keys and values of one head expanded to several: a stride of zero."""
    q = normal((130, 4, 64), torch.bfloat16, 1)
    k, v = (normal((130, 1, 64), torch.bfloat16, i) for i in (2, 3))
    a = check(q, k, v, [130])
    b = check(q, k.expand(130, 4, 64), v.expand(130, 4, 64), [130])
    assert a.shape == b.shape


def test_out_in_place_of_padding():
    """Rows of a wider buffer as the result: what lies between them stays."""
    q, k, v = (normal((70, h, 128), torch.float16, i) for i, h in enumerate((4, 2, 2)))
    buf = torch.full((70, 5, 136), 3.0, dtype=torch.float16, device=DEV)
    check(q, k, v, [70], out=buf[:, :4, :128])
    assert bool((buf[:, 4] == 3).all()) and bool((buf[:, :, 128:] == 3).all())
