"""Calls of the attention and cache entry points that their documentation allows or refuses: under inference mode, on
tensors of other shapes, with windows and scalings at the ends of their types."""
import pytest
import torch

from test_gpu_kv4_store import ints

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = dict(dtype=torch.bfloat16, device=DEV)


def everything(seed=0):
    """One call each; all results."""
    from flashbfp_b200 import attention, kv4
    g = torch.Generator(device=DEV).manual_seed(seed)
    d = 32
    cache = kv4.empty_cache(2, 1, 64, d, DEV)
    qkv = torch.randn(2, 4 * d, generator=g, device=DEV).bfloat16()
    w, ang, q = torch.zeros(d, **BF), torch.ones(64, d, **BF), torch.empty(2, 2, d, **BF)
    pos = ints([3, 9])
    kv4.kv4_append(cache, qkv, w, w, 1e-6, ang, ang, pos, q)
    k = torch.randn(2, 1, d, generator=g, device=DEV).bfloat16()
    kv4.kv4_write(cache, k, k, ints([4, 10]))
    back = kv4.kv4_read(cache, ints([3, 9]), ints([0, 2, 4]), rows=4)
    o = kv4.kv4_attention(q, cache, ints([4, 10]))
    p = attention.prompt_attention(q, *back, ints([0, 1, 2]), kv_starts=ints([0, 2, 4]))
    attention.check_device_errors()
    return [*cache[:4], q, *back, o, p]


def test_inference_mode():
    want = everything()
    with torch.inference_mode():
        got = everything()
    assert all(t.is_inference() for t in got)
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    with torch.no_grad():
        for a, b in zip(want, everything()):
            assert torch.equal(a, b)


def test_scalings_at_the_ends_of_fp32():
    from flashbfp_b200 import attention, kv4
    q, k, s = torch.ones(4, 2, 64, **BF), torch.ones(4, 1, 64, **BF), ints([0, 4])
    cache = kv4.empty_cache(4, 1, 32, 64, DEV)
    for scaling in (1e300, -1e39, 3e38):
        with pytest.raises(ValueError, match="finite"):
            attention.prompt_attention(q, k, k, s, scaling=scaling)
        with pytest.raises(ValueError, match="finite"):
            kv4.kv4_attention(q, cache, ints([0] * 4), scaling=scaling)
    for scaling in (1e-45, -1e-40, 1e30):                    # equal scores: the same mean whatever they are times
        assert torch.equal(attention.prompt_attention(q, k, k, s, scaling=scaling), q)


def test_both_results_in_one_place():
    from flashbfp_b200 import kv4
    cache = kv4.empty_cache(1, 2, 32, 64, DEV)
    x = torch.zeros(4, 2, 64, **BF)
    with pytest.raises(ValueError, match="one place"):
        kv4.kv4_read(cache, ints([0]), ints([0, 4]), out=[x, x])
    rows = torch.ones(4, 6, 64, **BF)                        # two parts of fused rows are two places
    kv4.kv4_read(cache, ints([0]), ints([0, 4]), out=[rows[:, 2:4], rows[:, 4:]])
    assert bool((rows[:, :2] == 1).all()) and not rows[:, 2:].any()
    kv4.kv4_read(cache, ints([0]), ints([0, 0]), out=[x[:0], x[:0]])


def test_append_refuses_other_shapes():
    from flashbfp_b200 import kv4
    d = 32
    cache = kv4.empty_cache(2, 1, 32, d, DEV)
    ok = dict(qkv=torch.zeros(2, 4 * d, **BF), w=torch.zeros(d, **BF), ang=torch.zeros(32, d, **BF), out=torch.zeros(2, 2, d, **BF))

    def f(**kw):
        a = {**ok, **kw}
        kv4.kv4_append(cache, a["qkv"], a["w"], a["w"], 1e-6, a["ang"], a["ang"], ints([0, 0]), a["out"])

    f()
    for bad, text in ((dict(qkv=torch.zeros(8 * d, **BF)), "do not hold heads"), (dict(qkv=torch.zeros(2, 4, d, **BF)), "do not hold heads"),
                      (dict(qkv=torch.zeros((), **BF)), "do not hold heads"), (dict(ang=torch.zeros(32 * d, **BF)), "one value per value"),
                      (dict(ang=torch.zeros(32, 1, d, **BF)), "one value per value"), (dict(out=torch.zeros(2, 3, d, **BF)), "q_out")):
        with pytest.raises(ValueError, match=text):
            f(**bad)
