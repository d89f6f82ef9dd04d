"""Refusals of the attention and cache calls' Python entry points."""
import pytest
import torch

from test_gpu_kv4_store import ints

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_prompt_attention_refuses():
    from flashbfp_b200.attention import prompt_attention as f
    bf = dict(dtype=torch.bfloat16, device=DEV)
    q, k, s = torch.zeros(8, 4, 64, **bf), torch.zeros(8, 2, 64, **bf), ints([0, 8])
    assert not f(q, k, k, s).any()
    with pytest.raises(NotImplementedError, match="bf16 or fp16"):
        f(q.float(), k.float(), k.float(), s)
    with pytest.raises(ValueError, match="one dtype"):
        f(q, k.half(), k, s)
    with pytest.raises(ValueError, match="three dimensions"):
        f(q[0], k, k, s)
    with pytest.raises(ValueError, match="shape"):
        f(q, k, k[:7], s)
    with pytest.raises(ValueError, match="heads"):
        f(q[:, :3], k, k, s)
    with pytest.raises(ValueError, match="multiple of 8"):
        f(q[..., :60], k[..., :60], k[..., :60], s)
    with pytest.raises(ValueError, match="int32"):
        f(q, k, k, s.long())
    with pytest.raises(ValueError, match="starts"):
        f(q, k, k, s[:1])
    with pytest.raises(ValueError, match="kv_starts"):
        f(q, k, k, s, kv_starts=ints([0, 4, 8]))
    with pytest.raises(RuntimeError, match="CUDA"):
        f(q, k, k, s.cpu())
    with pytest.raises(ValueError, match="window"):
        f(q, k, k, s, window=-1)
    with pytest.raises(ValueError, match="finite"):
        f(q, k, k, s, scaling=float("nan"))
    with pytest.raises(ValueError, match="contiguous"):
        f(q.transpose(1, 2).contiguous().transpose(1, 2), k, k, s)
    with pytest.raises(ValueError, match="overlap"):
        f(q, k, k, s, out=torch.zeros(8, 1, 64, **bf).expand(8, 4, 64))
    with pytest.raises(ValueError, match="dtype"):
        f(q, k, k, s, out=torch.zeros(8, 4, 64, device=DEV))
    with pytest.raises(RuntimeError, match="requires a gradient"):
        f(q, k, k, s, out=torch.zeros(8, 4, 64, requires_grad=True, **bf))
    with pytest.raises(ValueError, match="no keys"):
        f(q, k[:0], k[:0], s)
    with pytest.raises(ValueError, match="aligned|strides"):
        f(torch.zeros(8 * 4 * 64 + 1, **bf)[1:].view(8, 4, 64), k, k, s)
    assert f(q[:0], k, k, ints([0, 0])).shape == (0, 4, 64)
    g = q.clone().requires_grad_()
    assert not f(g, k, k, s).requires_grad


def test_cache_calls_refuse():
    from flashbfp_b200 import kv4
    bf = dict(dtype=torch.bfloat16, device=DEV)
    c = kv4.empty_cache(2, 2, 64, 64, DEV)
    k, q, pos = torch.zeros(2, 2, 64, **bf), torch.zeros(2, 4, 64, **bf), ints([0, 0])
    kv4.kv4_write(c, k, k, pos)
    with pytest.raises(TypeError, match="KV4Cache"):
        kv4.kv4_write(c[:4], k, k, pos)
    with pytest.raises(ValueError, match="pass starts"):
        kv4.kv4_write(c, k[:1], k[:1], pos)
    with pytest.raises(ValueError, match="pos"):
        kv4.kv4_write(c, k, k, pos[:1])
    with pytest.raises(ValueError, match="one dtype"):
        kv4.kv4_write(c, k, k.float(), pos)
    with pytest.raises(NotImplementedError, match="dtype"):
        kv4.kv4_write(c, k.double(), k.double(), pos)
    with pytest.raises(ValueError, match="shape"):
        kv4.kv4_write(c, k[..., :32], k[..., :32], pos)
    with pytest.raises(ValueError, match="starts"):
        kv4.kv4_read(c, pos, ints([0, 1]), rows=2)
    with pytest.raises(ValueError, match="number of rows"):
        kv4.kv4_read(c, pos, ints([0, 1, 2]))
    with pytest.raises(ValueError, match="overlap"):
        kv4.kv4_read(c, pos, ints([0, 1, 2]), out=[k[:1].expand(2, 2, 64), k])
    with pytest.raises(ValueError, match="k_scales"):
        kv4.kv4_write(kv4.KV4Cache(c.k_values, c.k_scales[:, :, :32], c.v_values, c.v_scales, 64), k, k, pos)
    with pytest.raises(ValueError, match="k_values"):
        kv4.kv4_write(kv4.KV4Cache(*c[:4], 96), k, k, pos)
    with pytest.raises(ValueError, match="32"):
        kv4.kv4_write(kv4.KV4Cache(*[t[:, :, :33].contiguous() for t in c[:4]], 64), k, k, pos)
    with pytest.raises(ValueError, match="q must be"):
        kv4.kv4_attention(q[:1], c, pos)
    with pytest.raises(ValueError, match="heads"):
        kv4.kv4_attention(q[:, :3], c, pos)
    with pytest.raises(NotImplementedError, match="bf16 or fp16"):
        kv4.kv4_attention(q.float(), c, pos)
    with pytest.raises(ValueError, match="shape and dtype"):
        kv4.kv4_attention(q, c, pos, out=q[:, :2])
    with pytest.raises(ValueError, match="window"):
        kv4.kv4_attention(q, c, pos, window=-2)
    with pytest.raises(ValueError, match="err"):
        kv4.kv4_attention(q, c, pos, err=ints([0, 0]))


def test_written_tensors_count_as_modified():
    from flashbfp_b200 import kv4
    c = kv4.empty_cache(1, 1, 32, 32, DEV)
    k = torch.zeros(1, 1, 32, device=DEV)
    before = [t._version for t in c[:4]]
    kv4.kv4_write(c, k, k, ints([0]))
    assert all(t._version > b for t, b in zip(c[:4], before))
    out = [torch.zeros(1, 1, 32, device=DEV) for _ in range(2)]
    kv4.kv4_read(c, ints([0]), ints([0, 1]), out=out)
    assert all(t._version > 0 for t in out)


def test_append_refuses():
    from flashbfp_b200 import kv4
    bf = dict(dtype=torch.bfloat16, device=DEV)
    c = kv4.empty_cache(2, 1, 32, 32, DEV)
    qkv, w, angles, out = torch.zeros(2, 4 * 32, **bf), torch.zeros(32, **bf), torch.zeros(32, 32, **bf), torch.zeros(2, 2, 32, **bf)
    pos = ints([0, 0])

    def f(cache=c, qkv=qkv, w=w, angles=angles, pos=pos, out=out, starts=None):
        kv4.kv4_append(cache, qkv, w, w, 1e-6, angles, angles, pos, out, starts=starts)

    f()
    wide = kv4.empty_cache(2, 1, 64, 32, DEV)
    for i, name in enumerate(("k_values", "k_scales", "v_values", "v_scales")):
        with pytest.raises(ValueError, match=name):              # a tensor of another length, a view, another type
            f(cache=kv4.KV4Cache(*[(wide if i and j == i else c)[j] for j in range(4)], 32) if i else
              kv4.KV4Cache(wide.k_values[:, :, :32], *c[1:4], 32))
        with pytest.raises(ValueError, match=name):
            f(cache=kv4.KV4Cache(*[t.to(torch.float16) if j == i else t for j, t in enumerate(c[:4])], 32))
    with pytest.raises(ValueError, match="do not hold heads"):
        f(qkv=qkv[:, :64].contiguous())
    with pytest.raises(ValueError, match="q_out"):
        f(out=out[:, :1])
    with pytest.raises(ValueError, match="positions"):
        f(angles=angles[:31])
    with pytest.raises(ValueError, match="pos"):
        f(pos=pos.long())
    with pytest.raises(ValueError, match="pass starts"):
        f(qkv=qkv[:1], out=out[:1])
    with pytest.raises(ValueError, match="starts"):
        f(starts=ints([0, 2]))
    with pytest.raises(RuntimeError, match="requires a gradient"):
        f(out=torch.zeros(2, 2, 32, requires_grad=True, **bf))
    with pytest.raises(RuntimeError, match="CUDA"):
        f(qkv=qkv.cpu())
