"""Prompts' attention with keys and values out of L2, where loads land late and out of order: the same bits as with
them in L2 (a row's sums are made in one order)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("heads,kv_heads,dim,lens,past,window", [
    (16, 8, 256, [128], 20000, 0), (16, 8, 256, [2048], 0, 0), (4, 2, 256, [900, 33, 1500, 700], 0, 300),
    (8, 2, 136, [1000, 1000], 3000, 0), (16, 8, 128, [1500, 40], 0, 500), (8, 8, 64, [3000], 0, 0)])
def test_cold_loads_give_what_warm_ones_give(heads, kv_heads, dim, lens, past, window):
    from flashbfp_b200 import attention
    g = torch.Generator(device=DEV).manual_seed(1)
    t, n = sum(lens), sum(lens) + past * len(lens)
    q, k, v = (torch.randn(r, h, dim, generator=g, device=DEV).bfloat16() for r, h in ((t, heads), (n, kv_heads), (n, kv_heads)))
    starts = torch.tensor([0] + lens, device=DEV).cumsum(0).int()
    kv_starts = torch.tensor([0] + [x + past for x in lens], device=DEV).cumsum(0).int()

    def call():
        return attention.prompt_attention(q, k, v, starts, kv_starts=kv_starts, window=window)

    call()
    warm = call()
    assert torch.isfinite(warm).all()
    flush = torch.empty(1 << 29, dtype=torch.uint8, device=DEV)          # four times L2
    for i in range(40):
        flush.fill_(i)
        assert torch.equal(call(), warm), i
    attention.check_device_errors()
