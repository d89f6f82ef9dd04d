"""Groups of the 4-bit cache whose scale is one of bf16's lowest subnormals, where rounding max|x| / 7 to a scale moves
it far: whole numbers stay within -7..7, and no value touches its neighbour."""
import pytest
import torch

from test_gpu_kv4_store import ints

pytestmark = pytest.mark.gpu
DEV = "cuda"


def held(x):
    """The definition in whole steps of 2^-149 for rows of tiny values: (whole numbers, scales in steps of 2^-133)."""
    steps = torch.ldexp(x.double(), torch.tensor(149)).round().long()              # exact: fp32 holds such steps
    g = steps.unflatten(-1, (-1, 32))
    top = g.abs().amax(-1)
    s = (2 * top + 7 * (1 << 16)) // (14 * (1 << 16))                              # nearest of top / 7 to 2^-133 ...
    tie = (2 * top + 7 * (1 << 16)) % (14 * (1 << 16)) == 0
    s = torch.where(tie & (s % 2 == 1), s - 1, s)                                  # ... even where in the middle
    unit = (s * (1 << 16)).clamp_min(1)[..., None]
    q = (2 * g.abs() + unit) // (2 * unit)
    q = torch.where(((2 * g.abs() + unit) % (2 * unit) == 0) & (q % 2 == 1), q - 1, q).clamp(max=7) * g.sign()
    return torch.where((s > 0)[..., None], q, torch.zeros_like(q)), s


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_lowest_scales(dtype):
    from flashbfp_b200 import kv4
    g = torch.Generator().manual_seed(3)
    tops = list(range(1, 80)) + [8, 9, 10, 16, 17, 24, 31, 38, 45, 52]
    n = len(tops)
    x = torch.zeros(n, 1, 64, dtype=torch.float64)
    for i, t in enumerate(tops):
        fine = (torch.rand(64, generator=g, dtype=torch.float64) * 2 - 1) * t
        x[i, 0] = fine.round() if dtype == torch.bfloat16 else (fine * (1 << 16)).round() / (1 << 16)
        for b in (0, 32):                              # the group's largest beside others, of either sign
            x[i, 0, b + 3 * (i % 10)] = t if (i + b // 32) % 2 else -t
            x[i, 0, b + 3 * (i % 10) + 1] = -1.0
    x = torch.ldexp(x, torch.tensor(-133)).to(dtype)
    q, s = held(x)
    cache = kv4.empty_cache(1, 1, n, 64, DEV)
    kv4.kv4_write(cache, x.to(DEV), -x.to(DEV), ints([0]), starts=ints([0, n]))
    kv4.check_device_errors()
    for values, scales, sign in ((cache.k_values, cache.k_scales, 1), (cache.v_values, cache.v_scales, -1)):
        got = torch.stack((values & 15, values >> 4), -1).flatten(-2).cpu().long()[0, 0, :n] - 8
        want = sign * q[:, 0].flatten(-2)
        assert torch.equal(scales.cpu().view(torch.int16)[0, 0, :n].long(), s[:, 0])
        assert torch.equal(got, want), (got - want).abs().max()
        assert got.abs().max() == 7
    back = kv4.kv4_read(cache, ints([0]), ints([0, n]), rows=n, dtype=torch.float32)[0]
    want = torch.ldexp((q * s[..., None]).flatten(-2).double(), torch.tensor(-133)).float()
    assert torch.equal(back.cpu(), want)


def test_append_lowest_scales():
    """The values of a fused row, which append leaves as they are."""
    from flashbfp_b200 import kv4
    d = 32
    x = torch.zeros(8, 3, d, dtype=torch.float64)
    for i in range(8):
        x[i, 2, :4] = torch.tensor([8 + 3 * i, -1.0, -(8 + 3 * i), 2.0])
    x = torch.ldexp(x, torch.tensor(-133))
    x[:, :2] = 1.0
    x = x.bfloat16()
    q, s = held(x[:, 2:])
    cache = kv4.empty_cache(8, 1, 32, d, DEV)
    ang = torch.ones(32, d, dtype=torch.bfloat16, device=DEV)
    w = torch.zeros(d, dtype=torch.bfloat16, device=DEV)
    out = torch.empty(8, 1, d, dtype=torch.bfloat16, device=DEV)
    kv4.kv4_append(cache, x.flatten(1).to(DEV), w, w, 1e-6, ang, torch.zeros_like(ang), ints([0] * 8), out)
    got = torch.stack((cache.v_values & 15, cache.v_values >> 4), -1).flatten(-2).cpu().long()[:, 0, 0] - 8
    assert torch.equal(got, q[:, 0, 0])
    assert torch.equal(cache.v_scales.cpu().view(torch.int16)[:, 0, 0, 0].long(), s[:, 0, 0])
