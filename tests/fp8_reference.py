"""The block-scaled 8-bit operators in fp64, straight from their definitions (used by the tests)."""
import math

import torch


def quantise(x):
    """fp64 rows -> (values on the e4m3 grid, scale codes [m, blocks]); blocks with an infinity or
    a NaN give NaN values and code 255."""
    x = x.double()
    m, k = x.shape
    nb = -(-k // 128)
    p = torch.nn.functional.pad(x, (0, nb * 128 - k)).view(m, nb, 128)
    amax = p.abs().amax(dim=2)                         # NaN propagates
    bad = ~torch.isfinite(amax)
    a = torch.where(bad, torch.ones_like(amax), amax)
    e = torch.ceil(torch.log2(a / 448.0))
    # log2 may round across an integer: settle by comparison
    e = torch.where(a > 448.0 * torch.exp2(e), e + 1, e)
    e = torch.where(a <= 448.0 * torch.exp2(e - 1), e - 1, e)
    e = torch.where(a == 0, torch.full_like(e, -127), e).clamp(min=-127)
    v = p * torch.exp2(-e)[:, :, None]
    mag = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -40))).clamp(min=-6)
    mag = torch.where(v.abs() >= torch.exp2(mag + 1), mag + 1, mag)
    step = torch.exp2(mag - 3)
    q = (torch.round(v / step) * step).clamp(-448.0, 448.0)
    q = torch.where(bad[:, :, None], torch.full_like(q, math.nan), q)
    codes = torch.where(bad, torch.full_like(e, 255), e + 127).int()
    return q.view(m, nb * 128)[:, :k], codes


def norm(x, w, eps):
    x = x.double()
    return x * torch.rsqrt(x.square().mean(dim=1, keepdim=True) + eps) * (1.0 + w.double())


def geglu(gu):
    g, u = gu.double().chunk(2, dim=1)
    return 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3))) * u


def codes_of(rows):
    """Scale codes [m, blocks] of an Fp8Rows."""
    m, k = rows.values.shape
    t = rows.scales.view(torch.uint8)
    return t.permute(0, 3, 2, 1, 4).reshape(t.shape[0] * 128, -1)[:m, :-(-k // 128)].int()


def tiles_of(codes, device):
    """Scale tiles (float8_e8m0fnu) from codes [m, blocks], zero behind the last row and block."""
    m, b = codes.shape
    full = torch.zeros(-(-m // 128) * 128, -(-b // 4) * 4, dtype=torch.uint8, device=device)
    full[:m, :b] = codes.to(device=device, dtype=torch.uint8)
    t = full.view(-1, 4, 32, full.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous()
    return t.view(torch.float8_e8m0fnu)
