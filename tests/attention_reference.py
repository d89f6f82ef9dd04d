"""Definitions in 64 bits for the tests of the prompts' attention and of the 4-bit cache, and the bounds
that its roundings allow.

``attend`` gives the result o and, for each value, how far rounding may move it:
  u |o|                     the result's own rounding, u = eps / 2 of its type
  + w sum_j p_j |v_j|       the weights: each is off by at most a factor 1 +- w, with
                            w = u_w + 2 e_s + 2^-19,
u_w the rounding of a weight to the type that enters the product with v, e_s the largest error of a
score: a dot product of D terms in fp32 is off by at most (D + 4) 2^-24 sum|q_d k_d| (times scaling), which
moves the weight and the sum that it is divided by by that factor each; 2^-19 covers exp2 (2 last
places), the products by log2(e) and the fp32 sums of the weights and of their products.
"""
import math

import torch


def bf16_nearest(x):
    """fp64 -> the nearest bf16 (ties to even), as fp64; subnormals too."""
    m, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 8).clamp(min=-133))
    return torch.round(x / step) * step


def stored(x):
    """Rows [..., D] of any float type: (bytes, scales as fp64, values as fp64) of the 4-bit cache."""
    d = x.shape[-1]
    g = -(-d // 32)
    z = torch.zeros(*x.shape[:-1], g * 32, dtype=torch.float64)
    z[..., :d] = x.double().cpu()
    z = z.view(*x.shape[:-1], g, 32)
    top = z.abs().amax(-1)
    bad = ~torch.isfinite(z).all(-1)
    s = bf16_nearest(torch.where(bad, torch.zeros_like(top), top) / 7.0)
    n = torch.where((s > 0)[..., None] & ~bad[..., None], torch.round(z / torch.where(s > 0, s, torch.ones_like(s))[..., None]),
                    torch.zeros_like(z))
    s = torch.where(bad, torch.full_like(s, math.nan), s)
    vals = (n * s[..., None]).flatten(-2)[..., :d]
    c = (n + 8).to(torch.uint8).flatten(-2)
    return c[..., 0::2] + 16 * c[..., 1::2], s, vals


def attend(q, k, v, seen, scaling, out_dtype, weight_u, step=0.0):
    """q [heads, rows, D], k and v [heads, keys, D] in fp64, seen [rows, keys] -> (o, bound). ``step``: half the
    smallest step of a weight times the largest value that it meets, relative to the row's largest weight
    (the sum that results are divided by is at least that): small weights are off by that much each."""
    s = q @ k.transpose(1, 2) * scaling
    e_s = float(((q.abs() @ k.abs().transpose(1, 2)) * abs(scaling) * seen).max()) * (q.shape[-1] + 4) * 2.0 ** -24 \
        if seen.any() else 0.0
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    v = torch.where(seen.any(0)[None, :, None], v, torch.zeros_like(v))          # what nobody sees may be NaN
    o = p @ v
    u = torch.finfo(out_dtype).eps / 2
    w = weight_u + 2 * e_s + 2.0 ** -19
    bound = u * o.abs() + (1 + u) * w * (p @ v.abs())
    bound = bound + step * seen.sum(-1)[None, :, None]
    if out_dtype == torch.float16:
        bound = bound + 2.0 ** -25                                                # half a subnormal step of the result
    return o, bound + 1e-30


def packed(q, k, v, starts, kv_starts, window, scaling, weight_u):
    """Attention of packed prompts: q [T, H, D], k, v [N, Hkv, D] (any device) -> (o, bound) [T, H, D] on
    the CPU in fp64; rows of no sequence are NaN in o."""
    t, h, d = q.shape
    grp = h // k.shape[1]
    o = torch.full((t, h, d), math.nan, dtype=torch.float64)
    bound = torch.zeros(t, h, d, dtype=torch.float64)
    dev = q.device
    for b in range(len(starts) - 1):
        q0, q1, k0, k1 = starts[b], starts[b + 1], kv_starts[b], kv_starts[b + 1]
        n, c = q1 - q0, k1 - k0
        if n == 0:
            continue
        at = torch.arange(c - n, c, device=dev)[:, None]
        j = torch.arange(c, device=dev)[None, :]
        seen = j <= at
        if window:
            seen = seen & (j > at - window)
        if c == 0:
            o[q0:q1] = 0
            continue
        qq = q[q0:q1].double().transpose(0, 1)
        kk, vv = (x[k0:k1].double().transpose(0, 1).repeat_interleave(grp, 0) for x in (k, v))
        # fp16 weights are 2^6 times as large as the row's largest makes them: half a step is 2^-25 / 2^6
        step = 2.0 ** -31 * float(vv.abs().max()) if q.dtype == torch.float16 and torch.isfinite(vv).all() else 0.0
        oo, bb = attend(qq, kk, vv, seen, scaling, q.dtype, weight_u, step)
        o[q0:q1], bound[q0:q1] = oo.transpose(0, 1).cpu(), bb.transpose(0, 1).cpu()
    return o, bound


def cached(q, cache, pos, window, scaling, weight_u):
    """Attention over a 4-bit cache: q [S, rows, H, D] -> (o, bound) on the CPU in fp64."""
    s, rows, h, d = q.shape
    hkv = cache.k_values.shape[1]
    grp = h // hkv

    def held(values, scales):
        n = torch.stack((values & 15, values >> 4), -1).flatten(-2).double() - 8
        return (n * scales.double().repeat_interleave(32, -1))[..., :d]

    o = torch.zeros(s, rows, h, d, dtype=torch.float64)
    bound = torch.zeros_like(o)
    positions = cache.k_values.shape[2]
    for b in range(s):
        inside = [i for i in range(rows) if 0 <= pos[b] + i < positions]
        if not inside:
            continue
        n = pos[b] + inside[-1] + 1
        lo = max(0, pos[b] + inside[0] + 1 - window) if window else 0
        k = held(cache.k_values[b, :, lo:n], cache.k_scales[b, :, lo:n]).repeat_interleave(grp, 0)
        v = held(cache.v_values[b, :, lo:n], cache.v_scales[b, :, lo:n]).repeat_interleave(grp, 0)
        at = torch.tensor([pos[b] + i for i in inside], device=q.device)[:, None]
        j = torch.arange(lo, n, device=q.device)[None, :]
        seen = j <= at
        if window:
            seen = seen & (j > at - window)
        # weights times scales are fp16, 2^8 times as large as the largest scale's power of two makes them:
        # half a step is 2^-25 / 2^8 of it, times |n| <= 7
        sc = cache.v_scales[b, :, lo:n].float()
        step = 7 * 2.0 ** -33 * float(torch.where(torch.isfinite(sc), sc, torch.zeros_like(sc)).max())
        oo, bb = attend(q[b, inside].double().transpose(0, 1), k, v, seen, scaling, q.dtype, weight_u, step)
        o[b, inside], bound[b, inside] = oo.transpose(0, 1).cpu(), bb.transpose(0, 1).cpu()
    return o, bound


def starts_of(lens):
    s = [0]
    for n in lens:
        s.append(s[-1] + n)
    return s
