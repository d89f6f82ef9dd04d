"""GeGLU to 8 bits where the exponential of a gate leaves fp32: blocks that hold nothing but very
negative gates, so that no larger value of the block sets the scale and hides them.

For a gate g below about -10.3, gelu_tanh(g) = g / (1 + 2^t) is below 2^-137, half of the smallest
8-bit step (2^-9 of the smallest scale 2^-127, halved): value 0 and scale code 0 for |up| <= 1. The
definition's exponent is t = 2 log2(e) sqrt(2 / pi) (g + 0.044715 g^3), negated.
"""
import math

import pytest
import torch

import fp8_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("k", [128, 640, 643])                # whole lanes, and rows that start anywhere
def test_blocks_of_very_negative_gates(dtype, k):
    from flashbfp_b200 import fp8
    dt = DTYPES[dtype]
    gates = [g for g in (-11.0, -20.0, -30.0, -1e3, -1e4, -65504.0, -1e10, -1e30, -1e38, torch.finfo(dt).min)
             if g >= torch.finfo(dt).min]
    gu = torch.zeros(len(gates) * 2, 2 * k, device=DEV, dtype=dt)
    for i, g in enumerate(gates):
        gu[2 * i: 2 * i + 2, :k] = g
        gu[2 * i, k:], gu[2 * i + 1, k:] = 1.0, -0.5
    r = fp8.geglu_fp8(gu)
    assert not r.values.float().any()
    assert not ref.codes_of(r).any()


def test_masked_gates_do_not_scale_with_up():
    """The lowest fp32 value as a gate stays 0 for large `up` too."""
    from flashbfp_b200 import fp8
    gu = torch.full((2, 512), torch.finfo(torch.float32).min, device=DEV)
    gu[0, 256:], gu[1, 256:] = 1e30, -1e4
    r = fp8.geglu_fp8(gu)
    assert not r.values.float().any() and not ref.codes_of(r).any()


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_gates_where_the_exponential_underflows(dtype):
    """Gates between -8 and -10.6, each with a block of its own, against the definition in fp64. With
    t rounded 6 times (a relative error that counts |t| times in the result), the exponential 2 ulp
    off and 6 more roundings, the relative error before the quantisation is (6 |t| + 10) 2^-24; what
    is below 2^-126 of the exponential or of its reciprocal flushes to 0, which counts |g| times,
    and two products may flush likewise."""
    from flashbfp_b200 import fp8
    dt = DTYPES[dtype]
    g = torch.linspace(-8.0, -10.6, 53, device=DEV).to(dt)
    gu = torch.cat([g[:, None].expand(-1, 128), torch.ones(53, 128, device=DEV, dtype=dt)], dim=1).contiguous()
    gd = g.double()
    t = -2.0 * math.sqrt(2.0 / math.pi) * (gd + 0.044715 * gd ** 3)
    y = gd / (1.0 + torch.exp(t))
    d = y.abs() * (6 * t.abs() + 10) * 2.0 ** -24 + (gd.abs() + 2) * 2.0 ** -126
    r = fp8.geglu_fp8(gu)
    codes = ref.codes_of(r)[:, 0]
    s = torch.exp2(codes.double() - 127)
    assert bool((y.abs() - d <= 448.0 * s).all())
    assert bool(((y.abs() + d > 224.0 * s) | (codes == 0)).all())
    got = r.values.double() * s[:, None]
    bound = (y.abs() + d) * 2.0 ** -4 + 2.0 ** -10 * s + d
    assert bool(((got - y[:, None]).abs() <= bound[:, None]).all())


def test_infinite_and_nan_gates():
    """+inf * up is infinite and -inf * 0 NaN: their blocks are NaN, all others as they are."""
    from flashbfp_b200 import fp8
    for dt in DTYPES.values():
        gu = torch.ones(3, 1024, device=DEV, dtype=dt)
        gu[0, 5], gu[1, 130], gu[2, 260] = float("inf"), float("-inf"), float("nan")
        r = fp8.geglu_fp8(gu)
        codes = ref.codes_of(r)
        for row in range(3):
            for b in range(4):
                assert (int(codes[row, b]) == 255) == (row == b)
        assert bool(torch.isnan(r.dequantize()[0, :128]).all())
