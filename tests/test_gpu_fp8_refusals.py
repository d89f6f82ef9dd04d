"""Calls of the block-scaled 8-bit path that are refused on the host (nothing is launched)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_row_refusals():
    from flashbfp_b200 import fp8
    x = torch.zeros(4, 64, device=DEV)
    w = torch.zeros(64, device=DEV)
    with pytest.raises(ValueError, match="two dimensions"):
        fp8.quantize_fp8(x[0])
    with pytest.raises(ValueError, match="contiguous rows"):
        fp8.quantize_fp8(x.t())
    with pytest.raises(ValueError, match="at least one value"):
        fp8.quantize_fp8(x[:, :0])
    with pytest.raises(NotImplementedError):
        fp8.quantize_fp8(x.double())
    with pytest.raises(ValueError, match="as many gate as up"):
        fp8.geglu_fp8(x[:, :63])
    with pytest.raises(ValueError, match="weight"):
        fp8.rmsnorm_fp8(x, w[:63], 1e-6)
    with pytest.raises(ValueError, match="weight"):
        fp8.rmsnorm_fp8(x, w.half(), 1e-6)
    with pytest.raises(ValueError, match="needs the residual"):
        fp8.rmsnorm_fp8(x, w, 1e-6, post_weight=w)
    with pytest.raises(ValueError, match="residual"):
        fp8.rmsnorm_fp8(x, w, 1e-6, residual=x[:3].clone())
    with pytest.raises(ValueError, match="overlap"):
        fp8.rmsnorm_fp8(x, w, 1e-6, residual=x[:1].clone().expand(4, -1))
    with pytest.raises(ValueError, match="at most 32768"):
        fp8.rmsnorm_fp8(torch.zeros(1, 32769, device=DEV), torch.zeros(32769, device=DEV), 1e-6)
    for out in (fp8.empty_rows(4, 80, DEV), fp8.empty_rows(3, 64, DEV)):
        with pytest.raises(ValueError, match="shape"):
            fp8.quantize_fp8(x, out=out)
    good = fp8.empty_rows(4, 64, DEV)
    with pytest.raises(ValueError, match="scales"):
        fp8.quantize_fp8(x, out=fp8.Fp8Rows(good.values, good.scales.reshape(-1)))
    with pytest.raises(ValueError, match="float8"):
        fp8.quantize_fp8(x, out=fp8.Fp8Rows(good.values.view(torch.uint8), good.scales))


def test_linear_refusals():
    from flashbfp_b200 import fp8
    x, w = fp8.quantize_fp8(torch.ones(4, 64, device=DEV)), fp8.quantize_fp8(torch.ones(8, 64, device=DEV))
    k80 = fp8.quantize_fp8(torch.ones(8, 80, device=DEV))
    with pytest.raises(ValueError, match="shape"):
        fp8.fp8_linear(x, k80)
    with pytest.raises(ValueError, match="bias"):
        fp8.fp8_linear(x, w, torch.zeros(7, device=DEV))
    with pytest.raises(NotImplementedError):
        fp8.fp8_linear(x, w, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="out"):
        fp8.fp8_linear(x, w, out=torch.zeros(4, 9, device=DEV))
    with pytest.raises(ValueError, match="dtype"):
        fp8.fp8_linear(x, w, out=torch.zeros(4, 8, device=DEV), out_dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="overlap"):
        fp8.fp8_linear(x, w, out=torch.zeros(1, 8, device=DEV).expand(4, -1))
    tight = torch.zeros(4 * 72, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn).view(4, 72)[:, :64]
    with pytest.raises(ValueError, match="multiple of 16 bytes apart"):
        fp8.fp8_linear(fp8.Fp8Rows(tight, x.scales), w)
    off = torch.zeros(4, 80, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)[:, 8:72]
    with pytest.raises(ValueError, match="aligned"):
        fp8.fp8_linear(fp8.Fp8Rows(off, x.scales), w)
    y = fp8.fp8_linear(x, w, out_dtype=torch.float32)           # and the call still works
    assert bool((y == 64).all())
