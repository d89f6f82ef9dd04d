"""The 8-bit operators give no gradients: what they write in place is refused where a gradient would be
lost, and counts as modified for tensors that autograd has saved."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rows(m=4, k=64):
    return torch.randn(m, k, device=DEV)


def test_written_tensors_count_as_modified():
    from flashbfp_b200 import fp8
    w, x, res = torch.zeros(64, device=DEV), rows(), rows()
    v = res._version
    fp8.rmsnorm_fp8(x, w, 1e-6)
    assert res._version == v
    fp8.rmsnorm_fp8(x, w, 1e-6, residual=res)
    assert res._version == v + 1
    big = rows(8, 200)
    v = big._version
    fp8.rmsnorm_fp8(x, w, 1e-6, residual=big[2:6, 3:67], post_weight=w)   # a view counts for its base
    assert big._version == v + 1
    assert x._version == 0 and w._version == 0
    out = fp8.empty_rows(4, 64, DEV)
    for call in (lambda: fp8.quantize_fp8(x, out=out), lambda: fp8.rmsnorm_fp8(x, w, 1e-6, out=out),
                 lambda: fp8.geglu_fp8(rows(4, 128), out=out)):
        a, b = out.values._version, out.scales._version
        call()
        assert (out.values._version, out.scales._version) == (a + 1, b + 1)
    y = rows(4, 4)
    v = y._version
    fp8.fp8_linear(out, out, out=y)
    assert y._version == v + 1


def test_backward_sees_that_a_saved_residual_was_replaced():
    from flashbfp_b200 import fp8
    h, p = rows(), torch.ones(64, device=DEV, requires_grad=True)
    loss = (h * p).sum()                                   # saves h
    fp8.rmsnorm_fp8(rows(), torch.zeros(64, device=DEV), 1e-6, residual=h)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_tensors_that_require_a_gradient():
    from flashbfp_b200 import fp8
    w, x = torch.zeros(64, device=DEV), rows()
    leaf = rows().requires_grad_()
    kept = leaf.detach().clone()
    for res in (leaf, leaf[1:3], leaf * 1.0):
        with pytest.raises(RuntimeError, match="residual is written in place and requires a gradient"):
            fp8.rmsnorm_fp8(x[:res.shape[0]], w, 1e-6, residual=res)
    r = fp8.quantize_fp8(leaf)                             # read only: results without a gradient
    y = torch.zeros(4, 4, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="out is written in place and requires a gradient"):
        fp8.fp8_linear(r, r, out=y)
    assert torch.equal(leaf.detach(), kept) and not y.any()
    assert not fp8.fp8_linear(r, r, leaf[0, :4]).requires_grad
    with torch.no_grad():
        fp8.rmsnorm_fp8(x, w, 1e-6, residual=leaf)
        fp8.fp8_linear(r, r, out=y)
    assert torch.equal(leaf.detach(), kept + x) and bool(y.any())
    with torch.inference_mode():
        res = rows()
        before = res.clone()
        fp8.rmsnorm_fp8(rows(), w, 1e-6, residual=res)
    fp8.rmsnorm_fp8(x, w, 1e-6, residual=res)              # an inference tensor keeps no version
    assert not torch.equal(res, before)
