"""The tcgen05 GEMV with its weights out of L2, where loads land late and out of order: what it gives is what it
gives with the weights in L2. Both sum the same terms in fp32; CTAs add their parts of a row (six at most)
in any order, so that two calls differ by 2 x 6 roundings of at most sum|w x|."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,m", [((3840, 15360), 1), ((3840, 15360), 16), ((8192, 3840), 4), ((4096, 4096), 1)])
def test_cold_weights_give_what_warm_ones_give(shape, m):
    from flashbfp_b200 import OABFCompressor, workloads
    from flashbfp_b200.linear import check_device_errors, packed_linear
    from flashbfp_b200.packed import from_compressed
    n, k = shape
    dev = torch.device("cuda", 0)
    W = workloads.decode_weight(n, k, seed=5, device=dev)
    dp, sp = OABFCompressor().compress_matrix_device(W)
    pw = from_compressed(dp, sp, dev)
    X = workloads.activations(m, k, seed=6, device=dev)
    Y = torch.empty(m, n, dtype=torch.float32, device=dev)
    for _ in range(2):
        packed_linear(X, pw, None, torch.float32, out=Y)
    warm = Y.clone()
    # the stored weights differ from W by less than their blocks' steps: twice sum|W x| is above their sum
    bound = 12 * 2.0 ** -24 * 2 * (X.float().abs() @ W.float().abs().t())
    flush = torch.empty(1 << 29, dtype=torch.uint8, device=dev)          # four times L2
    for i in range(60):
        flush.fill_(i)
        Y.zero_()
        packed_linear(X, pw, None, torch.float32, out=Y)
        off = (Y - warm).abs()
        assert bool((off <= bound).all()), (i, (off / bound).max().item())
    check_device_errors()
