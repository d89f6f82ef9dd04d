"""Split products whose last tile has CTAs without features of their own, queued back to back: each next
kernel's CTAs take over the shared memory that the last one's leave. Integer operands, so every
sum is exact and every result is compared for equality."""
import pytest
import torch

from test_gpu_fp8 import DEV, integer_rows

pytestmark = pytest.mark.gpu

SHAPES = [(90, 200, 8200), (70, 300, 4100), (100, 2000, 16000), (128, 4160, 4096), (333, 1999, 4090), (65, 33, 2000),
          (200, 97, 5000), (256, 160, 9000)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_chains_of_split_products(dtype):
    from flashbfp_b200 import fp8
    ops, want, outs = [], [], []
    for m, n, k in SHAPES:
        x, xd = integer_rows(m, k, m + n, lim=2)
        w, wd = integer_rows(n, k, n + k, lim=2)
        ops.append((x, w))
        want.append((xd @ wd.t()).to(dtype))
        assert want[-1].abs().max() < 2.0 ** 22
        outs.append([torch.zeros(m, n, device=DEV, dtype=dtype) for _ in range(6)])
    torch.cuda.synchronize()
    for rep in range(6):
        for i in range(len(SHAPES)):
            for _ in range(5):
                fp8.fp8_linear(*ops[i], out=outs[i][rep])
            j = (i + rep + 1) % len(SHAPES)
            fp8.fp8_linear(*ops[j], out=outs[j][rep])
    fp8.check_device_errors(DEV)
    for i, y in enumerate(want):
        for o in outs[i]:
            assert torch.equal(o, y), SHAPES[i]


def test_chains_of_products_on_cta_pairs():
    """One tile a pair and many, queued behind one another in turn."""
    from flashbfp_b200 import fp8
    shapes = [(257, 1100, 900), (512, 768, 2048), (1024, 2048, 1280), (2100, 1240, 700), (2048, 4096, 512),
              (3000, 5000, 256)]
    ops, want, outs = [], [], []
    for m, n, k in shapes:
        x, xd = integer_rows(m, k, m + n)
        w, wd = integer_rows(n, k, n + k)
        ops.append((x, w))
        want.append((xd @ wd.t()).float())
        outs.append([torch.zeros(m, n, device=DEV) for _ in range(2)])
    torch.cuda.synchronize()
    for rep in range(10):
        for i in range(len(shapes)):
            fp8.fp8_linear(*ops[i], out=outs[i][rep % 2])
            j = (i * 5 + rep) % len(shapes)
            fp8.fp8_linear(*ops[j], out=outs[j][rep % 2])
    fp8.check_device_errors(DEV)
    for i, y in enumerate(want):
        for o in outs[i]:
            assert torch.equal(o, y), shapes[i]
