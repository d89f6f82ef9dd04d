"""The block-scaled 8-bit linear path (flashbfp_b200/fp8.py) against its definition in fp64.

Quantisation of given values is one exact scaling and one rounding, so its bytes are compared for
equality. A product of small integers with power-of-two scales has exact fp32 sums (below 2^24
units), so its result is compared for equality too, at every shape. RMSNorm and GeGLU compute in
fp32 before they quantise: with d their relative error (derived at each test), a value is within
half a step of e4m3 (2^-4 relative, 2^-10 of the scale below the normal range) plus d.
"""
import pytest
import torch

import fp8_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
DEV = "cuda:0"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def same(a, b):
    """Equality with NaN equal to NaN."""
    return bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


def pad_bytes_are_zero(rows):
    m, k = rows.values.shape
    t = rows.scales.view(torch.uint8)
    full = t.permute(0, 3, 2, 1, 4).reshape(t.shape[0] * 128, -1)
    return not full[m:].any() and not full[:, -(-k // 128):].any()


def spread(m, k, dt, seed):
    """Rows whose blocks differ by many binades, some of them zero."""
    g = gen(seed)
    x = torch.randn(m, k, generator=g, device=DEV)
    e = torch.randint(-12, 13, (m, -(-k // 128)), generator=g, device=DEV).float()
    x = x * torch.exp2(e).repeat_interleave(128, dim=1)[:, :k]
    dead = torch.rand(m, -(-k // 128), generator=g, device=DEV) < 0.05
    x = x.masked_fill(dead.repeat_interleave(128, dim=1)[:, :k], 0.0)
    return x.to(dt)


# ---------------------------------------------------------------------------- quantise
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("m,k", [(1, 1), (1, 16), (1, 3840), (2, 127), (3, 128), (5, 129), (7, 511), (31, 512),
                                 (33, 513), (127, 1000), (128, 640), (129, 4096), (300, 2049), (1000, 80)])
def test_quantize_is_exact(m, k, dtype):
    from flashbfp_b200 import fp8
    x = spread(m, k, DTYPES[dtype], m * 7919 + k)
    r = fp8.quantize_fp8(x)
    q, codes = ref.quantise(x)
    assert torch.equal(ref.codes_of(r), codes)
    assert torch.equal(r.values.double(), q)
    assert pad_bytes_are_zero(r)
    s = r.scale_matrix().double().repeat_interleave(128, dim=1)[:, :k]
    assert torch.equal(r.dequantize(torch.float64), q * s)


def test_quantize_edges():
    """Block maxima around 448 * 2^e and at the ends of fp32, halfway values, infinities and NaN."""
    from flashbfp_b200 import fp8
    x = torch.zeros(20, 256, device=DEV)
    for i, e in enumerate((-130, -126, -20, 0, 1, 100, 118)):
        x[i, 0] = 448.0 * 2.0 ** e                            # exactly the largest value
        x[i, 128] = torch.nextafter(torch.tensor(448.0 * 2.0 ** e), torch.tensor(float("inf")))
    x[7, 0], x[7, 128] = 3.4028234663852886e38, 1e-45          # the largest and the smallest fp32
    x[8, :128] = torch.arange(128, device=DEV) / 16.0          # many halfway values of the grid
    x[8, 128:] = -torch.arange(128, device=DEV) * 2.0 ** -10
    x[8, 128] = 448.0
    x[9, 5], x[10, 200], x[11, 3] = float("inf"), float("-inf"), float("nan")
    x[12, 3], x[12, 4] = float("nan"), float("inf")
    r = fp8.quantize_fp8(x)
    q, codes = ref.quantise(x)
    assert torch.equal(ref.codes_of(r), codes)
    assert same(r.values.double(), q)
    assert int(codes[9, 0]) == 255 and int(codes[9, 1]) == 0 and int(codes[10, 1]) == 255


def test_quantize_strides_and_out():
    from flashbfp_b200 import fp8
    big = spread(40, 1000, torch.bfloat16, 3)
    for view in (big[:, 3:803], big[::3, :640], big[5:6, 1:130], big[:1].expand(9, -1)):
        r = fp8.quantize_fp8(view)
        q, codes = ref.quantise(view)
        assert torch.equal(r.values.double(), q) and torch.equal(ref.codes_of(r), codes)
    # values with rows further apart than they are long: the bytes between stay as they were
    store = torch.full((8, 1024), 7, dtype=torch.uint8, device=DEV)
    v = store.view(torch.float8_e4m3fn)[:, 16:16 + 600]
    out = fp8.Fp8Rows(v, fp8.empty_rows(8, 600, DEV).scales)
    got = fp8.quantize_fp8(big[:8, :600], out=out)
    assert got is out
    assert torch.equal(v.double(), ref.quantise(big[:8, :600])[0])
    assert bool((store[:, :16] == 7).all()) and bool((store[:, 616:] == 7).all())
    # one column (any stride between columns) and no rows at all
    assert torch.equal(fp8.quantize_fp8(big[:, 4:5]).values.double(), ref.quantise(big[:, 4:5])[0])
    assert fp8.quantize_fp8(big[:0]).values.shape == (0, 1000)


def check_quantised(r, y, d):
    """r against exact values y (fp64), computed with absolute error at most d (a tensor) before
    the quantisation."""
    m, k = y.shape
    nb = -(-k // 128)
    codes = ref.codes_of(r)

    def block_max(t):
        return torch.nn.functional.pad(t.abs(), (0, nb * 128 - k)).view(m, nb, 128).amax(dim=2)

    # the scale is right for some block maximum within the error
    amax, da = block_max(y), block_max(d)
    s = torch.exp2(codes.double() - 127)
    assert bool((amax - da <= 448.0 * s).all())
    assert bool(((amax + da > 448.0 * s / 2) | (codes == 0)).all())
    full = s.repeat_interleave(128, dim=1)[:, :k]
    err = (r.values.double() * full - y).abs()
    bound = (y.abs() + d) * 2.0 ** -4 + 2.0 ** -10 * full + d
    assert bool((err <= bound).all()), float((err - bound).max())
    assert pad_bytes_are_zero(r)
    # and nearly every value is the correctly rounded one
    q, c = ref.quantise(y)
    off = (q * torch.exp2(c.double() - 127).repeat_interleave(128, dim=1)[:, :k] != r.values.double() * full)
    assert off.double().mean().item() <= 1e-3


# ---------------------------------------------------------------------------- RMSNorm
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("mode", ["plain", "add", "post"])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 3840), (2, 16), (3, 77), (5, 513), (130, 256), (17, 4090), (4, 8192),
                                 (3, 16384), (2, 16400), (2, 32768), (3, 8199), (2, 20001), (1500, 48), (700, 1040)])
def test_rmsnorm(m, k, mode, dtype):
    """Relative error of the fp32 part: a mean of k squares (each thread sums 16 or 32, then a tree
    and at most 32 warp sums: at most 96 roundings, halved by the root), rsqrt (2 ulp), at most
    four products: within 64 * 2^-24 per norm. After an addition it counts relative to the
    addends."""
    from flashbfp_b200 import fp8
    dt = DTYPES[dtype]
    g = gen(m * 31 + k)
    x = (torch.randn(m, k, generator=g, device=DEV) * 3).to(dt)
    w = (0.3 * torch.randn(k, generator=g, device=DEV)).to(dt)
    res = torch.randn(m, k, generator=g, device=DEV).to(dt) if mode != "plain" else None
    wp = (0.3 * torch.randn(k, generator=g, device=DEV)).to(dt) if mode == "post" else None
    eps, u = 1e-6, 64 * 2.0 ** -24
    first = ref.norm(x, wp, eps) if mode == "post" else x.double()
    h = first if res is None else first + res.double()
    y = ref.norm(h, w, eps)
    # error of h, then of its norm: the row's scale moves by at most the error's share of the row
    dh = torch.zeros_like(h)
    if mode == "post":
        dh = u * first.abs()
    if mode != "plain":
        dh = dh + 2.0 ** -24 * (h.abs() + dh)
    rel = dh.square().sum(dim=1, keepdim=True).sqrt() / h.square().sum(dim=1, keepdim=True).sqrt().clamp(min=1e-30)
    scale = torch.where(h == 0, torch.zeros_like(h), (y / torch.where(h == 0, torch.ones_like(h), h)).abs())
    d = u * y.abs() + dh * scale * 1.01 + 1.01 * rel * y.abs()
    kept = res.clone() if res is not None else None
    r = fp8.rmsnorm_fp8(x, w, eps, residual=res, post_weight=wp)
    check_quantised(r, y, d)
    if res is not None:
        tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
        assert bool(((res.double() - h).abs() <= HALF_STEP[dt] * (h.abs() + dh) + dh + tiny).all())
        assert not torch.equal(res, kept) or m * k == 1


def test_rmsnorm_zero_infinite_and_nan_rows():
    from flashbfp_b200 import fp8
    x = torch.randn(5, 700, device=DEV, generator=gen(1))
    w = torch.zeros(700, device=DEV)
    x[1] = 0
    x[2, 699] = float("nan")
    x[3, 5] = float("inf")
    r = fp8.rmsnorm_fp8(x, w, 1e-6)
    codes = ref.codes_of(r)
    assert not r.values[1].float().any() and not codes[1].any()       # zero row: zeros, smallest scale
    assert bool(torch.isnan(r.dequantize()[2]).all())                 # the mean is NaN: the whole row is
    # an infinity: the mean is infinite, every other value becomes 0 and its own block NaN
    assert bool(torch.isnan(r.dequantize()[3, :128]).all()) and not r.values[3, 128:].float().any()
    ok = fp8.rmsnorm_fp8(x[[0, 4]].contiguous(), w, 1e-6)             # other rows are untouched by them
    assert torch.equal(ok.values.float(), r.values[[0, 4]].float())


def test_rmsnorm_strided_rows_and_residual():
    from flashbfp_b200 import fp8
    g = gen(9)
    wide = torch.randn(6, 1501, device=DEV, generator=g).bfloat16()
    resw = torch.randn(6, 1303, device=DEV, generator=g).bfloat16()
    w = torch.randn(900, device=DEV, generator=g).bfloat16()
    for dt in (torch.bfloat16, torch.float32):
        wide, resw, w = wide.to(dt), resw.to(dt), w.to(dt)
        for c0, c1 in ((0, 4), (1, 4), (8, 16), (3, 7), (5, 2), (0, 13)):      # every start within 16 bytes
            for k in (900, 512, 511, 896, 5):
                x, r0 = wide[:, c0:c0 + k], resw.clone()
                res = r0[:, c1:c1 + k]
                a = fp8.rmsnorm_fp8(x, w[:k], 1e-5, residual=res)
                rc = resw[:, c1:c1 + k].contiguous()
                b = fp8.rmsnorm_fp8(x.contiguous(), w[:k].contiguous(), 1e-5, residual=rc)
                # the sums of squares have the same order: rows of any alignment have the same lanes
                assert torch.equal(a.values.float(), b.values.float()) and torch.equal(ref.codes_of(a), ref.codes_of(b))
                assert torch.equal(res, rc)
                assert torch.equal(r0[:, :c1], resw[:, :c1]) and torch.equal(r0[:, c1 + k:], resw[:, c1 + k:])


def test_rmsnorm_of_the_residual_itself():
    """x may be the residual: h = 2 x, in place; and one row given for all rows."""
    from flashbfp_b200 import fp8
    g = gen(4)
    w = torch.zeros(1024, device=DEV)
    x = torch.randn(600, 1024, device=DEV, generator=g)
    a, b = x.clone(), x.clone()
    r = fp8.rmsnorm_fp8(a, w, 1e-6, residual=a)
    q = fp8.rmsnorm_fp8(x, w, 1e-6, residual=b)
    assert torch.equal(a, 2 * x) and torch.equal(a, b)
    assert torch.equal(r.values.float(), q.values.float()) and torch.equal(ref.codes_of(r), ref.codes_of(q))
    one = fp8.rmsnorm_fp8(x[:1].expand(500, -1), w, 1e-6)
    assert torch.equal(one.dequantize(), fp8.rmsnorm_fp8(x[:1], w, 1e-6).dequantize().expand(500, -1))


# ---------------------------------------------------------------------------- GeGLU
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("m,k", [(1, 1), (1, 15360), (3, 130), (16, 512), (129, 1001)])
def test_geglu(m, k, dtype):
    """Relative error of the fp32 part: the exponent's argument t (|t| <= 2 sqrt(2/pi) (|g| +
    0.044715 |g|^3), 6 roundings) enters through exp, whose relative error is that of t times |t|
    plus 2 ulp; the sum, the quotient and the product add 4 more: (6 |t| + 8) 2^-24, with
    underflow where exp(-t) leaves fp32."""
    from flashbfp_b200 import fp8
    dt = DTYPES[dtype]
    g = gen(m * 17 + k)
    gu = (torch.randn(m, 2 * k, generator=g, device=DEV) * 2).to(dt)
    if k > 100:
        gu[0, :40] = torch.linspace(-14, 14, 40, device=DEV).to(dt)
    y = ref.geglu(gu)
    ga, up = gu.double().chunk(2, dim=1)
    # the definition by exp, which fp64 tanh loses for very negative gates
    t = 1.5957691216057308 * (ga + 0.044715 * ga ** 3)
    y = ga / (1.0 + torch.exp(-t)) * up
    d = y.abs() * (6 * t.abs() + 8) * 2.0 ** -24 + 1e-38 * (1 + up.abs())
    check_quantised(fp8.geglu_fp8(gu), y, d)


def test_geglu_large_gates():
    """Gates whose exponential overflows: 0 for negative ones, gate * up for positive ones."""
    from flashbfp_b200 import fp8
    gu = torch.zeros(1, 256, device=DEV)
    gu[0, :4] = torch.tensor([-1e4, -30.0, 30.0, 1e4], device=DEV)
    gu[0, 128:] = 1.0
    got = fp8.geglu_fp8(gu).dequantize()
    assert got[0, :2].tolist() == [0.0, 0.0]
    assert abs(got[0, 2].item() - 30.0) <= 30 / 16 + 32 and abs(got[0, 3].item() - 1e4) <= 1e4 / 16


# ---------------------------------------------------------------------------- the product
def integer_rows(m, k, seed, lim=3):
    """Rows of small integers (exact in e4m3) with scales 2^-1 .. 2^1 per block, as an operand and
    as fp64 values."""
    from flashbfp_b200 import fp8
    g = gen(seed)
    v = torch.randint(-lim, lim + 1, (m, k), generator=g, device=DEV).float()
    nb = -(-k // 128)
    codes = torch.randint(126, 129, (m, nb), generator=g, device=DEV).int()
    r = fp8.empty_rows(m, k, DEV)
    r.values.copy_(v)
    r = fp8.Fp8Rows(r.values, ref.tiles_of(codes, DEV))
    dense = v.double() * torch.exp2(codes.double() - 127).repeat_interleave(128, dim=1)[:, :k]
    return r, dense


SHAPES = [(1, 1, 1), (1, 128, 128), (1, 200, 3840), (2, 129, 127), (3, 1000, 129), (16, 256, 512), (17, 130, 640),
          (31, 512, 1030), (33, 384, 2000), (64, 300, 4096), (65, 129, 300), (100, 1024, 1024), (128, 128, 16),
          (129, 257, 1500), (200, 640, 384), (256, 512, 512), (257, 1100, 900), (333, 1999, 4090), (512, 768, 2048),
          (700, 513, 260), (1024, 2048, 1280), (1500, 300, 100), (90, 200, 8200), (128, 3840, 3000),
          (300, 1000, 8200), (130, 2000, 128), (2100, 1240, 700)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_of_integers_is_exact(m, n, k):
    from flashbfp_b200 import fp8
    x, xd = integer_rows(m, k, 3 * m + n)
    w, wd = integer_rows(n, k, 5 * n + k)
    want = xd @ wd.t()
    assert want.abs().max() < 2.0 ** 22                       # quarters: exact fp32 sums
    y = fp8.fp8_linear(x, w, out_dtype=torch.float32)
    fp8.check_device_errors(DEV)
    assert y.shape == (m, n) and torch.equal(y.double(), want)
    b = torch.randint(-50, 50, (n,), device=DEV, generator=gen(1)).float()
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        y = fp8.fp8_linear(x, w, b.to(dt), out_dtype=dt)
        assert torch.equal(y, (want + b.to(dt).double()).to(dt)), dt


@pytest.mark.parametrize("m,n,k", [(1, 8192, 3840), (16, 3840, 4096), (128, 3840, 15360), (512, 8192, 3840),
                                   (1000, 2048, 3840), (2048, 4096, 3840)])
def test_linear_of_real_values(m, n, k):
    """Real activations and weights at decoder sizes: fp32 out within k / 32 + 32 accumulation
    steps of 2^-23 of the sum of magnitudes, and within 2^-17 in relative L2 (the steps' errors
    are random signs: sqrt(k / 32 + 32) 2^-23 times the magnitudes' sum, itself below sqrt(k) of
    the result: at most 2^-23 * 23 * 2^-1 * sqrt(15360) < 2^-12; held to the tighter 2^-17)."""
    from flashbfp_b200 import fp8
    g = gen(m + n)
    x = fp8.quantize_fp8(torch.randn(m, k, generator=g, device=DEV) * torch.exp(torch.randn(m, 1, generator=g, device=DEV)))
    w = fp8.quantize_fp8(0.02 * torch.randn(n, k, generator=g, device=DEV))
    xd, wd = x.dequantize(torch.float64), w.dequantize(torch.float64)
    want, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
    y = fp8.fp8_linear(x, w, out_dtype=torch.float32).double()
    assert bool(((y - want).abs() <= (k / 32 + 32) * 2.0 ** -23 * mag).all())
    assert ((y - want).norm() / want.norm()).item() <= 2.0 ** -17
    yb = fp8.fp8_linear(x, w)
    assert yb.dtype == torch.bfloat16
    assert ((yb.double() - want).norm() / want.norm()).item() <= 2.0 ** -8
    again = fp8.fp8_linear(x, w)
    assert torch.equal(again, yb)                             # same bits every time
    fp8.check_device_errors(DEV)


def test_linear_nan_rows_stay_in_their_rows():
    from flashbfp_b200 import fp8
    for m in (5, 100, 300):
        x, xd = integer_rows(m, 640, 1)
        w, wd = integer_rows(200, 640, 2)
        codes = ref.codes_of(x).clone()
        codes[3, 2] = 255
        x = fp8.Fp8Rows(x.values, ref.tiles_of(codes, DEV))
        y = fp8.fp8_linear(x, w, out_dtype=torch.float32)
        want = xd @ wd.t()
        assert bool(torch.isnan(y[3]).all())
        keep = [i for i in range(m) if i != 3]
        assert torch.equal(y[keep].double(), want[keep])


def test_linear_strides_and_empty():
    from flashbfp_b200 import fp8
    x, xd = integer_rows(40, 700, 4)
    w, wd = integer_rows(150, 700, 5)
    want = xd @ wd.t()
    store = torch.full((40, 400), 9.0, device=DEV)
    for c0 in (0, 3, 200):
        store.fill_(9.0)
        out = fp8.fp8_linear(x, w, out=store[:, c0:c0 + 150])
        assert torch.equal(out.double(), want)
        assert bool((store[:, :c0] == 9).all()) and bool((store[:, c0 + 150:] == 9).all())
    # operands with rows further apart, and a column range that starts on a multiple of 16
    big = torch.zeros(40, 1600, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    big[:, 32:732].copy_(x.values)
    assert torch.equal(fp8.fp8_linear(fp8.Fp8Rows(big[:, 32:732], x.scales), w, out_dtype=torch.float32).double(), want)
    none = fp8.Fp8Rows(x.values[:0], fp8.empty_rows(0, 700, DEV).scales)
    assert fp8.fp8_linear(none, w).shape == (0, 150)


def test_offsets_past_32_bits():
    """More than 2^31 values in and out: the last rows, and the rows on either side of 2^31."""
    from flashbfp_b200 import fp8
    m, k = 33000, 65540                               # k: not a multiple of 16
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=DEV)
    rows = [0, 2 ** 31 // k - 1, 2 ** 31 // k, 2 ** 31 // k + 1, m - 1]
    x[rows] = torch.randn(len(rows), k, device=DEV, generator=gen(1)).bfloat16()
    r = fp8.quantize_fp8(x)
    q, codes = ref.quantise(x[rows])
    assert torch.equal(r.values[rows].double(), q)
    t = r.scales.view(torch.uint8)
    for i, row in enumerate(rows):
        got = t[row // 128, :, row % 32, row % 128 // 32].reshape(-1)[:codes.shape[1]].int()
        assert torch.equal(got, codes[i])
    assert not r.values[1:100].view(torch.uint8).any()
    del x, r, t
    n = 1_000_003
    xi, xd = integer_rows(2200, 128, 7)
    wi, wd = integer_rows(n, 128, 8)
    y = fp8.fp8_linear(xi, wi)
    for sl in (slice(0, 3), slice(2140, 2150), slice(2197, 2200)):
        assert torch.equal(y[sl], (xd[sl] @ wd.t()).to(torch.bfloat16))
    fp8.check_device_errors(DEV)


def test_first_calls_inside_a_capture():
    """Kernels whose first launch is captured (another output type and tile than any warm call's)."""
    from flashbfp_b200 import fp8
    x, xd = integer_rows(70, 4100, 1)
    w, wd = integer_rows(300, 4100, 2)
    fp8.fp8_linear(fp8.Fp8Rows(x.values[:1], x.scales), w)          # the error word exists
    y, z = torch.zeros(70, 300, device=DEV, dtype=torch.float16), torch.zeros(20, 300, device=DEV, dtype=torch.float16)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        fp8.fp8_linear(x, w, out=y)
        fp8.fp8_linear(fp8.Fp8Rows(x.values[:20], x.scales), w, out=z)
    graph.replay()
    want = (xd @ wd.t()).to(torch.float16)
    assert torch.equal(y, want) and torch.equal(z, want[:20])


def test_two_graphs_and_a_third_stream():
    """Two captured chains replayed at the same time as eager calls: nothing is shared between them."""
    from flashbfp_b200 import fp8
    g = gen(6)
    w = fp8.quantize_fp8(0.02 * torch.randn(640, 3000, generator=g, device=DEV))
    lnw = torch.zeros(3000, device=DEV, dtype=torch.bfloat16)
    xs = [torch.randn(m, 3000, generator=g, device=DEV).bfloat16() for m in (1, 90, 300)]

    def chain(x, out):
        return fp8.fp8_linear(fp8.rmsnorm_fp8(x, lnw, 1e-6), w, out=out)

    want = [chain(x, None) for x in xs]
    outs = [torch.zeros_like(y) for y in want]
    streams = [torch.cuda.Stream(DEV) for _ in xs]
    graphs = []
    torch.cuda.synchronize()
    for x, o in zip(xs[:2], outs):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            chain(x, o)
        graphs.append(gr)
    for _ in range(20):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        with torch.cuda.stream(streams[2]):
            chain(xs[2], outs[2])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    fp8.check_device_errors(DEV)


def test_stream_and_graph():
    """The whole chain on a side stream, and captured once and replayed on new inputs."""
    from flashbfp_b200 import fp8
    g = gen(5)
    k, n = 1024, 512
    w = fp8.quantize_fp8(0.02 * torch.randn(n, k, generator=g, device=DEV))
    lnw = torch.zeros(k, device=DEV, dtype=torch.bfloat16)
    x = torch.randn(7, k, generator=g, device=DEV).bfloat16()
    res = torch.randn(7, k, generator=g, device=DEV).bfloat16()

    def chain(x, res, out):
        return fp8.fp8_linear(fp8.rmsnorm_fp8(x, lnw, 1e-6, residual=res), w, out=out)

    y0 = chain(x, res.clone(), torch.empty(7, n, device=DEV, dtype=torch.bfloat16))
    torch.cuda.synchronize()
    side = torch.cuda.Stream(DEV)
    xs, rs, ys = x.clone(), res.clone(), torch.empty_like(y0)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(xs, rs, ys)
    side.synchronize()
    assert torch.equal(ys, y0)
    graph = torch.cuda.CUDAGraph()
    xs.zero_()
    with torch.cuda.graph(graph):
        chain(xs, rs, ys)
    for s in (1, 2):
        x2 = torch.randn(7, k, generator=gen(50 + s), device=DEV).bfloat16()
        xs.copy_(x2)
        rs.copy_(res)
        graph.replay()
        want_res = res.clone()
        want = chain(x2, want_res, torch.empty_like(y0))
        assert torch.equal(ys, want) and torch.equal(rs, want_res)
    fp8.check_device_errors(DEV)
