"""The block-scaled 8-bit linear path as measurable cases: what a decoder layer runs around an
e4m3 product whose operands carry one power-of-two scale per 128 values of a row.

  quantize   rows of bf16 / fp16 / fp32 values to e4m3 with their scales
  rmsnorm    RMSNorm(x; 1 + w) to e4m3 with scales, plain, after the residual's addition, or between
             a layer's halves (post-norm, residual addition, next pre-norm)
  geglu      gelu_tanh(gate) * up to e4m3 with scales
  linear     y = x w^T (+ bias) of two such operands

A scale is the smallest power of two 2^(c - 127), 0 <= c <= 254, with max|block| / scale <= 448.
Scales are one byte each (c, dtype float8_e8m0fnu) in tiles of 128 rows by 4 blocks: element
[row / 128, block / 4, row % 32, row % 128 / 32, block % 4]; tile entries past the last row or
block hold c = 0. Values past a row's end are not part of the values tensor, whose rows start 16
bytes apart (or a multiple of it).

``run`` computes a case in plain torch operations in fp32, or, with ``own`` true, through
flashbfp_b200.fp8. ``exact`` gives the definition's result in fp64.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6
DEV = "cuda"


# ---------------------------------------------------------------------------- cases
def listed():
    return [
        # one decoded token through the fused q|k|v rows of the 12B-class layer
        dict(name="linear qkv m1", op="linear", m=1, n=8192, k=3840, dtype="bf16", bias=False),
        # a batch of 16 sequences decoding: gate|up, the layer's largest matrix
        dict(name="linear gate_up m16", op="linear", m=16, n=30720, k=3840, dtype="bf16", bias=False),
        # a 128-token prompt chunk through down_proj: few output rows, a long sum
        dict(name="linear down m128", op="linear", m=128, n=3840, k=15360, dtype="bf16", bias=False),
        # a 2048-token prompt through gate|up
        dict(name="linear gate_up m2048", op="linear", m=2048, n=30720, k=3840, dtype="bf16", bias=False),
        # odd sizes everywhere, fp32 output with a bias: a ragged batch into a head of its own
        dict(name="linear ragged m333", op="linear", m=333, n=1999, k=4090, dtype="fp32", bias=True),
        # between a layer's halves for one decoded token
        dict(name="rmsnorm post m1", op="rmsnorm", m=1, k=3840, dtype="bf16", mode="post"),
        # the same for a 2048-token prompt
        dict(name="rmsnorm post m2048", op="rmsnorm", m=2048, k=3840, dtype="bf16", mode="post"),
        # residual addition and norm of the 70B-class hidden size, a long prompt
        dict(name="rmsnorm add m8192", op="rmsnorm", m=8192, k=8192, dtype="bf16", mode="add"),
        # MLP activation for a batch of 16 decoding sequences
        dict(name="geglu m16", op="geglu", m=16, k=15360, dtype="bf16"),
        # the same for a 2048-token prompt
        dict(name="geglu m2048", op="geglu", m=2048, k=15360, dtype="bf16"),
        # attention output of a 128-token prompt chunk on its way into o_proj
        dict(name="quantize m128", op="quantize", m=128, k=4096, dtype="bf16"),
        # a weight matrix quantised at load time: the 12B-class down_proj in fp32
        dict(name="quantize weight", op="quantize", m=3840, k=15360, dtype="fp32"),
    ]


def _size(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm; half of them as they fall (odd ones
    among them), half rounded to a multiple of 64."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v >= 96:
        v = (v + 32) // 64 * 64
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["linear", "linear", "rmsnorm", "geglu", "quantize"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    while True:
        if op == "linear":
            c = dict(op=op, m=_size(rng, 1, 4096), n=_size(rng, 64, 32768), k=_size(rng, 64, 16384),
                     dtype=dtype, bias=rng.random() < 0.5)
            if c["m"] * c["n"] * c["k"] <= 2048 * 30720 * 3840 and c["n"] * c["k"] <= 30720 * 3840 \
                    and c["m"] * c["n"] * BYTES[dtype] <= 2048 * 30720 * 2:
                return c
        elif op == "rmsnorm":
            c = dict(op=op, m=_size(rng, 1, 8192), k=_size(rng, 64, 16384), dtype=dtype,
                     mode=rng.choice(["plain", "add", "post"]))
            if c["m"] * c["k"] * BYTES[dtype] <= 8192 * 8192 * 2:
                return c
        else:
            c = dict(op=op, m=_size(rng, 1, 8192), k=_size(rng, 64, 28672), dtype=dtype)
            if c["m"] * c["k"] * BYTES[dtype] <= 2048 * 15360 * 2:
                return c


def _blocks(k):
    return -(-k // 128)


def _scale_shape(m, k):
    return (-(-m // 128), -(-k // 512), 32, 4, 4)


def work(case):
    """Bytes: every input once, every output once. Operations: of a linear, its multiply-adds."""
    m, k, e = case["m"], case["k"], BYTES[case["dtype"]]
    rows = m * k + m * _blocks(k)                       # e4m3 values and their scales
    if case["op"] == "linear":
        n = case["n"]
        b = rows + n * k + n * _blocks(k) + m * n * e + (n * e if case["bias"] else 0)
        return {"bytes": b, "flops": 2 * m * n * k}
    if case["op"] == "rmsnorm":
        touched = {"plain": 1, "add": 3, "post": 3}[case["mode"]]
        b = touched * m * k * e + k * e * (2 if case["mode"] == "post" else 1) + rows
        return {"bytes": b, "flops": 10 * m * k}
    if case["op"] == "geglu":
        return {"bytes": 2 * m * k * e + rows, "flops": 15 * m * k}
    return {"bytes": m * k * e + rows, "flops": 3 * m * k}


# ---------------------------------------------------------------------------- inputs
def _activations(m, k, g):
    """Rows as a decoder's hidden states have them: normal values, rows of different size, and a
    few channels far above the others."""
    x = torch.randn(m, k, generator=g, device=DEV)
    x *= torch.exp(0.5 * torch.randn(m, 1, generator=g, device=DEV))
    ch = 1.0 + 15.0 * (torch.rand(k, generator=g, device=DEV) < 0.01).float()
    return x * ch


def _weights(n, k, g):
    """N(0, 0.02) with 1.5% of the entries ten times as large."""
    w = 0.02 * torch.randn(n, k, generator=g, device=DEV)
    return w * (1.0 + 9.0 * (torch.rand(n, k, generator=g, device=DEV) < 0.015).float())


def _rows_buffers(m, k):
    """An e4m3 values tensor (rows padded to 16 bytes) and its scale tiles, for a result."""
    v = torch.zeros(m, -(-k // 16) * 16, dtype=torch.float8_e4m3fn, device=DEV)[:, :k]
    s = torch.zeros(_scale_shape(m, k), dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu)
    return v, s


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    m, k, dt = case["m"], case["k"], DTYPES[case["dtype"]]
    s = {"case": dict(case)}
    if case["op"] == "linear":
        n = case["n"]
        # both operands as the program holds them: already e4m3 with their scale tiles
        for name, rows, dense in (("x", m, _activations(m, k, g)), ("w", n, _weights(n, k, g))):
            v, sc = _rows_buffers(rows, k)
            q, tiles = _quantize_plain(dense)
            v.copy_(q)
            s[name], s[name + "_scales"] = v, tiles
            del dense, q
        s["bias"] = torch.randn(n, generator=g, device=DEV).to(dt) if case["bias"] else None
        s["y"] = torch.empty(m, n, dtype=dt, device=DEV)
        return s
    s["values"], s["scales"] = _rows_buffers(m, k)
    if case["op"] == "geglu":
        s["gate_up"] = _activations(m, 2 * k, g).to(dt)
        return s
    s["x"] = _activations(m, k, g).to(dt)
    if case["op"] == "rmsnorm":
        s["weight"] = (0.2 * torch.randn(k, generator=g, device=DEV)).to(dt)
        s["residual"] = _activations(m, k, g).to(dt) if case["mode"] != "plain" else None
        s["post"] = (0.2 * torch.randn(k, generator=g, device=DEV)).to(dt) if case["mode"] == "post" else None
    return s


# ---------------------------------------------------------------------------- plain form, fp32
def _tile(codes):
    """Scale codes [m, blocks] (uint8) as tiles of 128 rows by 4 blocks."""
    m, b = codes.shape
    mt, kt = -(-m // 128), -(-b // 4)
    full = torch.zeros(mt * 128, kt * 4, dtype=torch.uint8, device=codes.device)
    full[:m, :b] = codes
    tiles = full.view(mt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).contiguous()
    return tiles.view(torch.float8_e8m0fnu)


def _untile(scales, m, b):
    """Scale tiles as a matrix of codes [m, blocks]."""
    t = scales.view(torch.uint8)
    mt, kt = t.shape[:2]
    return t.permute(0, 3, 2, 1, 4).reshape(mt * 128, kt * 4)[:m, :b]


def _quantize_plain(x):
    """fp32 rows to (e4m3 values, scale tiles)."""
    m, k = x.shape
    b = _blocks(k)
    p = torch.nn.functional.pad(x, (0, b * 128 - k)).view(m, b, 128)
    amax = p.abs().amax(dim=2)
    # the exponent of amax / 448 rounded up: 448 = 1.75 * 2^8, so one more where amax's mantissa
    # is above 1.75
    code = ((amax.view(torch.int32) + 0x1FFFFF) >> 23) - 8
    code = torch.where(torch.isfinite(amax), code.clamp(min=0), torch.full_like(code, 255))
    inv = torch.ldexp(torch.ones_like(amax), 127 - code)
    inv = torch.where(code == 255, torch.full_like(inv, math.nan), inv)
    q = (p * inv[:, :, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return q.view(m, b * 128)[:, :k], _tile(code.to(torch.uint8))


def _dequantize(values, scales, dtype):
    m, k = values.shape
    b = _blocks(k)
    s = torch.ldexp(torch.ones(m, b, dtype=dtype, device=values.device), _untile(scales, m, b).int() - 127)
    return values.to(dtype) * s.repeat_interleave(128, dim=1)[:, :k]


def _norm(x, w):
    return x * torch.rsqrt(x.square().mean(dim=1, keepdim=True) + EPS) * (1.0 + w.float())


def _run_plain(s):
    c = s["case"]
    if c["op"] == "linear":
        y = _dequantize(s["x"], s["x_scales"], torch.float32) @ _dequantize(s["w"], s["w_scales"], torch.float32).t()
        if s["bias"] is not None:
            y = y + s["bias"].float()
        return [y.to(s["y"].dtype)]
    if c["op"] == "quantize":
        return list(_quantize_plain(s["x"].float()))
    if c["op"] == "geglu":
        gate, up = s["gate_up"].float().chunk(2, dim=1)
        u = math.sqrt(2.0 / math.pi) * (gate + 0.044715 * gate * gate * gate)
        # gelu_tanh(g) = g (1 + tanh u) / 2 = g / (1 + exp(-2 u)), without the cancellation
        return list(_quantize_plain(gate / (1.0 + torch.exp(-2.0 * u)) * up))
    h = s["x"].float()
    if s["post"] is not None:
        h = _norm(h, s["post"])
    if s["residual"] is not None:
        h = h + s["residual"].float()
    q, t = _quantize_plain(_norm(h, s["weight"]))
    if s["residual"] is None:
        return [q, t]
    s["residual"].copy_(h)                             # the residual stream, updated in place
    return [q, t, s["residual"]]


# ---------------------------------------------------------------------------- the framework's calls
def _run_own(s):
    from flashbfp_b200 import fp8
    c = s["case"]
    if c["op"] == "linear":
        return [fp8.fp8_linear(fp8.Fp8Rows(s["x"], s["x_scales"]), fp8.Fp8Rows(s["w"], s["w_scales"]),
                               s["bias"], out=s["y"])]
    out = fp8.Fp8Rows(s["values"], s["scales"])
    if c["op"] == "quantize":
        fp8.quantize_fp8(s["x"], out=out)
    elif c["op"] == "geglu":
        fp8.geglu_fp8(s["gate_up"], out=out)
    else:
        fp8.rmsnorm_fp8(s["x"], s["weight"], EPS, residual=s["residual"], post_weight=s["post"], out=out)
        if s["residual"] is not None:
            return [s["values"], s["scales"], s["residual"]]
    return [s["values"], s["scales"]]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------- the definition, fp64
def _exact_quantize(x):
    """Values on the e4m3 grid and scale tiles of fp64 rows, as fp64 tensors."""
    m, k = x.shape
    b = _blocks(k)
    p = torch.zeros(m, b * 128, dtype=torch.float64, device=x.device)
    p[:, :k] = x
    p = p.view(m, b, 128)
    ratio = p.abs().amax(dim=2, keepdim=True) / 448.0
    mant, ex = torch.frexp(ratio)                       # ratio = mant * 2^ex, mant in [0.5, 1)
    ex = torch.where(mant == 0.5, ex - 1, ex)           # the smallest e with ratio <= 2^e
    ex = torch.where(ratio == 0, torch.full_like(ex, -127), ex).clamp(min=-127)
    v = torch.ldexp(p, -ex)
    # the spacing of e4m3 at |v|: 2^(floor(log2 |v|) - 3), at least 2^-9
    _, ve = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (ve - 4).clamp(min=-9))
    q = (torch.round(v / step) * step).clamp(-448.0, 448.0).view(m, b * 128)[:, :k]
    sc = torch.full((-(-m // 128) * 128, -(-b // 4) * 4), 2.0 ** -127, dtype=torch.float64, device=x.device)
    sc[:m, :b] = torch.ldexp(torch.ones_like(ratio), ex).view(m, b)
    sc = sc.view(-1, 4, 32, -(-b // 4), 4).permute(0, 3, 2, 1, 4).contiguous()
    return q.contiguous(), sc


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        x, w = (_dequantize(s[n], s[n + "_scales"], torch.float64) for n in ("x", "w"))
        y = torch.zeros(case["m"], case["n"], dtype=torch.float64, device=DEV)
        if s["bias"] is not None:
            y += s["bias"].double()
        return [torch.addmm(y, x, w.T)]
    if case["op"] == "quantize":
        return list(_exact_quantize(s["x"].double()))
    if case["op"] == "geglu":
        g, u = s["gate_up"][:, :case["k"]].double(), s["gate_up"][:, case["k"]:].double()
        t = math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)
        return list(_exact_quantize(g * torch.sigmoid(2.0 * t) * u))

    def norm(v, w):
        return v / torch.sqrt((v * v).sum(dim=1, keepdim=True) / v.shape[1] + EPS) * (1.0 + w.double())

    h = s["x"].double() if s["post"] is None else norm(s["x"].double(), s["post"])
    h = h if s["residual"] is None else h + s["residual"].double()
    out = list(_exact_quantize(norm(h, s["weight"])))
    return out if s["residual"] is None else out + [h]
