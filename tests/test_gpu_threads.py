"""A host thread whose first CUDA call is one of the framework's: no context is current on it yet, and
its outputs come from memory that the allocator holds already."""
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

FP8 = """
import threading, torch
from flashbfp_b200 import fp8
def run(m):
    got.append((m, fp8.fp8_linear(xs[m], w, out=outs[m])))
w = fp8.quantize_fp8(torch.ones(8, 64, device="cuda:0"))
xs = {m: fp8.quantize_fp8(torch.ones(m, 64, device="cuda:0")) for m in (1, 40, 90, 300)}
outs = {m: torch.zeros(m, 8, device="cuda:0") for m in xs}
torch.cuda.synchronize()
got, ts = [], [threading.Thread(target=run, args=(m,)) for m in xs]
[t.start() for t in ts]; [t.join() for t in ts]
fp8.check_device_errors("cuda:0")
assert len(got) == 4 and all(bool((y == 64).all()) for _, y in got) and len(fp8._ERROR_WORDS) == 1
print("ok")
"""

OABF = """
import threading, torch
from flashbfp_b200 import OABFCompressor, packed, workloads
from flashbfp_b200.linear import check_device_errors, gemv_workspace, packed_linear
dev = torch.device("cuda", 0)
dp, sp = OABFCompressor().compress_matrix_device(workloads.decode_weight(512, 1024, seed=3, device=dev))
pw = packed.from_compressed(dp, sp, dev)
xs = {m: torch.randn(m, 1024, device=dev).bfloat16() for m in (1, 16, 40, 300)}
outs = {m: torch.zeros(m, 512, device=dev, dtype=torch.bfloat16) for m in xs}
gemv_workspace(dev, pw.npad)
torch.cuda.synchronize()
got = []
def run(m):
    got.append((m, packed_linear(xs[m], pw, out=outs[m], prefill="fused")))
for m in xs:                                   # one fresh thread after the other: they share a workspace
    t = threading.Thread(target=run, args=(m,)); t.start(); t.join(); torch.cuda.synchronize()
check_device_errors(dev)
assert len(got) == 4
for m, y in got:
    # the GEMV's splits are added by atomics, in any order: two roundings to bf16 of nearly equal sums
    want = packed_linear(xs[m], pw, prefill="fused").float()
    assert bool(want.any()) and (y.float() - want).norm() <= 2.0 ** -7 * want.norm()
print("ok")
"""


@pytest.mark.parametrize("code", [FP8, OABF], ids=["fp8_linear", "packed_linear"])
def test_first_call_of_a_thread(code):
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stderr[-2000:]
