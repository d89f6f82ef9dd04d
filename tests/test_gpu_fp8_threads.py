"""Calls of the 8-bit path from several threads at once, each with a stream of its own."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_two_threads_at_once():
    from flashbfp_b200 import fp8
    g = torch.Generator(device=DEV).manual_seed(3)
    w = fp8.quantize_fp8(0.02 * torch.randn(1000, 1500, generator=g, device=DEV))
    ln = 0.1 * torch.randn(1500, generator=g, device=DEV).bfloat16()
    xs = [torch.randn(m, 1500, generator=g, device=DEV).bfloat16() for m in (1, 40, 90, 300)]

    def chain(x):
        res = x.clone()
        y = fp8.fp8_linear(fp8.rmsnorm_fp8(x, ln, 1e-6, residual=res), w)
        return y, res, fp8.geglu_fp8(y).values

    want = [chain(x) for x in xs]
    torch.cuda.synchronize()
    bad, start = [], threading.Barrier(len(xs))

    def work(i):
        try:
            st = torch.cuda.Stream(DEV)
            start.wait()
            with torch.cuda.stream(st):
                for _ in range(50):
                    got = chain(xs[i])
                st.synchronize()
            if not all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want[i])):
                bad.append(i)
        except Exception as e:                       # a thread's failure is the test's
            bad.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    fp8.check_device_errors(DEV)
