"""A decoder's own stream starts behind the stream that it was made on: weights that are still being
quantised or joined there, and buffers still being cleared, are ready before its first token."""
import pytest
import torch

from test_gpu_decode import _tiny

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _logits(dec, ids):
    dec.prefill(ids)
    dec.step()
    dec.check()
    return dec.logits[0].clone()


@pytest.mark.parametrize("weights", ["fp8", "oabf"])
def test_tokens_right_after_construction(weights):
    from flashbfp_b200 import OABFCompressor
    from flashbfp_b200.decode import GemmaDecoder
    from flashbfp_b200.model import compress_gemma_model
    model = _tiny(1).to(DEV, torch.bfloat16)
    if weights == "oabf":
        model = compress_gemma_model(model, OABFCompressor())
    ids = torch.randint(0, 512, (40,), generator=torch.Generator().manual_seed(7)).tolist()

    def make():
        return GemmaDecoder.from_hf(model, max_ctx=64, max_prefill=40, weights=weights)

    dec = make()
    torch.cuda.synchronize()
    want = _logits(dec, ids)
    dec.release()
    del dec
    big = torch.empty(1 << 28, dtype=torch.uint8, device=DEV).fill_(255)   # what fresh buffers may hold
    del big
    make()                                                   # the allocator's blocks, once more
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)                           # some 0.1 s on the current stream
    dec = make()
    got = _logits(dec, ids)
    dec.release()
    if weights == "fp8":
        assert torch.equal(got, want)
    else:       # the OABF linears' splits are added by atomics: bf16 values within two roundings a layer
        assert ((got.float() - want.float()).norm() / want.float().norm()).item() <= 2e-2
