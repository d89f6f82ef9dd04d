"""The decoder on the 4-bit cache with a tensor-parallel reducer (of one rank: the sums, the packed chunks' picks and the
fused exchange run as they do on several): what it gives without one.

The first layer's cache holds the same bytes: nothing before it is summed over ranks. Behind it the row-parallel
products are summed in another order, so that bf16 rounds some the other way. Before a cached row is quantised the two
sides differ by no more than the 2e-2 that tensor parallelism is allowed without quantisation, which is the difference
that test_gpu_decode_int4 starts from: what 4 bits make of it is derived there (BOUND)."""
import pytest
import torch

from test_gpu_decode import _tiny
from test_gpu_decode_int4 import BOUND, _ids

pytestmark = pytest.mark.gpu


def test_packed_chunks_and_steps_with_a_reducer():
    import torch.distributed as dist
    from flashbfp_b200 import OABFCompressor
    from flashbfp_b200.decode import GemmaDecoder
    from flashbfp_b200.model import compress_gemma_model
    from flashbfp_b200.tp import NVLinkAllReduce
    dev = torch.device("cuda", 0)
    ours = not dist.is_initialized()
    if ours:
        dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    try:
        whole = compress_gemma_model(_tiny(6, 32, 512).to(dev, torch.bfloat16), OABFCompressor())
        kw = dict(max_ctx=64, max_prefill=24, batch=3, kv_cache="int4")
        single = GemmaDecoder.from_hf(whole, **kw)
        tp = GemmaDecoder(single.shape, single.layers, single.embed, single.final_norm, single.lm_head,
                          reducer=NVLinkAllReduce(24 * 512), **kw)
        prompts = [_ids(n, n) for n in (7, 20, 1)]
        for chunks in ([prompts[0], prompts[1][:9], prompts[2]], [[], prompts[1][9:], []], [[5], [], [6, 7]]):
            for dec in (single, tp):
                dec.prefill_packed(chunks)
                dec.check()
            some = [b for b, c in enumerate(chunks) if c]
            a, b = tp.logits[some].float(), single.logits[some].float()
            assert ((a - b).norm() / b.norm()).item() <= BOUND
            assert torch.equal(tp.tok[some], tp.logits[some].argmax(-1)) and tp.pos.tolist() == single.pos.tolist()
        for _ in range(3):
            for dec in (single, tp):
                dec.tok.copy_(torch.tensor([1, 2, 3], device=dev))
                torch.cuda.synchronize()
                dec.step()
                dec.check()
            a, b = tp.logits.float(), single.logits.float()
            assert ((a - b).norm() / b.norm()).item() <= BOUND
        for x, y in zip(tp.cache4[0][:4], single.cache4[0][:4]):
            assert torch.equal(x, y)
        outs = tp.generate(prompts, 5)
        tp.capture()
        assert tp.generate(prompts, 5) == outs
        single.release()
        tp.release()
    finally:
        if ours:
            dist.destroy_process_group()
