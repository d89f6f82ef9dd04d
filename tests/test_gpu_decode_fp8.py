"""GemmaDecoder on block-scaled 8-bit linears: the run of quantise, norm, GeGLU and product together.

A tiny random-init Gemma-3 through ``from_hf(..., weights="fp8")``, against Hugging Face on the
same model whose targeted linears hold the dequantised 8-bit weights. What is left between the
two is the rounding of the linears' inputs to e4m3: a value moves by at most 2^-4 and, spread
evenly over a step of 2^-3 to 2^-4 of it, by 2^-5 in root mean square, so a product of such rows
moves by 2^-5 of its size. Each of the model's four residual branches (attention and MLP of two
layers) runs two products in a row: at most 2 * 2^-5 of the branch. The branches are normalised
to the same size, so the sum of four of them (with the embedding, which is exact) moves by at most
2 * 2^-5 in relative L2; the bound is 1.5 times that for the non-linear parts between (0.094).
"""
import pytest
import torch

from test_gpu_decode import _run, _tiny

pytestmark = pytest.mark.gpu
BOUND = 1.5 * 2 * 2.0 ** -5


def _dequantised(model):
    from flashbfp_b200 import fp8
    from flashbfp_b200.model import find_linear_layers
    for _, _, lin, _ in find_linear_layers(model):
        lin.weight.data.copy_(fp8.quantize_fp8(lin.weight.data).dequantize(torch.bfloat16))
    return model


def test_fp8_decoder_matches_hugging_face():
    from flashbfp_b200.decode import GemmaDecoder
    dev = torch.device("cuda", 0)
    dec = GemmaDecoder.from_hf(_tiny(1).to(dev, torch.bfloat16), max_ctx=160, max_prefill=140, weights="fp8")
    ref = _dequantised(_tiny(1).to(dev, torch.bfloat16))
    ids = torch.randint(0, 512, (150,), generator=torch.Generator().manual_seed(7)).tolist()
    with torch.no_grad():
        want = ref(torch.tensor([ids], device=dev)).logits[0].float()
    ours = _run(dec, ids[:24])
    for i in range(24):
        rel = ((ours[i] - want[i]).norm() / want[i].norm()).item()
        assert rel <= BOUND, (i, rel)
    # prompt chunks (few rows, more than a scale tile of them, and both in turn), then single tokens
    for chunks in ((5,), (140,), (130, 3)):
        dec.reset(0)
        n = 0
        for c in chunks:
            dec.prefill(ids[n:n + c])
            n += c
        dec.stream.synchronize()
        got = [dec.logits[0].float().clone()]
        for t in ids[n:n + 4]:
            with torch.cuda.stream(dec.stream):
                dec.tok.fill_(int(t))
            dec.step()
            dec.stream.synchronize()
            got.append(dec.logits[0].float().clone())
        dec.check()
        for j, g in enumerate(got):
            rel = ((g - want[n - 1 + j]).norm() / want[n - 1 + j].norm()).item()
            assert rel <= BOUND, (chunks, n - 1 + j, rel)
    # the captured step gives the same bits
    dec.capture()
    again = _run(dec, ids[:24])
    assert torch.equal(again, ours)
    toks = dec.generate(ids[:4], 6)
    assert len(toks) == 6 and all(0 <= t < 512 for t in toks)
    dec.release()


def test_fp8_batch_and_refusals():
    from flashbfp_b200 import OABFCompressor, fp8
    from flashbfp_b200.decode import DecodeLayer, GemmaDecoder
    from flashbfp_b200.model import compress_gemma_model
    dev = torch.device("cuda", 0)
    model = _tiny(2).to(dev, torch.bfloat16)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (5, 19, 2)]
    single = GemmaDecoder.from_hf(model, max_ctx=48, max_prefill=16, weights="fp8")
    batch = GemmaDecoder.from_hf(model, max_ctx=48, max_prefill=16, batch=3, weights="fp8")
    batch.capture()
    batch.reset(0)
    for b, p in enumerate(prompts):
        for i in range(0, len(p), 16):
            batch.prefill(p[i:i + 16], seq=b)
    follow = torch.randint(0, 512, (3,), generator=g).tolist()
    with torch.cuda.stream(batch.stream):
        batch.tok.copy_(torch.tensor(follow, device=dev))
    batch.step()
    batch.check()
    for b, p in enumerate(prompts):
        single.reset(0)
        for i in range(0, len(p), 16):
            single.prefill(p[i:i + 16])
        with torch.cuda.stream(single.stream):
            single.tok.fill_(follow[b])
        single.step()
        single.check()
        # a row's quantisation does not depend on the other rows; lm_head's sums may differ in order
        want = single.logits[0].float()
        assert ((batch.logits[b].float() - want).norm() / want.norm()).item() <= 1e-2, b
    # mixed layers are refused, and a compressed model
    ly = batch.layers[0]
    mixed = DecodeLayer(**{**ly.__dict__, "o": ly.o.dequantize(torch.bfloat16)})
    with pytest.raises(ValueError, match="all or none"):
        GemmaDecoder(batch.shape, [mixed, batch.layers[1]], batch.embed, batch.final_norm, batch.lm_head, 48)
    assert isinstance(ly.qkv, fp8.Fp8Rows)
    with pytest.raises(TypeError, match="weights='fp8'"):
        GemmaDecoder.from_hf(compress_gemma_model(model, OABFCompressor()), max_ctx=16, weights="fp8")
    batch.release()
