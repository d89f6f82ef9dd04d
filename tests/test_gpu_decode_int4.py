"""GemmaDecoder on the 4-bit cache: append, attention, reading back and the prompts' attention as they run
together.

Reference: Hugging Face's model with the same dequantised weights whose attention sees keys and values as
the cache holds them (quantised to 4 bits after norm and rotation, queries left as they are). Rounding to 4
bits is a step: where the two sides differ by d before it, a share |d| / s of the values lands a whole step s
apart, so that the mean square of the difference is s E|d|. A group's step is max / 7, of 32 near-normal
values 0.3 of their root mean square r (their maximum is 2.07 r on average); d is at most 2e-2 r, the
bf16 decoder's bound for all that rounds to bf16 at other points, E|d| 1.6e-2 r. So keys and values differ by
sqrt(0.3 * 1.6e-2) = 7e-2 in root mean square, and an attention branch, which takes both, by 0.1. Two of the
model's four branches of equal size are attention: their sum moves by sqrt(2) 0.1 / sqrt(4) = 7e-2, 1.5
times that for the non-linear parts between, and the 2e-2 of the bf16 roundings themselves: 0.125. (That
attention over a given cache is exact to its roundings is tested by itself.)

The decoder against itself: prompts in chunks of any cut, packed or not, stepped or replayed, leave the same
bytes in the cache of the first layer, whose input does not depend on how it is attended to.
"""
import pytest
import torch

from attention_reference import stored
from test_gpu_decode import _dequantised_reference, _run, _tiny

pytestmark = pytest.mark.gpu
BOUND = 2e-2 + 1.5 * 7e-2


def _quantised_attention(model):
    """Hugging Face's eager attention over keys and values as the 4-bit cache holds them."""
    from transformers.models.gemma3 import modeling_gemma3 as g3

    def held(x):
        return stored(x)[2].to(x.dtype).to(x.device)

    def attend(module, query, key, value, attention_mask, dropout=0.0, scaling=None, **kw):
        groups = query.shape[1] // key.shape[1]
        k, v = (held(t).repeat_interleave(groups, 1) for t in (key, value))
        s = (query.float() @ k.float().transpose(2, 3)) * (module.scaling if scaling is None else scaling)
        if attention_mask is not None:
            s = s + attention_mask[:, :, :, :k.shape[2]].float()
        w = torch.softmax(s, dim=-1)
        return (w @ v.float()).to(query.dtype).transpose(1, 2).contiguous(), w

    from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS
    ALL_ATTENTION_FUNCTIONS.register("held_in_4_bits", attend)
    model.config._attn_implementation = "held_in_4_bits"
    from transformers.masking_utils import ALL_MASK_ATTENTION_FUNCTIONS
    ALL_MASK_ATTENTION_FUNCTIONS.register("held_in_4_bits", ALL_MASK_ATTENTION_FUNCTIONS["eager"])
    assert g3 is not None
    return model


def _decoder(seed, **kw):
    from flashbfp_b200 import OABFCompressor
    from flashbfp_b200.decode import GemmaDecoder
    from flashbfp_b200.model import compress_gemma_model
    dev = torch.device("cuda", 0)
    model = compress_gemma_model(_tiny(seed, kw.pop("window", 4), 512).to(dev, torch.bfloat16), OABFCompressor())
    return model, GemmaDecoder.from_hf(model, kv_cache="int4", **kw)


def _ids(n, seed):
    return torch.randint(0, 512, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def test_steps_and_chunks_match_hugging_face_on_held_keys():
    model, dec = _decoder(1, max_ctx=300, max_prefill=140, window=100)
    ref = _quantised_attention(_dequantised_reference(_tiny(1, 100, 512).to("cuda", torch.bfloat16)))
    ids = _ids(200, 7)
    with torch.no_grad():
        want = ref(torch.tensor([ids], device="cuda")).logits[0].float()
    ours = _run(dec, ids[:150])
    for i in range(150):
        rel = ((ours[i] - want[i]).norm() / want[i].norm()).item()
        assert rel <= BOUND, (i, rel)
    for chunks in ((5,), (140,), (130, 3, 60)):
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
    dec.capture()
    again = _run(dec, ids[:60])
    rel = ((again - ours[:60]).norm() / ours[:60].norm()).item()
    assert rel <= 1e-3, rel
    with pytest.raises(ValueError, match="prompt chunk"):
        dec.prefill(ids[:141])
    dec.release()


def test_packed_prompts_equal_single_ones():
    """Three prompts of different lengths in packed chunks: the first layer's cache holds the same bytes as when each
    prompt went in alone, and the logits agree within the bound for re-ordered sums."""
    model, batch = _decoder(4, max_ctx=64, max_prefill=16, batch=3)
    from flashbfp_b200.decode import GemmaDecoder
    single = GemmaDecoder.from_hf(model, max_ctx=64, max_prefill=16, kv_cache="int4")
    prompts = [_ids(n, n) for n in (5, 19, 2)]
    batch.reset(0)
    batch.prefill_packed([prompts[0], prompts[1][:9], prompts[2]])
    batch.prefill_packed([[], prompts[1][9:], []])
    batch.check()
    assert batch.pos.tolist() == [5, 19, 2]
    for b, p in enumerate(prompts):
        single.reset(0)
        for i in range(0, len(p), 16):
            single.prefill(p[i:i + 16])
        single.check()
        for x, y in zip(batch.cache4[0][:4], single.cache4[0][:4]):
            assert torch.equal(x[b, :, :len(p)], y[0, :, :len(p)]), b
        rel = ((batch.logits[b].float() - single.logits[0].float()).norm() / single.logits[0].float().norm()).item()
        assert rel <= 1e-2, (b, rel)
        assert batch.pos[b].item() == single.pos[0].item()
    outs = batch.generate(prompts, 6)
    assert len(outs) == 3 and all(len(o) == 6 and all(0 <= t < 512 for t in o) for o in outs)
    batch.capture()
    assert batch.generate(prompts, 6) == outs
    with pytest.raises(ValueError, match="one chunk per sequence"):
        batch.prefill_packed([[1], [2]])
    with pytest.raises(ValueError, match="1..16"):
        batch.prefill_packed([[1] * 10, [2] * 10, []])
    batch.release()
    single.release()


def test_fp8_linears_over_the_4_bit_cache():
    from flashbfp_b200.decode import GemmaDecoder
    model = _tiny(3, 8).to("cuda", torch.bfloat16)
    dec = GemmaDecoder.from_hf(model, max_ctx=96, max_prefill=32, weights="fp8", kv_cache="int4")
    prompt = _ids(40, 9)
    first = dec.generate(prompt, 8)
    assert dec.generate(prompt, 8) == first
    dec.release()


def test_longer_contexts_than_the_bf16_cache_holds_and_positions_outside():
    from flashbfp_b200.decode import GemmaDecoder
    model, dec = _decoder(5, max_ctx=12000, max_prefill=4096, window=64)
    with pytest.raises(ValueError, match="10000"):
        GemmaDecoder.from_hf(model, max_ctx=12000)
    ids = _ids(9000, 11)
    for i in range(0, 9000, 4096):
        dec.prefill(ids[i:i + 4096])
    dec.step()
    dec.check()
    assert dec.pos.item() == 9001 and torch.isfinite(dec.logits).all()
    dec.reset(dec.cache4[0].positions)
    dec.step()
    with pytest.raises(RuntimeError, match="position outside"):
        dec.check()
    dec.reset(0)
    with torch.cuda.stream(dec.stream):
        dec.pos.fill_(50)                              # behind the decoder's back: not silently short
    dec.prefill(ids[:3])
    with pytest.raises(RuntimeError, match="position outside"):
        dec.check()
    with pytest.raises(ValueError, match="'bf16' or 'int4'"):
        GemmaDecoder.from_hf(model, max_ctx=64, kv_cache="fp4")
    dec.release()


def test_append_equals_norm_rotation_and_write():
    """The fused append against its parts: q and the rotated k as fbfp_qk_rope_cache rounds them, k and v as kv4_write
    holds them."""
    from flashbfp_b200 import _lib, kv4
    from flashbfp_b200.decode import rope_tables
    dev = torch.device("cuda", 0)
    L, P = _lib.lib(), _lib.ptr
    for d, h, kvh in ((64, 4, 2), (256, 16, 8), (48, 3, 1), (16, 2, 2)):
        g = torch.Generator(device=dev).manual_seed(d)
        rows, seqs = 37, 3
        qkv = torch.randn(rows + 2, (h + 2 * kvh) * d, generator=g, device=dev).bfloat16()
        qn, kn = (0.2 * torch.randn(d, generator=g, device=dev).bfloat16() for _ in range(2))
        cos, sin = rope_tables(10000.0, d, 96, dev)
        starts = torch.tensor([0, 20, 20, 37], dtype=torch.int32, device=dev)
        pos = torch.tensor([3, 60, 79], dtype=torch.int32, device=dev)
        cache = kv4.empty_cache(seqs, kvh, 96, d, dev)
        want = kv4.empty_cache(seqs, kvh, 96, d, dev)
        q = torch.full((rows + 2, h, d), 9.0, dtype=torch.bfloat16, device=dev)
        kv4.kv4_append(cache, qkv, qn, kn, 1e-6, cos, sin, pos, q, starts=starts)
        kv4.check_device_errors()
        kc, vc = (torch.zeros(kvh, 96, d, dtype=torch.bfloat16, device=dev) for _ in range(2))
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        st = _lib.stream_ptr(dev)
        for b, (r0, r1) in enumerate(((0, 20), (20, 20), (20, 37))):
            if r0 == r1:
                continue
            part = qkv[r0:r1].contiguous()
            qq = torch.empty(r1 - r0, h, d, dtype=torch.bfloat16, device=dev)
            p = pos[b:b + 1]
            _lib.check(L.fbfp_qk_rope_cache(P(part), r1 - r0, h, kvh, d, P(qn), P(kn), 1e-6, P(cos), P(sin), P(p), 96,
                                            P(qq), P(kc), P(vc), P(err), st), "rope")
            # both sum a head's squares in fp32, in another order: a norm may round the other way, by a bf16 step
            off = (q[r0:r1].float() - qq.float()).abs()
            assert (off <= 2.0 ** -6 * qq.float().abs().amax(-1, keepdim=True)).all()
            assert (off > 0).float().mean().item() <= 0.02
            p0 = pos[b].item()
            keys, vals = (c[:, p0:p0 + r1 - r0].transpose(0, 1) for c in (kc, vc))
            kv4.kv4_write(want, keys, vals, torch.tensor([p0 if i == b else 0 for i in range(seqs)], dtype=torch.int32, device=dev),
                          starts=torch.tensor([0 if i <= b else r1 - r0 for i in range(seqs + 1)], dtype=torch.int32, device=dev))
        assert bool((q[rows:] == 9).all())
        assert torch.equal(cache.v_values, want.v_values) and torch.equal(cache.v_scales, want.v_scales)
        assert (cache.k_values != want.k_values).float().mean().item() <= 0.02
        with pytest.raises(ValueError, match="pass starts"):
            kv4.kv4_append(cache, qkv, qn, kn, 1e-6, cos, sin, pos, q)
        with pytest.raises(ValueError, match="positions"):
            kv4.kv4_append(cache, qkv, qn, kn, 1e-6, cos[:50], sin[:50], pos, q, starts=starts)
        with pytest.raises(ValueError, match="bfloat16"):
            kv4.kv4_append(cache, qkv.float(), qn, kn, 1e-6, cos, sin, pos, q, starts=starts)
