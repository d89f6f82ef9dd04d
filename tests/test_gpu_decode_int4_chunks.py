"""A long prompt in many chunks over the 4-bit cache: few buffers are made to read it back, and the chunks give what one
sequence alone in larger ones gives."""
import pytest
import torch

from test_gpu_decode_int4 import _decoder, _ids

pytestmark = pytest.mark.gpu


def test_buffers_grow_few_times():
    model, dec = _decoder(5, max_ctx=12000, max_prefill=100, window=64)
    ids, seen = _ids(11000, 3), []
    torch.cuda.synchronize()
    for i in range(0, 11000, 100):
        dec.prefill(ids[i:i + 100])
        at = dec.back[0].data_ptr(), dec.back[0].shape[0]
        if at not in seen:
            seen.append(at)
    dec.check()
    assert [r for _, r in seen] == [1024, 2048, 4096, 8192, dec.cache4[0].positions]
    many = dec.logits.float().clone()
    dec.release()
    from flashbfp_b200.decode import GemmaDecoder
    one = GemmaDecoder.from_hf(model, max_ctx=12000, max_prefill=4000, kv_cache="int4")
    for i in range(0, 11000, 4000):
        one.prefill(ids[i:i + 4000])
    one.check()
    for x, y in zip(dec.cache4[0][:4], one.cache4[0][:4]):      # the first layer's input does not depend on the chunks
        assert torch.equal(x[:, :, :11000], y[:, :, :11000])
    assert torch.isfinite(many).all()
    one.release()


@pytest.mark.parametrize("captured", [False, True])
def test_positions_behind_max_ctx_are_recorded(captured):
    """max_ctx is the limit, as with the bf16 cache, though the 4-bit cache's length is a multiple of 32."""
    model, dec = _decoder(5, max_ctx=41, max_prefill=16, batch=2)
    assert dec.cache4[0].positions == 64
    dec.reset([38, 0])
    if captured:
        dec.capture()
    for _ in range(3):
        dec.step()
    dec.check()
    dec.step()                                           # position 41
    with pytest.raises(RuntimeError, match=r"outside the KV cache \(41\)"):
        dec.check()
    dec.reset([30, 0])
    dec.prefill(_ids(11, 1))                             # up to 40
    dec.check()
    dec.reset([0, 30])
    dec.prefill_packed([[], _ids(12, 1)])
    with pytest.raises(RuntimeError, match="outside"):
        dec.check()
    dec.reset(41)
    dec.prefill_packed([_ids(3, 2), []])
    with pytest.raises(RuntimeError, match="outside"):
        dec.check()
    dec.release()


def test_positions_before_the_cache_are_recorded():
    model, dec = _decoder(5, max_ctx=64, max_prefill=8)
    for call in (lambda: dec.step(), lambda: dec.prefill([3]), lambda: dec.prefill([3, 4, 5])):
        dec.reset(-1)
        call()
        with pytest.raises(RuntimeError, match="outside"):
            dec.check()
    dec.reset(0)
    dec.prefill([3])
    dec.check()
    dec.release()
