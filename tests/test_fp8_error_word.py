"""The device word in which a product records a wait that gave up: one per device, whoever asks first
(no GPU: the device calls are stand-ins)."""
import contextlib
import threading
import time

import pytest
import torch

from flashbfp_b200 import fp8

INDEX = 5


@pytest.fixture
def device(monkeypatch):
    """Stand-ins that know which device is current and let other threads in where the real calls do."""
    state = {"current": 0, "capturing": ()}

    @contextlib.contextmanager
    def use(index):
        before, state["current"] = state["current"], index
        try:
            yield
        finally:
            state["current"] = before

    made = torch.zeros
    monkeypatch.setattr(torch.cuda, "device", use)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda index=None: time.sleep(0.05))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["current"] in state["capturing"])
    monkeypatch.setattr(torch, "zeros", lambda *a, device=None, **k: made(*a, **k))
    monkeypatch.setattr(fp8, "_ERROR_WORDS", {})
    return state


def test_first_calls_of_two_threads_share_a_word(device):
    got, start = [], threading.Barrier(4)

    def ask():
        start.wait()
        got.append(fp8._error_word(INDEX))

    threads = [threading.Thread(target=ask) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(set(got)) == 1                       # what a kernel may hold is never replaced
    assert got[0] == fp8._ERROR_WORDS[INDEX].data_ptr()
    assert fp8._error_word(INDEX) == got[0]


def test_a_capture_is_looked_for_on_the_operands_device(device):
    device["capturing"] = (INDEX,)
    with pytest.raises(RuntimeError, match="outside a CUDA graph capture"):
        fp8._error_word(INDEX)
    assert INDEX not in fp8._ERROR_WORDS
    device["capturing"] = (0,)                      # the current device's stream has nothing to do with it
    assert fp8._error_word(INDEX) == fp8._ERROR_WORDS[INDEX].data_ptr()
    assert device["current"] == 0
