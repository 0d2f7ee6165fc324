"""CPU checks of how the 8-bit training operators are called: the context that calls of several threads share."""
import threading

import torch

import fvsr_lcsa as f
from fvsr_lcsa import train8


def test_first_calls_of_two_threads_share_one_context(monkeypatch):
    """Two threads that make a device's first call at once get the same context, and no context that a call holds is destroyed. Creation
    is a stub in which each thread waits for the other (for a while: one of them only, if the other is kept out)."""
    device = torch.device("cuda", 61)   # no such device: nothing but the stubs is called
    made, ended, got = [], [], []
    both = threading.Barrier(2)

    def create(name, index, out):
        assert name == "fvsr_ctx_create" and index == device.index
        try:
            both.wait(1.0)
        except threading.BrokenBarrierError:
            pass
        made.append(len(made) + 1)
        out._obj.value = made[-1]

    monkeypatch.setattr(f, "call", create)
    monkeypatch.setattr(f.lib, "fvsr_ctx_destroy", lambda handle: ended.append(handle.value))
    threads = [threading.Thread(target=lambda: got.append(train8._ctx(device).value)) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    try:
        assert made == [1] and got == [1, 1] and not ended
        assert train8._ctx(device).value == f.Context.get(device).handle.value == 1
    finally:
        f.Context._by_device.pop(device.index, None)
        getattr(train8, "_contexts", {}).pop(device.index, None)
    assert ended == [1]
