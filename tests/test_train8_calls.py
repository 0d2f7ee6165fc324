"""CPU checks of how the 8-bit training operators are called: the context that calls of several threads share, operands of a
wrong kind, tensors that require a gradient."""
import threading

import pytest
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


def test_operands_of_a_wrong_kind_are_refused_by_name():
    """A tensor in a Blocks8's place, the other way round, None and numbers: the framework's error, with the operand's name."""
    bf = torch.bfloat16
    x, w, st = torch.zeros((4, 256), dtype=bf), torch.ones(256), torch.zeros((4, 2))
    q, w8, dy = f.Blocks8.empty(4, 256, "cpu"), f.Blocks8.empty(24, 256, "cpu"), torch.zeros((4, 24), dtype=bf)
    for name, call in (
            ("out", lambda: f.quantize8(x, out=x)),
            ("q", lambda: f.dequantize8(x)),
            ("q", lambda: f.dequantize8(None)),
            ("out", lambda: f.dequantize8(q, out=q)),
            ("out", lambda: f.layer_norm(x, out=q)),
            ("out", lambda: f.layer_norm(x, quantized=True, out=x)),
            ("weight", lambda: f.layer_norm(x, 1.0)),
            ("bias", lambda: f.layer_norm(x, w, [0.0] * 256)),
            ("x", lambda: f.layer_norm(q)),
            ("stats", lambda: f.layer_norm_backward(x, x, None)),
            ("stats", lambda: f.layer_norm_backward(x, q, (0.0, 1.0))),
            ("x", lambda: f.layer_norm_backward(x, None, st)),
            ("dy", lambda: f.layer_norm_backward(q, x, st)),
            ("out", lambda: f.layer_norm_backward(x, x, st, out=q)),
            ("x", lambda: f.linear8(None, w8)),
            ("weight", lambda: f.linear8(x, None)),
            ("bias", lambda: f.linear8(x, w8, 0.5)),
            ("out", lambda: f.linear8(x, w8, out=q)),
            ("x8", lambda: f.linear8_weight_grad(dy, None)),
            ("dy", lambda: f.linear8_weight_grad(q, q)),
            ("out", lambda: f.linear8_weight_grad(dy, q, out=w8)),
            ("Blocks8", lambda: f.Blocks8(None, q.scales, 256)),
            ("Blocks8", lambda: f.Blocks8(q.codes, 1, 256)),
            ("Blocks8", lambda: f.Blocks8(q.codes, q.scales, 256.0)),
            ("stream", lambda: f.quantize8(None, stream=0)),
            ("stream", lambda: f.linear8([1.0], w8, stream=0))):
        with pytest.raises(f.FVSRError, match=f"^{name} failed"):
            call()


def test_a_gradient_is_not_dropped_without_a_word():
    """Where autograd records, a tensor that requires a gradient is refused; under no_grad, and inside an autograd function, the call
    goes on (here as far as the check of its device)."""
    bf = torch.bfloat16
    x, w, st = torch.zeros((4, 256), dtype=bf), torch.ones(256), torch.zeros((4, 2))
    q, w8, dy, b = f.Blocks8.empty(4, 256, "cpu"), f.Blocks8.empty(24, 256, "cpu"), torch.zeros((4, 24), dtype=bf), torch.zeros(24)
    r = lambda t: t.clone().requires_grad_()  # noqa: E731
    calls = (("x", lambda: f.quantize8(r(x))),
             ("out", lambda: f.dequantize8(q, out=r(x))),
             ("x", lambda: f.layer_norm(r(x)[None], w)),
             ("weight", lambda: f.layer_norm(x, r(w))),
             ("bias", lambda: f.layer_norm(x, w, torch.nn.Parameter(w), quantized=True)),
             ("out", lambda: f.layer_norm(x, out=r(x))),
             ("dy", lambda: f.layer_norm_backward(r(x), x, st)),
             ("x", lambda: f.layer_norm_backward(x, r(x), st)),
             ("stats", lambda: f.layer_norm_backward(x, q, r(st))),
             ("weight", lambda: f.layer_norm_backward(x, q, st, r(w))),
             ("x", lambda: f.linear8(r(x), w8)),
             ("bias", lambda: f.linear8(q, w8, r(b))),
             ("dy", lambda: f.linear8_weight_grad(r(dy), q)))
    for name, call in calls:
        with pytest.raises(f.FVSRError, match=f"^{name} failed.*requires a gradient") as e:
            call()
        assert e.value.status == f._abi.ERR_UNSUPPORTED

    class Inside(torch.autograd.Function):
        @staticmethod
        def forward(ctx, t):
            return f.layer_norm(t, w)[0]

    with torch.no_grad():
        for _, call in calls:
            with pytest.raises(f.FVSRError, match="HIP device"):
                call()
    with pytest.raises(f.FVSRError, match="HIP device"):
        Inside.apply(r(x))
