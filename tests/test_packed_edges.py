"""CPU checks of the packed and 8-bit operators at the edges of what they take: tangents, axes."""
import pytest
import torch
from torch.autograd import forward_ad

import fvsr_lcsa as f

bf = torch.bfloat16


def test_a_tensor_with_a_tangent_is_refused():
    """Forward-mode differentiation would lose it without a word, whether autograd records or not. Inside an autograd function the calls
    take what they are given: the next refusal is of the CPU tensors here."""
    x, w, rstd = torch.zeros((6, 256), dtype=bf), torch.ones(256), torch.ones(6)
    q, k = torch.zeros((6, 4, 64), dtype=bf), torch.zeros((6, 2, 64), dtype=bf)
    lse, cu = torch.zeros(4, 6), torch.tensor([0, 2, 6], dtype=torch.int32)
    pos, freq = torch.zeros((1, 6), dtype=torch.int32), torch.zeros(8, dtype=torch.float64)
    w8 = f.Blocks8.empty(128, 256, "cpu")
    x8, stats = f.Blocks8.empty(6, 256, "cpu"), torch.zeros(6, 2)
    calls = {
        "x": [(lambda t: f.rms_norm(t, w), x), (lambda t: f.quantize8(t), x), (lambda t: f.layer_norm(t, w), x), (lambda t: f.linear8(t, w8), x)],
        "weight": [(lambda t: f.rms_norm(x, t), w), (lambda t: f.layer_norm(x, t), w)],
        "bias": [(lambda t: f.linear8(x, w8, t), w[:128])],
        "residual": [(lambda t: f.rms_norm(x, residual=t), x)],
        "dy": [(lambda t: f.rms_norm_backward(t, x, rstd), x), (lambda t: f.layer_norm_backward(t, x, stats), x),
               (lambda t: f.linear8_weight_grad(t, x8), x[:, :128].contiguous())],
        "total": [(lambda t: f.rms_norm_backward(x, t, rstd), x)],
        "q": [(lambda t: f.rotary(t, k, pos, freq, (8,)), q), (lambda t: f.packed_attention(t, k, k, cu), q)],
        "k": [(lambda t: f.rotary_backward(q, t, pos, freq, (8,)), k), (lambda t: f.packed_attention(q, t, k, cu), k)],
        "v": [(lambda t: f.packed_attention(q, k, t, cu), k)],
        "do": [(lambda t: f.packed_attention_backward(t, q, k, k, q, lse, cu), q)],
        "lse": [(lambda t: f.packed_attention_backward(q, q, k, k, q, t, cu), lse)],
    }

    class Inside(torch.autograd.Function):
        @staticmethod
        def forward(call, t):
            with pytest.raises(f.FVSRError, match="HIP device"):
                call(t)
            return t.clone()

        @staticmethod
        def setup_context(ctx, inputs, output):
            pass

        @staticmethod
        def jvp(ctx, none, tangent):
            return tangent.clone()

    for name, of in calls.items():
        for call, t in of:
            with forward_ad.dual_level():
                dual = forward_ad.make_dual(t, torch.ones_like(t))
                for mode in (torch.no_grad, torch.enable_grad):
                    with mode(), pytest.raises(f.FVSRError, match=f"^{name} failed.*tangent") as e:
                        call(dual)
                    assert e.value.status == f._abi.ERR_UNSUPPORTED
                with pytest.raises(f.FVSRError, match="HIP device"):
                    call(forward_ad.unpack_dual(dual).primal)
                Inside.apply(call, dual)
            with pytest.raises(f.FVSRError, match="HIP device"):
                call(t)


def test_axes_are_whole_numbers_as_they_are_now():
    """Pairs that are no whole numbers are refused, not cut off; numbers that change in place are read anew in each call."""
    q = torch.zeros((6, 2, 64), dtype=bf)
    pos, freq = torch.zeros((2, 6), dtype=torch.int32), torch.zeros(20, dtype=torch.float64)
    for axes in ((10.5, 10.5), (10.9, 10), ("10", "10"), "aa", (10, float("nan")), (10, float("inf")), (10, 2 ** 40), ((10,), 10), 20, None):
        with pytest.raises(f.FVSRError, match="axes"):
            f.rotary(q, None, pos, freq, axes)
    held = [torch.tensor(10), torch.tensor(10)]
    for axes in ((10, 10), [4, 16], (10.0, 10.0), torch.tensor([10, 10]), held):
        with pytest.raises(f.FVSRError, match="HIP device"):
            f.rotary(q, None, pos, freq, axes)
    held[0].fill_(9)
    with pytest.raises(f.FVSRError, match="frequencies.*19"):
        f.rotary(q, None, pos, freq, held)
