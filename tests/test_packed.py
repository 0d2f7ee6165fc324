"""CPU checks of the packed operators: what the binding and the C entry points refuse, before any device work, and the float64
forms that the GPU tests compare with, against differences of themselves."""
import ctypes as C
import math

import pytest
import torch

import fvsr_lcsa as f
from fvsr_lcsa import _abi
from fvsr_lcsa._abi import Heads, Packed
from packed_reference import attention64, rms64, rms_grad64, turn64

E = f.FVSRError
bf = torch.bfloat16


def heads(n=6, h=4, d=64, dtype=bf):
    return torch.zeros((n, h, d), dtype=dtype)


def cu(*x):
    return torch.tensor(x, dtype=torch.int32)


# ---- refusals ------------------------------------------------------------------------------------------------------------
def test_rms_norm_refusals():
    x, w = torch.zeros((4, 256), dtype=bf), torch.ones(256)
    for bad in (x.half(), x.t(), x[None].expand(2, 4, 256), torch.zeros(4), torch.zeros((4, 0)), None, x[:, ::2]):
        with pytest.raises(E, match="x"):
            f.rms_norm(bad)
    for kw in ({"weight": w[:255]}, {"weight": w.half()}, {"weight": torch.ones(512)[::2]}):
        with pytest.raises(E, match="weight"):
            f.rms_norm(x, **kw)
    for r in (x.float(), x[:3], 3):
        with pytest.raises(E, match="residual"):
            f.rms_norm(x, residual=r)
    with pytest.raises(E, match="out_sum"):
        f.rms_norm(x, out_sum=x)
    with pytest.raises(E, match="out"):
        f.rms_norm(x, quantized=True, out=f.Blocks8.empty(4, 255, "cpu"))
    with pytest.raises(E, match="HIP device"):
        f.rms_norm(x)
    with pytest.raises(E, match="requires a gradient"):
        f.rms_norm(x.float().requires_grad_())
    with pytest.raises(E, match="rstd"):
        f.rms_norm_backward(x, x, torch.zeros(4, 1))
    with pytest.raises(E, match="total"):
        f.rms_norm_backward(x, x.float(), torch.zeros(4))
    with pytest.raises(E, match="dsum"):
        f.rms_norm_backward(x, x, torch.zeros(4), dsum=x[:2])
    with pytest.raises(E, match="dy"):
        f.rms_norm_backward(torch.zeros((4, 512), dtype=bf)[:, :256], x, torch.zeros(4))


def test_rotary_refusals():
    q, k = heads(), heads(h=2)
    pos, freq = torch.zeros((2, 6), dtype=torch.int32), torch.zeros(20, dtype=torch.float64)
    for axes in ((), (1, 1, 1, 1), (33,), (0, 0), (-1, 3), None, (20, 13)):
        with pytest.raises(E, match="axes"):
            f.rotary(q, k, pos, freq, axes)
    for bad in (pos.float(), pos[:1], pos[:, :5], None):
        with pytest.raises(E, match="positions"):
            f.rotary(q, k, bad, freq, (10, 10))
    for bad in (freq.float(), freq[:19], None):
        with pytest.raises(E, match="frequencies"):
            f.rotary(q, k, pos, bad, (10, 10))
    with pytest.raises(E, match="k"):
        f.rotary(q, k[:5], pos, freq, (10, 10))
    with pytest.raises(E, match="k"):
        f.rotary(q, k.float(), pos, freq, (10, 10))
    with pytest.raises(E, match="out"):
        f.rotary(q, k, pos, freq, (10, 10), out=(q[:, :1].expand(6, 4, 64), k))
    with pytest.raises(E, match="out"):
        f.rotary(q, None, pos, freq, (10, 10), out=(q, k))
    for bad in (q, (q,), (q, k, k), (q, q[:, :2])):
        with pytest.raises(E, match="out"):
            f.rotary(q, k, pos, freq, (10, 10), out=bad)
    with pytest.raises(E, match="q"):
        f.rotary(q.transpose(1, 2), k, pos, freq, (10, 10))
    with pytest.raises(E, match="HIP device"):
        f.rotary(q, k, pos, freq, (10, 10))


def test_packed_attention_refusals():
    q, k = heads(), heads(h=2)
    c = cu(0, 2, 6)
    for bad in (q.float(), q[:, :, :60], heads(d=136), q[0], None):
        with pytest.raises(E, match="q"):
            f.packed_attention(bad, k, k, c)
    for bad in (heads(h=3), heads(d=32, h=2), k[:5]):
        with pytest.raises(E, match="k"):
            f.packed_attention(q, bad, bad, c)
    with pytest.raises(E, match="v"):
        f.packed_attention(q, k, k[:, :1], c)
    for bad in (c.long(), c[:1], c[None], None, [0, 6]):
        with pytest.raises(E, match="cu_q"):
            f.packed_attention(q, k, k, bad)
    with pytest.raises(E, match="cu_k"):
        f.packed_attention(q, k, k, c, cu(0, 6))
    with pytest.raises(E, match="used_k"):
        f.packed_attention(q, k, k, c, used_k=c)
    for bad in (0, -1.0, math.inf, math.nan):
        with pytest.raises(E, match="scale"):
            f.packed_attention(q, k, k, c, scale=bad)
    with pytest.raises(E, match="out"):
        f.packed_attention(q, k, k, c, out=heads(h=2))
    with pytest.raises(E, match="out"):
        f.packed_attention(q, k, k, c, out=torch.zeros(6 * 4 * 64 + 4, dtype=bf)[4:].view(6, 4, 64))
    with pytest.raises(E, match="HIP device"):
        f.packed_attention(q, k, k, c)
    with pytest.raises(E, match="requires a gradient"):
        f.packed_attention(q.clone().requires_grad_(), k, k, c)
    lse = torch.zeros(4, 6)
    with pytest.raises(E, match="lse"):
        f.packed_attention_backward(q, q, k, k, q, lse.t(), c)
    with pytest.raises(E, match="do"):
        f.packed_attention_backward(q[:5], q, k, k, q, lse, c)
    for bad in ((q, k), q, (q, k, None), (q, k, k[:5]), (q, k, k)):
        with pytest.raises(E, match="out"):
            f.packed_attention_backward(q, q, k, k, q, lse, c, out=bad)
    with pytest.raises(E, match="HIP device"):
        f.packed_attention_backward(q, q, k, k, q, lse, c)


def status(name, *args):
    return getattr(_abi.lib, name)(*args), _abi.lib.fvsr_last_error().decode()


def test_c_entry_points_refuse_before_device_work():
    p, ctx = C.c_void_p(16), C.c_void_p(8)   # never dereferenced: validation fails first
    assert status("fvsr_rms_norm", None, 1, p, 8, None, 1, 8, 1e-6, 0, None, p, None, None, None, None, None)[0] == _abi.ERR_INVALID_ARG
    for rows, ch, stride, dt, y in ((-1, 8, 8, 1, p), (1, 0, 8, 1, p), (1, 8, 7, 1, p), (1, 8, 8, 2, p), (1, 8, 8, 1, None)):
        assert status("fvsr_rms_norm", ctx, dt, p, stride, None, rows, ch, 1e-6, 0, None, y, None, None, None, None,
                      None)[0] == _abi.ERR_INVALID_ARG
    assert status("fvsr_rms_norm", ctx, 1, p, 16385, None, 1, 16385, 1e-6, 0, None, p, None, None, None, None, None)[0] == _abi.ERR_UNSUPPORTED
    assert status("fvsr_rms_norm", ctx, 1, p, 8, None, 1 << 40, 8, 1e-6, 0, None, p, None, None, None, None, None)[0] == _abi.ERR_UNSUPPORTED
    assert "workspace" in status("fvsr_rms_norm_backward", ctx, 1, p, p, 8, p, None, 4000, 8, 0, None, p, p, None, 0, None)[1]

    def view(heads=4, ts=256, hs=64, data=16):
        return C.byref(Heads(data, heads, ts, hs))

    def packed(**kw):
        a = dict(cu_q=16, cu_k=16, used_k=None, sequences=2, tokens_q=6, tokens_k=6, channels=64, causal=0, scale=0.125) | kw
        return C.byref(Packed(*a.values()))

    call = lambda p_, q=None, k=None, o=None: status("fvsr_packed_attention", ctx, p_, q or view(), k or view(2), k or view(2), o or view(),
                                                     None, 0, None, 0, None)
    for kw in ({"sequences": 0}, {"cu_q": None}, {"cu_k": None}, {"tokens_q": -1}, {"scale": 0.0}, {"scale": math.nan}):
        assert call(packed(**kw))[0] == _abi.ERR_INVALID_ARG, kw
    for kw in ({"channels": 60}, {"channels": 136}, {"tokens_k": 1 << 31}, {"tokens_q": 0x7ffffe00}, {"sequences": 1 << 21},
               {"scale": 1e-31}, {"scale": 1e31}):
        assert call(packed(**kw))[0] == _abi.ERR_UNSUPPORTED, kw
    assert call(packed(), k=view(3))[0] == _abi.ERR_INVALID_ARG
    assert call(packed(), q=view(data=24))[0] == _abi.ERR_INVALID_ARG
    assert call(packed(), q=view(ts=252))[0] == _abi.ERR_INVALID_ARG
    assert call(packed(), q=view(ts=1 << 23))[0] == _abi.ERR_UNSUPPORTED
    assert "workspace" in call(packed(tokens_k=60000))[1]      # few queries: the keys are split
    assert status("fvsr_packed_attention_backward", ctx, packed(), view(), view(), view(2), view(2), view(), None, view(), view(2), view(2), 0,
                  None, 0, None)[0] == _abi.ERR_INVALID_ARG
    rot = lambda tokens=4, ch=64, axes=(8, 8), k=None, ko=None: status(
        "fvsr_rotary", ctx, 1, view(), view(), k, ko, tokens, ch, p, 0, p, len(axes), (C.c_int32 * 4)(*axes), 0, 0, None)
    for kw in ({"tokens": -1}, {"ch": 63}, {"axes": ()}, {"axes": (1, 1, 1, 1)}, {"axes": (-1, 2)}, {"axes": (32, 1)}, {"k": view()}):
        assert rot(**kw)[0] == _abi.ERR_INVALID_ARG, kw
    assert rot(ch=1026)[0] == _abi.ERR_UNSUPPORTED


def test_workspaces():
    def size(**kw):
        a = dict(cu_q=16, cu_k=16, used_k=None, sequences=2, tokens_q=2, tokens_k=60000, channels=128, causal=0, scale=0.125) | kw
        return _abi.lib.fvsr_packed_attention_workspace(C.byref(Packed(*a.values())), 4, 2)
    assert size() > 0 and size(tokens_q=4000, tokens_k=4000) == 0 and size(tokens_k=600) == 0 and size(tokens_q=0) == 0
    assert 0 < size(channels=64) < size()

    def back(tq, tk, heads, seqs=1, causal=0, channels=128):
        p = Packed(16, 16, None, seqs, tq, tk, channels, causal, 0.125)
        return _abi.lib.fvsr_packed_attention_backward_workspace(C.byref(p), heads, heads) - tq * heads * 16
    block = (2 * 128 * 128 + 256) * 4      # a part's sums of a block of 128 keys
    assert back(17280, 17280, 12) == (137 * 12 - 6 * 256) * 3 * block      # what is left of 137 slots after six rounds, three parts each
    assert back(17280, 17280, 12, causal=1) == 0 and back(16384, 16384, 12) == 0 and back(17280, 17280, 12, seqs=6) == 0
    norm = _abi.lib.fvsr_rms_norm_backward_workspace      # none where one workgroup has all rows
    assert norm(128, 128) == norm(32, 512) == norm(8, 1536) == norm(1, 16384) == norm(0, 64) == 0 and norm(129, 128) == 5 * 128 * 4
    assert norm(2, 16384) == 0 and norm(3, 16384) == 2 * 16384 * 4
    assert back(4096, 1280, 1) == 12 * 8 * block and back(4096, 0, 1) == 0 and back(64, 64, 12) == 0


# ---- the plain forms against differences ---------------------------------------------------------------------------------
def test_rms_gradient_is_the_formulas():
    g = torch.Generator().manual_seed(1)
    x, w, dy, ds = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((3, 17), (17,), (3, 17), (3, 17)))
    _, _, rstd = rms64(x, None, w, 1e-3)
    dx, dw, _, _ = rms_grad64(dy, x, rstd, w, ds)
    f_ = lambda x, w: (rms64(x, None, w, 1e-3)[1] * dy).sum() + (x * ds).sum()
    for at, grad in ((0, dx), (1, dw)):
        v = [x, w]
        step = torch.randn(v[at].shape, generator=g, dtype=torch.float64)
        up, down = list(v), list(v)
        up[at], down[at] = v[at] + 1e-5 * step, v[at] - 1e-5 * step
        assert abs(float((f_(*up) - f_(*down)) / 2e-5 - (grad * step).sum())) < 1e-8


@pytest.mark.parametrize("causal", [False, True])
def test_attention_gradient_is_the_formulas(causal):
    g = torch.Generator().manual_seed(2)
    q, do = (torch.randn((7, 4, 8), generator=g, dtype=torch.float64) for _ in range(2))
    k, v = (torch.randn((9, 2, 8), generator=g, dtype=torch.float64) for _ in range(2))
    how = dict(cu_q=[0, 3, 7], cu_k=[0, 5, 9], causal=causal, used=[5, 3])
    r = attention64(q, k, v, do=do, **how)
    f_ = lambda q, k, v: (attention64(q, k, v, **how)["o"] * do).sum()
    for at, name in enumerate(("dq", "dk", "dv")):
        x = [q, k, v]
        step = torch.randn(x[at].shape, generator=g, dtype=torch.float64)
        up, down = list(x), list(x)
        up[at], down[at] = x[at] + 1e-5 * step, x[at] - 1e-5 * step
        assert abs(float((f_(*up) - f_(*down)) / 2e-5 - (r[name] * step).sum())) < 1e-8


def test_turning_back_is_the_gradient():
    g = torch.Generator().manual_seed(3)
    x, dy = (torch.randn((5, 2, 14), generator=g, dtype=torch.float64) for _ in range(2))
    how = (torch.randint(0, 99, (2, 5), generator=g), f.rotary_frequencies((3, 2), device="cpu"), (3, 2))
    for halves in (False, True):   # a linear map: <dy, A x> = <A^T dy, x>
        assert abs(float((dy * turn64(x, *how, halves)).sum() - (turn64(dy, *how, halves, back=True) * x).sum())) < 1e-12


def test_frequencies_and_positions():
    fr = f.rotary_frequencies((22, 21, 21), device="cpu")
    assert fr.dtype == torch.float64 and fr.shape == (64,) and float(fr[0]) == 1 == float(fr[22]) == float(fr[43])
    assert float(fr[11]) == pytest.approx(10000 ** -0.5)
    p = f.grid_positions(2, 3, 4, t0=7, device="cpu")
    assert p.dtype == torch.int32 and p.shape == (3, 24)
    assert p[:, 0].tolist() == [7, 0, 0] and p[:, 23].tolist() == [8, 2, 3] and p[:, 5].tolist() == [7, 1, 1]
