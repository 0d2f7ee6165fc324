"""CPU checks of the 8-bit training operators: what the binding and the C entry points refuse, before any device work."""
import ctypes as C

import pytest
import torch

import fvsr_lcsa as f
from fvsr_lcsa import _abi
from fvsr_lcsa.train8 import CODES, SCALES

E = f.FVSRError
bf = torch.bfloat16


def blocks(rows, features):
    return f.Blocks8.empty(rows, features, "cpu")


def test_blocks8_holds_whole_runs():
    q = blocks(5, 300)
    assert q.codes.shape == (5, 384) and q.scales.shape == (5, 4) and q.shape == (5, 300) and q.rows == 5
    assert _abi.lib.fvsr_blocks8_code_bytes(5, 300) == 5 * 384 and _abi.lib.fvsr_blocks8_scale_bytes(5, 300) == 20
    assert _abi.lib.fvsr_blocks8_scale_bytes(5, 513) == 40 and _abi.lib.fvsr_blocks8_code_bytes(0, 8) == 0
    for codes, scales, n in ((q.codes, q.scales, 385), (q.codes, q.scales, 256), (q.codes[:, :256], q.scales, 256),
                             (q.codes[:4], q.scales, 300), (q.codes.view(torch.uint8), q.scales, 300),
                             (q.codes, q.scales.view(torch.uint8), 300), (q.codes, q.scales, 0),
                             (torch.empty((384, 5), dtype=CODES).t(), q.scales, 300)):
        with pytest.raises(E, match="Blocks8"):
            f.Blocks8(codes, scales, n)


def test_quantize8_refusals():
    x = torch.zeros((4, 256), dtype=bf)
    for bad in (x.half(), x.to(torch.int32), x.t(), x[None].expand(2, 4, 256), torch.zeros(4), torch.zeros((4, 0)), None):
        with pytest.raises(E, match="x"):
            f.quantize8(bad)
    with pytest.raises(E, match="out"):
        f.quantize8(x, out=blocks(4, 128))
    with pytest.raises(E, match="HIP device"):
        f.quantize8(x)
    with pytest.raises(E, match="unsupported dtype"):
        f.dequantize8(blocks(4, 8), torch.float16)
    with pytest.raises(E, match="out"):
        f.dequantize8(blocks(4, 8), out=torch.zeros((4, 9), dtype=bf))
    with pytest.raises(E, match="HIP device"):
        f.dequantize8(blocks(4, 8))


def test_layer_norm_refusals():
    x, w = torch.zeros((4, 256), dtype=bf), torch.ones(256)
    for kw in ({"weight": w[:255]}, {"weight": w.half()}, {"weight": torch.ones(512)[::2]}):
        with pytest.raises(E, match="weight"):
            f.layer_norm(x, **kw)
    with pytest.raises(E, match="bias"):
        f.layer_norm(x, w, torch.zeros(257))
    for out in (x.float(), x[:3], torch.zeros((256, 4), dtype=bf).t()):
        with pytest.raises(E, match="out"):
            f.layer_norm(x, out=out)
    with pytest.raises(E, match="out"):
        f.layer_norm(x, quantized=True, out=blocks(4, 255))
    with pytest.raises(E, match="HIP device"):
        f.layer_norm(x, w)
    dy, st = torch.zeros((4, 256), dtype=bf), torch.zeros((4, 2))
    for args in ((dy, x.float(), st), (dy, x[:3], st), (dy, blocks(4, 255), st), (dy, x, st[:3]), (dy, x, st.double()),
                 (dy, x, torch.zeros((2, 4)).t()), (dy.half(), x, st)):
        with pytest.raises(E, match="x|stats|dy"):
            f.layer_norm_backward(*args)
    with pytest.raises(E, match="out"):
        f.layer_norm_backward(dy, x, st, out=dy.float())
    with pytest.raises(E, match="HIP device"):
        f.layer_norm_backward(dy, blocks(4, 256), st, w)


def test_linear8_refusals():
    x, w8 = torch.zeros((4, 256), dtype=bf), blocks(24, 256)
    with pytest.raises(E, match="Blocks8"):
        f.linear8(x, torch.zeros((24, 256), dtype=bf))
    for bad in (x[:, :128].contiguous(), blocks(4, 255)):
        with pytest.raises(E, match="weight expects 256"):
            f.linear8(bad, w8)
    with pytest.raises(E, match="at least one row"):
        f.linear8(x, blocks(0, 256))
    with pytest.raises(E, match="bias"):
        f.linear8(x, w8, torch.zeros(25))
    with pytest.raises(E, match="unsupported dtype"):
        f.linear8(x, w8, dtype=torch.float16)
    with pytest.raises(E, match="out"):
        f.linear8(x, w8, out=torch.zeros((4, 24)))
    with pytest.raises(E, match="HIP device"):
        f.linear8(blocks(4, 256), w8)
    dy = torch.zeros((4, 24), dtype=bf)
    with pytest.raises(E, match="dy"):
        f.linear8_weight_grad(dy.float(), blocks(4, 256))
    with pytest.raises(E, match="rows"):
        f.linear8_weight_grad(dy, blocks(5, 256))
    with pytest.raises(E, match="x8"):
        f.linear8_weight_grad(dy, x)
    with pytest.raises(E, match="out"):
        f.linear8_weight_grad(dy, blocks(4, 256), out=torch.zeros((24, 256), dtype=bf))
    with pytest.raises(E, match="HIP device"):
        f.linear8_weight_grad(dy, blocks(4, 256))


def _rc(name, *args):
    return getattr(_abi.lib, name)(*args), _abi.lib.fvsr_last_error().decode()


def test_c_entry_points_refuse_bad_arguments():
    """A NULL context, and with a context-shaped pointer (never read before the checks that fail here) bad sizes, types,
    alignments and workspaces."""
    inv, uns = _abi.ERR_INVALID_ARG, _abi.ERR_UNSUPPORTED
    mem = C.create_string_buffer(4096)
    p = (C.addressof(mem) + 255) & ~255
    ctx = p
    F32, BF = _abi.DTYPE_F32, _abi.DTYPE_BF16
    assert _rc("fvsr_quantize8", None, F32, p, 1, 8, p, p, None) == (inv, "ctx is NULL")
    assert _rc("fvsr_quantize8", ctx, 7, p, 1, 8, p, p, None)[0] == inv
    assert _rc("fvsr_quantize8", ctx, F32, p, -1, 8, p, p, None)[0] == inv
    assert _rc("fvsr_quantize8", ctx, F32, p, 1, 0, p, p, None)[0] == inv
    assert _rc("fvsr_quantize8", ctx, F32, p, 1, (1 << 20) + 1, p, p, None)[0] == uns
    assert _rc("fvsr_quantize8", ctx, F32, None, 1, 8, p, p, None)[0] == inv
    assert _rc("fvsr_quantize8", ctx, F32, p, 1, 8, p + 8, p, None)[0] == inv
    assert _rc("fvsr_quantize8", ctx, F32, p, 1, 8, p, p + 2, None)[0] == inv
    assert _rc("fvsr_quantize8", ctx, F32, None, 0, 8, None, None, None)[0] == _abi.OK          # no rows: nothing to do
    assert _rc("fvsr_dequantize8", ctx, p, p, 1, 8, F32, None, None)[0] == inv
    assert _rc("fvsr_dequantize8", ctx, None, p, 1, 8, F32, p, None)[0] == inv
    ln = lambda *a: _rc("fvsr_layer_norm", *a)  # noqa: E731
    assert ln(ctx, BF, p, 1, 16385, 1e-6, F32, None, None, p, None, None, None, None, None, None)[0] == uns
    assert ln(ctx, BF, p, 1, 8, -1.0, F32, None, None, p, None, None, None, None, None, None)[0] == inv
    assert ln(ctx, BF, p, 1, 8, float("nan"), F32, None, None, p, None, None, None, None, None, None)[0] == inv
    assert ln(ctx, F32, p, 1, 8, 1e-6, BF, p, None, p, None, None, None, None, None, None)[0] == inv
    assert ln(ctx, BF, p, 1, 8, 1e-6, F32, None, None, None, None, None, p, p, p, None)[0] == inv
    assert ln(ctx, BF, p, 1, 8, 1e-6, F32, None, None, None, p, None, None, None, None, None)[0] == inv
    bw = lambda *a: _rc("fvsr_layer_norm_backward", *a)  # noqa: E731
    need = _abi.lib.fvsr_layer_norm_backward_workspace(3, 8)
    assert need > 0
    assert bw(ctx, BF, p, p, p, p, p, 3, 8, F32, None, p, None, None, None, 0, None)[0] == inv      # both x and x_codes
    assert bw(ctx, BF, p, None, None, None, p, 3, 8, F32, None, p, None, None, None, 0, None)[0] == inv
    assert bw(ctx, BF, p, p, None, None, p, 3, 8, F32, None, p, p, None, None, 0, None)[0] == inv
    assert bw(ctx, BF, p, p, None, None, p, 3, 8, F32, None, p, p, None, p, need - 1, None)[0] == inv
    assert bw(ctx, BF, p, p, None, None, p, 3, 8, F32, None, p, p, None, p + 4, need, None)[0] == inv
    li = lambda *a: _rc("fvsr_linear8", *a)  # noqa: E731
    assert li(ctx, BF, p, 1, 8, p, p, p, p, 0, F32, None, 0, BF, p, p, 1 << 20, None)[0] == inv
    assert li(ctx, 9, p, 1, 8, p, p, p, p, 8, F32, None, 0, BF, p, p, 1 << 20, None)[0] == inv
    assert li(ctx, BF, p, 1, 8, p, p, p, p, 8, 9, p, 0, BF, p, p, 1 << 20, None)[0] == inv
    assert li(ctx, BF, p, 1, 8, p, p, p, p, 8, F32, None, 0, 9, p, p, 1 << 20, None)[0] == inv
    assert li(ctx, BF, p, 1, 8, None, p, p, p, 8, F32, None, 0, BF, p, p, 1 << 20, None)[0] == inv
    assert li(ctx, BF, p, 1, 8, p, p, p, None, 8, F32, None, 0, BF, p, p, 1 << 20, None)[0] == inv
    assert li(ctx, BF, p, 1, 8, p, p, p, p, 8, F32, None, 0, BF, None, p, 1 << 20, None)[0] == inv
    wg = lambda *a: _rc("fvsr_linear8_weight_grad", *a)  # noqa: E731
    assert wg(ctx, p, 1, 8, p, p, 8, F32, None, None, p, 1 << 20, None)[0] == inv
    assert wg(ctx, None, 1, 8, p, p, 8, F32, p, None, p, 1 << 20, None)[0] == inv
    assert wg(ctx, p, 1, 0, p, p, 8, F32, p, None, p, 1 << 20, None)[0] == inv
    need = _abi.lib.fvsr_linear8_weight_grad_workspace(1, 8, 8)
    if need:
        assert wg(ctx, p, 1, 8, p, p, 8, F32, p, p, p, need - 1, None)[0] == inv


def test_c_weight_gradient_wants_whole_rows_aligned():
    """dY's rows are copied 16 bytes at a time where they are whole 16 bytes: then it starts at a multiple of 16."""
    mem = C.create_string_buffer(4096)
    p = (C.addressof(mem) + 255) & ~255
    rc, msg = _rc("fvsr_linear8_weight_grad", p, p + 2, 1, 8, p, p, 8, _abi.DTYPE_F32, p, None, p, 1 << 20, None)
    assert rc == _abi.ERR_INVALID_ARG and "16-byte aligned" in msg
