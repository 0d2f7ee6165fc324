"""The 8-bit training operators at the edges of their ranges, against float64 plain forms (tolerances as in test_gpu_train8.py)."""
import math

import pytest
import torch

import fvsr_lcsa as f
from test_gpu_train8 import check_norm_grad, gen_of
from train8_reference import U, quantize64, within

pytestmark = pytest.mark.gpu
bf, f32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [bf, f32])
@pytest.mark.parametrize("c", [1, 5, 8, 9, 120, 200, 203, 520, 1000, 1031, 1544, 1999, 2056, 4100, 8200, 16376])
def test_layer_norm_backward_of_rows_of_one_large_value(dev, dtype, c):
    """Rows of equal values whose mean times 1 / standard deviation passes fp32's largest number (2^109 * 10^6): every channel's normed
    value is 0 all the same, also where lanes of the team lie past the row's end. Sums of equal powers of two are exact, so the
    statistics are."""
    rows, eps = 11, 1e-12
    g = gen_of(c, 21)
    x = torch.full((rows, c), 2.0 ** 109, dtype=dtype, device=dev)
    x[1::2] *= -1
    dy = torch.randn((rows, c), generator=g).to(dtype).to(dev)
    w, b = torch.randn(c, generator=g).to(dev), torch.randn(c, generator=g).to(dev)
    y, stats, x8 = f.layer_norm(x, w, b, eps, want_stats=True, want_x8=True)
    assert torch.equal(stats[:, 0], x[:, 0].float()) and torch.equal(y, b.to(dtype).expand(rows, c))
    within(stats[:, 1:], torch.full((rows, 1), 1e6, dtype=torch.float64, device=dev), 48 * U * 1e6, "rstd")   # variance 0
    for kept in (x, x8):
        for weight in (w, None):
            dx, dw, db = f.layer_norm_backward(dy, kept, stats, weight)
            assert not dw.any()
            check_norm_grad(dy, x, stats, weight, dx, dw, db)


@pytest.mark.parametrize("dtype", [bf, f32])
def test_the_largest_numbers_come_back_finite(dev, dtype):
    """Finite values from 240 * 2^120 up to the type's largest are kept as 240 * 2^120 (256 would stand for 2^128), within 2^-4 of what
    they were: in a tensor's own pass, in the norm's, and in what the products make of them. Infinities stay NaN, neighbours as they are."""
    top = 240 * 2.0 ** 120
    near = [240.0, 244.0, 247.0, 248.0, 249.0, 252.0, 255.0] + ([] if dtype == bf else [247.9999, 248.0001, 255.99998])
    vals = torch.tensor([v * 2.0 ** 120 for v in near] + [torch.finfo(dtype).max, 1.1 * 2.0 ** 127, 2.0 ** 100], dtype=torch.float64)
    rows = 2 * len(vals)
    x = torch.randn((rows, 300), generator=gen_of(31), dtype=torch.float64) * 2.0 ** 118
    for i, v in enumerate(vals):
        x[2 * i, 17], x[2 * i + 1, 299] = v, -v
    x = x.to(dtype).to(dev)
    assert x.isfinite().all()
    want = quantize64(x)[0].clamp(-top, top)
    largest = torch.nn.functional.pad(x.double().abs(), (0, 84)).reshape(rows, 3, 128).amax(2).repeat_interleave(128, 1)[:, :300]
    bound = torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -17 * largest)
    for q in (f.quantize8(x), f.layer_norm(x, want_x8=True)[2]):
        back = f.dequantize8(q, dtype)
        assert back.isfinite().all() and torch.equal(back.double(), want)
        assert ((back.double() - x.double()).abs() <= bound).all()
        assert q.codes.view(torch.uint8)[0, 17] == 0x77 and q.scales.view(torch.uint8)[0, 0] == 247
    # 2^-20 times one channel: the products see the same values
    for ch in (17, 299):
        w = torch.zeros((16, 300), dtype=bf, device=dev)
        w[3, ch] = 2.0 ** -20
        y = f.linear8(x, f.quantize8(w), dtype=f32)
        assert torch.equal(y[:, 3].double(), want[:, ch] * 2.0 ** -20) and not y[:, :3].any() and not y[:, 4:].any()
    dy = torch.zeros((rows, 8), dtype=bf, device=dev)
    dy[2, 5] = 2.0 ** -20
    dw = f.linear8_weight_grad(dy, f.quantize8(x))[0]
    assert torch.equal(dw[5].double(), want[2] * 2.0 ** -20)
    x[0, 18], x[0, 19] = math.inf, -math.inf
    q = f.quantize8(x)
    back = f.dequantize8(q, f32)
    assert back[0, 18:20].isnan().all() and back.isnan().sum() == 2 and back[0, 17] == top
