"""The 8-bit training operators at the edges of their ranges, against float64 plain forms (tolerances as in test_gpu_train8.py)."""
import pytest
import torch

import fvsr_lcsa as f
from test_gpu_train8 import check_norm_grad, gen_of
from train8_reference import U, within

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
