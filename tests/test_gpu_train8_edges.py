"""The 8-bit training operators at the edges of their ranges, against float64 plain forms (tolerances as in test_gpu_train8.py)."""
import math

import pytest
import torch

import fvsr_lcsa as f
from test_gpu_train8 import check_norm_grad, gen_of, unaligned
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


# ---- sums of small whole numbers: exact in fp32 in any order, so results are equal, not close -------------------------------------------
CODES = (0x00, 0x38, 0x40, 0x44, 0x48, 0xb8, 0xc0, 0xc4)   # 0, 1, 2, 3, 4, -1, -2, -3 in e4m3


def whole_blocks(gen, rows, features, dev):
    """An 8-bit matrix of whole numbers from -3 to 4 under the scale 1."""
    q = f.Blocks8.empty(rows, features, dev)
    codes = torch.tensor(CODES, dtype=torch.uint8)[torch.randint(0, 8, (rows, features), generator=gen)]
    q.codes.view(torch.uint8).zero_()
    q.codes.view(torch.uint8)[:, :features] = codes.to(dev)
    q.scales.view(torch.uint8).zero_()
    q.scales.view(torch.uint8)[:, :-(-features // 128)] = 127
    return q


def whole(gen, shape, dtype, dev):
    return torch.randint(-3, 4, shape, generator=gen).to(dtype).to(dev)


@pytest.mark.parametrize("rows,k,n", [(1, 128, 8), (63, 300, 17), (777, 523, 270), (1000, 136, 200), (2048, 256, 512), (5000, 256, 264),
                                      (20000, 300, 520), (4000, 300, 1501), (9000, 1400, 5700), (129, 1000, 4200)])
def test_weight_gradients_of_whole_numbers(dev, rows, k, n):
    """dW and db, every element: at most 20000 products of at most 12, below 2^24."""
    g = gen_of(rows, k, n, 41)
    x8, dy = whole_blocks(g, rows, k, dev), whole(g, (rows, n), bf, dev)
    want, bias = dy.double().t() @ f.dequantize8(x8, f32).double(), dy.double().sum(0)
    for d in (dy, unaligned(dy)):
        dw, db = f.linear8_weight_grad(d, x8)
        assert torch.equal(dw.double(), want) and torch.equal(db.double(), bias)
    assert rows == 1 or (bias != 0).any()


def test_weight_gradients_of_whole_numbers_past_32_bits(dev):
    """More than 2^32 bytes of 8-bit tokens, every token's share in dW and db: 262444 products of at most 12, below 2^24."""
    k, n = 16384, 24
    rows = (1 << 32) // k + 300
    g = gen_of(43)
    block = whole_blocks(g, 4099, k, dev)
    x8 = f.Blocks8.empty(rows, k, dev)
    for at in range(0, rows, 4099):
        m = min(4099, rows - at)
        x8.codes[at:at + m], x8.scales[at:at + m] = block.codes[:m], block.scales[:m]
    dy = whole(g, (rows, n), bf, dev)
    dw, db = f.linear8_weight_grad(dy, x8)
    assert torch.equal(db.double(), dy.double().sum(0))
    # the tokens of one place in the repeated block are equal: dW = (sum of their dY)^T block
    folded = torch.nn.functional.pad(dy.double(), (0, 0, 0, -rows % 4099)).reshape(-1, 4099, n).sum(0)
    assert torch.equal(dw.double(), folded.t() @ f.dequantize8(block, f32).double())
    y = f.linear8(x8, whole_blocks(g, n, k, dev), dtype=f32)
    at = rows // 4099 * 4099
    assert torch.equal(y[:4099], y[4099:8198]) and torch.equal(y[at:], y[:rows - at]) and torch.equal(y[at - 4099:at], y[:4099])


@pytest.mark.parametrize("rows,k,n", [(1, 1536, 1536), (5, 130, 17), (33, 700, 100), (64, 2000, 300), (100, 1536, 264), (512, 4096, 520),
                                      (777, 523, 270), (2900, 1100, 2840), (3001, 260, 3003)])
def test_products_of_whole_numbers(dev, rows, k, n):
    """Few tokens, tiles, tiles whose depth is cut into parts, large tiles: products of at most 16, of which the matrix cores cut nothing
    (multiples of 2^(E - 13), E <= 4), sums below 2^24."""
    g = gen_of(rows, k, n, 47)
    x8, w8, b = whole_blocks(g, rows, k, dev), whole_blocks(g, n, k, dev), whole(g, (n,), f32, dev)
    want = f.dequantize8(x8, f32).double() @ f.dequantize8(w8, f32).double().t()
    assert torch.equal(f.linear8(x8, w8, dtype=f32).double(), want)
    assert torch.equal(f.linear8(x8, w8, b, dtype=f32).double(), want + b.double())
    assert torch.equal(f.linear8(x8, w8, b.to(bf)), (want + b.double()).to(bf))


@pytest.mark.parametrize("rows,c", [(1, 8), (777, 523), (20000, 300), (2500, 2047), (4100, 4101), (700, 16384)])
@pytest.mark.parametrize("dtype", [bf, f32])
def test_bias_gradients_of_norms_of_whole_numbers(dev, dtype, rows, c):
    g = gen_of(rows, c, 53)
    x, dy = torch.randn((rows, c), generator=g).to(dtype).to(dev), whole(g, (rows, c), dtype, dev)
    _, stats, x8 = f.layer_norm(x, want_stats=True, want_x8=True)
    for kept in (x, x8):
        assert torch.equal(f.layer_norm_backward(dy, kept, stats)[2].double(), dy.double().sum(0))
