"""The 8-bit training operators against float64 plain forms (tests/train8_reference.py).

Tolerances, per value, with U = 2^-24 (half a step of fp32) and h half a step of the output's type (2^-8 bf16, 2^-24 fp32):
  8-bit codes and scales, and values brought back: equal (the scale is a power of two, so nothing is rounded but the code)
  layer norm: h |y| for the output; a sum over a row adds at most 32 values in a lane, then over 64 lanes and 16 waves pairwise or in
      order: its error is below 64 U of the sum of magnitudes. The mean is thus off by 64 U mean|x|, which moves n by that times
      rstd; the variance by about 64 U of itself, rstd by 40 U; with the last products and sums below 64 U |n w| + 4 U |b|
  its gradient (stats are inputs): n is off by 3 U |n| + U rstd |mean|-sized roundings of x - mean (U rstd |x - mean| = U |n|) and of
      the product: 4 U |n|; m1 and m2 by 70 U of their sums of magnitudes over C: with the rest below 80 U rstd (|g| + mean|g| +
      |n| mean|g n|), plus h |dx|; dweight and dbias: at most rows / 2048 + 8 values in a lane, 4 waves, 32 workgroups' parts in a
      thread, 16 threads: below (rows / 2048 + 160) U of the sum of magnitudes
  weight gradients: exact factors, products added in some order, each addition at most U of the sum of magnitudes: (rows + 8) U
      sum |a b|, plus h |dW|
  8-bit products: the matrix cores add the products of 8 neighbouring channels after cutting each to a multiple of 2^(E - 13), E the
      largest sum of the two codes' exponents in the 8 (-6 below the normal codes) plus the scales'; what 8 products lose is below 8 *
      2^(E - 13), and 2^E at most the product of the larger of each side's largest value and 2^-6 of its scale: so the 8 are off by
      less than 2^-10 times that. Those sums are added in fp32: (K + 8) U sum |a b| as above, plus h |y|. (That cut, bit for bit,
      is what one instruction gave for 102,400 random sums of 8 products.) GELU has a slope below 1.13, its exponential (argument
      A) and reciprocal an error below (16 + 4 |A|) U
"""
import math

import pytest
import torch

import fvsr_lcsa as f
from train8_reference import HALF, RUN, U, gelu64, norm64, norm_grad64, quantize64, within

pytestmark = pytest.mark.gpu
bf, f32 = torch.bfloat16, torch.float32


def tokens(gen, rows, c, dtype, dev):
    """Channels of different gains and means, a few large; a row of zeros and one of equal values among them."""
    x = torch.randn((rows, c), generator=gen) * torch.exp(torch.randn(c, generator=gen)) + torch.randn(c, generator=gen)
    if c > 3:
        x[:, 3] *= 30
    if rows > 2:
        x[1] = 0
        x[2] = 1.75
    return x.to(dtype).to(dev)


def gen_of(*seed):
    return torch.Generator().manual_seed(hash(seed) % (1 << 31))


def values(q):
    runs = q.codes.shape[1] // RUN
    v = q.codes.double().reshape(q.rows, runs, RUN) * q.scales[:, :runs, None].double()
    return v.reshape(q.rows, -1)


def unaligned(x):
    """The same tokens at an address that is a multiple of the element size only."""
    flat = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)
    v = flat[1:].view(x.shape)
    v.copy_(x)
    return v


def check_blocks(q, x, what=""):
    """q is x in 8 bits, bit for bit, its padding zeros."""
    want, e = quantize64(x)
    v = values(q)
    c = x.shape[1]
    assert torch.equal(v[:, :c].nan_to_num(7e77), want.nan_to_num(7e77)), what
    assert torch.equal(q.scales.view(torch.uint8)[:, :e.shape[1]].long(), e.long() + 127), what
    assert not q.codes.view(torch.uint8)[:, c:].any() and not q.scales.view(torch.uint8)[:, e.shape[1]:].any(), what


# ---- 8-bit activations ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [bf, f32])
@pytest.mark.parametrize("rows,c", [(1, 1), (3, 7), (5, 8), (2, 127), (17, 128), (4, 129), (33, 520), (9, 1003), (130, 1536)])
def test_quantize8_and_back(dev, dtype, rows, c):
    x = tokens(gen_of(rows, c), rows, c, dtype, dev)
    for t in (x, unaligned(x)):
        q = f.quantize8(t)
        check_blocks(q, x)
        for to in (bf, f32):
            back = f.dequantize8(q, to)
            assert torch.equal(back, quantize64(x)[0].to(to))
            o = unaligned(torch.zeros((rows, c), dtype=to, device=dev))
            assert f.dequantize8(q, to, out=o) is o and torch.equal(o, back)


@pytest.mark.parametrize("dtype", [bf, f32])
def test_quantize8_of_special_values(dev, dtype):
    """Every bf16 magnitude's border: powers of two, 448 * 2^e and its neighbours, ties, the smallest and largest numbers; infinities
    and NaN become NaN and leave the scale to the others; a run with nothing finite."""
    tops = torch.tensor([2.0 ** e for e in range(-133, 128, 9)] + [448 * 2.0 ** e for e in (-130, -40, -8, 0, 9, 100)])
    x = torch.zeros((3 * len(tops), 256))
    for i, t in enumerate(tops):
        for j, s in enumerate((1.0, 1 + 2.0 ** -7, 1 - 2.0 ** -8)):
            x[3 * i + j, 5] = (t * s).clamp(max=3.38e38)
            x[3 * i + j, 6:130] = t * torch.linspace(-1, 1, 124)
            x[3 * i + j, 200] = t * 2.0 ** -9
            x[3 * i + j, 130:140] = t * (1 + torch.arange(10) / 16) / 2
    x[0, 9], x[1, 9], x[2, 9], x[4, 128:] = math.inf, -math.inf, math.nan, math.nan
    x = x.to(dtype).to(dev)
    check_blocks(f.quantize8(x), x)
    v = f.dequantize8(f.quantize8(x), f32)
    assert v[0, 9].isnan() and v[1, 9].isnan() and v[4, 128:].isnan().all() and v.isnan().sum() == 3 + 128


def test_quantize8_past_32_bits(dev):
    """More than 2^32 bytes of codes and 2^31 elements: the last rows are what they are alone."""
    rows, c = (1 << 32) // 8192 + 5, 8192
    x = torch.zeros((rows, c), dtype=bf, device=dev)
    tail = tokens(gen_of(1), 7, c, bf, dev)
    x[-7:] = tail
    q = f.quantize8(x)
    check_blocks(f.Blocks8(q.codes[-7:], q.scales[-7:], c), tail)
    assert torch.equal(f.dequantize8(q, out=x)[-7:], f.dequantize8(f.quantize8(tail)))


# ---- layer norm -------------------------------------------------------------------------------------------------------
NORM_SHAPES = [(1, 1), (5, 7), (3, 128), (6, 513), (9, 1003), (40, 1536), (3, 2048), (2, 2049), (4, 4096), (3, 5000), (2, 8192),
               (2, 8193), (2, 16384)]


def check_norm(x, w, b, y, stats, eps):
    want, mean, rstd = norm64(x, w, b, eps)
    n = (x.double() - mean) * rstd
    wd = torch.ones(1, device=x.device).double() if w is None else w.double().abs()
    dn = 64 * U * (x.double().abs().mean(1, keepdim=True) * rstd + n.abs())
    tol = dn * wd + 4 * U * (0 if b is None else b.double().abs()) + HALF[y.dtype] * want.abs()
    within(y, want, tol * (1 + 2.0 ** -7), "y")
    if stats is not None:
        within(stats[:, :1], mean, 66 * U * x.double().abs().mean(1, keepdim=True), "mean")
        # a variance of nearly 0 (rows of equal values) is the square of the mean's own error at most
        off = (66 * U * x.double().abs().mean(1, keepdim=True)) ** 2 * rstd ** 3
        within(stats[:, 1:], rstd, 48 * U * rstd + off, "rstd")


@pytest.mark.parametrize("dtype", [bf, f32])
@pytest.mark.parametrize("rows,c", NORM_SHAPES)
def test_layer_norm(dev, dtype, rows, c):
    g = gen_of(rows, c, 2)
    x = tokens(g, rows, c, dtype, dev)
    w, b = torch.randn(c, generator=g).to(dev), torch.randn(c, generator=g).to(dev)
    for i, (ww, bb, t) in enumerate([(None, None, x), (w, b, x), (w.to(bf), b.to(bf), unaligned(x)), (w, b.to(bf), unaligned(x)),
                                     (None, b, x), (w.to(bf), None, x)]):
        print(f"  layer_norm {dtype} {rows} x {c} variant {i}", flush=True)
        y, stats, x8 = f.layer_norm(t, ww, bb, 1e-5, want_stats=True, want_x8=True)
        check_norm(x, ww, bb, y, stats, 1e-5)
        check_blocks(x8, x, "x8")
        y8, none, none8 = f.layer_norm(t, ww, bb, 1e-5, quantized=True)
        assert none is None and none8 is None
        # from the 32-bit values, which the fp32 tokens' y is; of bf16 tokens y is their rounding: compare through fp32 tokens
        if dtype == f32:
            assert torch.equal(values(y8), values(f.quantize8(y)))
        else:
            y32 = f.layer_norm(x.float(), ww, bb, 1e-5)[0]
            assert torch.equal(values(y8), values(f.quantize8(y32)))


def test_layer_norm_of_rows_with_nan_and_infinity(dev):
    """A NaN or infinity takes its own row, and nothing of the padding or of other rows; dweight only where its channel is."""
    x = tokens(gen_of(4), 9, 200, f32, dev)
    x[3, 5], x[6, 7] = math.nan, math.inf
    w, b = torch.ones(200, device=dev), torch.ones(200, device=dev)
    y, stats, x8 = f.layer_norm(x, w, b, want_stats=True, want_x8=True)
    bad = torch.tensor([3, 6], device=dev)
    rest = torch.tensor([0, 1, 2, 4, 5, 7, 8], device=dev)
    assert y[bad].isnan().all() and not y[rest].isnan().any()
    y8 = f.layer_norm(x, w, b, quantized=True)[0]
    assert not y8.codes.view(torch.uint8)[:, 200:].any()
    assert torch.equal(y8.codes.float().isnan()[:, :200], y.isnan())
    alone = f.layer_norm(x[rest].contiguous(), w, b)[0]
    assert torch.equal(y[rest], alone)


def check_norm_grad(dy, x, stats, w, dx, dw, db):
    rows = dy.shape[0]
    wx, ww, wb, n = norm_grad64(dy, x, stats, w)
    g = (dy.double() if w is None else dy.double() * w.double()).abs()
    n, rstd = n.abs(), stats[:, 1:].double()
    tol = 80 * U * rstd * (g + g.mean(1, keepdim=True) + n * (g * n).mean(1, keepdim=True)) + HALF[dx.dtype] * wx.abs()
    within(dx, wx, tol * (1 + 2.0 ** -7), "dx")
    k = (rows / 2048 + 160) * U
    if dw is not None:
        within(dw, ww, (k + 4 * U) * (dy.double().abs() * n).sum(0), "dweight")
        within(db, wb, k * dy.double().abs().sum(0), "dbias")


@pytest.mark.parametrize("dtype", [bf, f32])
@pytest.mark.parametrize("rows,c", NORM_SHAPES + [(2500, 136)])
def test_layer_norm_backward(dev, dtype, rows, c):
    g = gen_of(rows, c, 3)
    x = tokens(g, rows, c, dtype, dev)
    dy = torch.randn((rows, c), generator=g).to(dtype).to(dev)
    w = torch.randn(c, generator=g).to(dev)
    _, stats, x8 = f.layer_norm(x, want_stats=True, want_x8=True)
    for ww, kept, u in ((w, x, False), (w.to(bf), x8, False), (None, x8, True), (w, x, True)):
        print(f"  layer_norm_backward {dtype} {rows} x {c} 8-bit {kept is x8} unaligned {u}", flush=True)
        d = unaligned(dy) if u else dy
        k = unaligned(kept) if u and kept is x else kept
        dx, dw, db = f.layer_norm_backward(d, k, stats, ww)
        check_norm_grad(dy, x if kept is x else quantize64(x)[0], stats, ww, dx, dw, db)
        again = f.layer_norm_backward(d, k, stats, ww)
        assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))
        only, none, none2 = f.layer_norm_backward(d, k, stats, ww, want_params=False)
        assert torch.equal(only, dx) and none is None and none2 is None
    same = dy.clone()
    assert f.layer_norm_backward(same, x, stats, w, out=same)[0] is same
    assert torch.equal(same, f.layer_norm_backward(dy, x, stats, w)[0])


@pytest.mark.parametrize("dtype", [bf, f32])
@pytest.mark.parametrize("c", [2, 5, 9, 15, 121, 130, 135, 385, 1031, 1537, 2047, 2049, 4100, 8195, 16383])
def test_layer_norm_backward_of_odd_rows(dev, dtype, c):
    """Rows whose last 8 channels straddle two lanes, runs, waves."""
    rows = 21
    g = gen_of(rows, c, 5)
    x = tokens(g, rows, c, dtype, dev)
    dy = torch.randn((rows, c), generator=g).to(dtype).to(dev)
    w = torch.randn(c, generator=g).to(dtype).to(dev)
    _, stats, x8 = f.layer_norm(x, want_stats=True, want_x8=True)
    for kept in (x, x8):
        dx, dw, db = f.layer_norm_backward(dy, kept, stats, w)
        check_norm_grad(dy, x if kept is x else quantize64(x)[0], stats, w, dx, dw, db)
    same = dy.clone()
    f.layer_norm_backward(same, x8, stats, w, out=same)
    assert torch.equal(same, dx)


def test_layer_norm_backward_of_neighbouring_runs(dev):
    """A row's last channel alone in a run of 2^-127's scale, beside a run of the largest one: neither reaches the other."""
    x = torch.ones((4, 129), device=dev)
    x[1, :128], x[1, 128] = 1.2e19, 0
    x[2, 128] = 3e38
    dy = torch.randn((4, 129), generator=gen_of(3)).to(dev)
    x8 = f.quantize8(x)
    stats = torch.tensor([[0.0, 1e-25]], device=dev).repeat(4, 1)
    dx, dw, db = f.layer_norm_backward(dy, x8, stats)
    check_norm_grad(dy, quantize64(x)[0], stats, None, dx, dw, db)


def test_nothing_is_written_past_the_ends(dev):
    """Results of odd widths in the middle of a larger buffer, whose other elements stay as they were."""
    rows, k, n = 133, 261, 267

    def ends(call, shape, dtype):
        size = shape[0] * shape[1]
        buf = torch.full((size + 64,), 7.5, dtype=dtype, device=dev)
        call(buf[31:31 + size].view(shape))
        assert (buf[:31] == 7.5).all() and (buf[31 + size:] == 7.5).all() and not (buf[31:31 + size] == 7.5).all()

    for dtype in (bf, f32):
        x = tokens(gen_of(8), rows, k, dtype, dev)
        x8, w8 = f.quantize8(x), f.quantize8(tokens(gen_of(9), n, k, bf, dev))
        _, stats, _ = f.layer_norm(x, want_stats=True)
        dy = tokens(gen_of(10), rows, n, bf, dev)
        ends(lambda o: f.layer_norm(x, out=o), (rows, k), dtype)
        ends(lambda o: f.layer_norm_backward(x, x8, stats, out=o), (rows, k), dtype)
        ends(lambda o: f.dequantize8(x8, dtype, out=o), (rows, k), dtype)
        ends(lambda o: f.linear8_weight_grad(dy, x8, dtype, out=o), (n, k), dtype)
        for m in (3, 70, rows):
            q = f.Blocks8(x8.codes[:m], x8.scales[:m], k)
            ends(lambda o: f.linear8(q, w8, dtype=dtype, out=o), (m, n), dtype)
        many = f.quantize8(tokens(gen_of(11), 2900, k, bf, dev))
        wide = f.quantize8(tokens(gen_of(12), 3001, k, bf, dev))
        ends(lambda o: f.linear8(many, wide, dtype=dtype, out=o), (2900, 3001), dtype)


def test_layer_norm_backward_against_differences(dev):
    """Directional derivatives of sum(dy * layer_norm(x, w, b)) by central differences of the float64 plain form, h = 1e-6 relative:
    their own error is of the order h^2 and 1e-16 / h, below 1e-8; the kernel's fp32 sums over 300 x 96 terms below 1e-4 of their
    magnitude."""
    g = gen_of(11)
    x, dy = torch.randn((300, 96), generator=g, dtype=torch.float64), torch.randn((300, 96), generator=g, dtype=torch.float64)
    w, b = torch.randn(96, generator=g, dtype=torch.float64), torch.randn(96, generator=g, dtype=torch.float64)
    x, dy, w, b = (t.float().double().to(dev) for t in (x, dy, w, b))
    stats = f.layer_norm(x.float(), want_stats=True)[1]
    dx, dw, db = f.layer_norm_backward(dy.float(), x.float(), stats, w.float())
    loss = lambda *a: float((dy * norm64(*a)[0]).sum())  # noqa: E731
    h = 1e-6
    for grad, at in ((dx, 0), (dw, 1), (db, 2)):
        v = torch.randn(grad.shape, generator=g, dtype=torch.float64).to(dev)
        up, down = [[t + s * h * v if i == at else t for i, t in enumerate((x, w, b))] for s in (1, -1)]
        slope = (loss(*up) - loss(*down)) / (2 * h)
        assert abs(float((grad.double() * v).sum()) - slope) < 1e-4 * float((grad.double() * v).abs().sum())


# ---- linear layers ----------------------------------------------------------------------------------------------------
LINEAR_SHAPES = [(1, 1, 1), (1, 128, 8), (2, 37, 5), (3, 300, 17), (16, 256, 64), (17, 129, 130), (64, 512, 128), (100, 640, 250),
                 (129, 1003, 129), (300, 384, 257), (513, 768, 520), (1, 1536, 9216), (5, 2000, 1000), (700, 4096, 300)]


def linear_case(rows, k, n, dev):
    g = gen_of(rows, k, n)
    x = tokens(g, rows, k, bf, dev)
    w = (torch.randn((n, k), generator=g) / math.sqrt(k)).to(bf).to(dev)
    b = torch.randn(n, generator=g).to(dev)
    return g, x, w, b


def eights(v):
    """Of each 8 neighbouring channels the larger of the largest magnitude and 2^-6 of their scale; v: 8-bit values in float64."""
    v = torch.nn.functional.pad(v.abs().nan_to_num(0.0), (0, -v.shape[1] % RUN))
    _, e = quantize64(v)     # the values' own scale: that of what they came from, or half of it where rounding reached 448
    scale = 2 * torch.exp2(e.double() - 6).repeat_interleave(RUN // 8, 1)
    return torch.maximum(v.reshape(v.shape[0], -1, 8).amax(-1), scale)


def product_off(a, w):
    return (a.shape[1] + 8) * U * (a.abs() @ w.abs().t()) + 2.0 ** -10 * (eights(a) @ eights(w).t())


def check_linear(y, a, w, b, gelu):
    """a, w: the 8-bit values in float64"""
    s = a @ w.t()
    off = product_off(a, w)
    if b is not None:
        s = s + b.double()
        off = off + 2 * U * (s.abs() + b.double().abs())
    want = s
    if gelu:
        want = gelu64(s)
        arg = 2 * math.sqrt(2 / math.pi) * (s + 0.044715 * s ** 3).abs() / math.log(2)
        off = 1.13 * off + (16 + 4 * arg) * U * want.abs() + 1e-30
    within(y, want, (off + HALF[y.dtype] * want.abs()) * (1 + 2.0 ** -7), "y")


@pytest.mark.parametrize("rows,k,n", LINEAR_SHAPES)
def test_linear8(dev, rows, k, n):
    _, x, w, b = linear_case(rows, k, n, dev)
    w8, x8 = f.quantize8(w), f.quantize8(x)
    a64, w64 = quantize64(x)[0], quantize64(w)[0]
    for bias, gelu, dtype, given in ((None, False, f32, x), (b, False, bf, x8), (b.to(bf), True, bf, x8), (b, True, f32, x8)):
        print(f"  linear8 {rows} x {k} x {n} gelu {gelu} {dtype} 8-bit x {given is x8}", flush=True)
        y = f.linear8(given, w8, bias, gelu=gelu, dtype=dtype)
        check_linear(y, a64, w64, bias, gelu)
        o = unaligned(torch.zeros((rows, n), dtype=dtype, device=dev))
        assert f.linear8(given, w8, bias, gelu=gelu, dtype=dtype, out=o) is o and torch.equal(o, y)
    assert torch.equal(f.linear8(x, w8, b), f.linear8(x8, w8, b))
    assert torch.equal(f.linear8(unaligned(x), w8, b), f.linear8(x8, w8, b))
    xf = x.float()
    assert torch.equal(f.linear8(xf[None], w8, b), f.linear8(x8, w8, b)[None])


@pytest.mark.parametrize("rows,k,n", [(3000, 300, 3000), (2950, 128, 3001), (9000, 400, 3000), (2900, 1100, 2840), (600, 2100, 520),
                                      (300, 4200, 131)])
def test_linear8_of_many_tiles(dev, rows, k, n):
    """Enough tiles that a workgroup takes whole CUs, one or several tiles each, ragged ones among them and 1 to 9 runs deep; and few
    tiles of many runs, which are cut into parts."""
    _, x, w, b = linear_case(rows, k, n, dev)
    w8, x8 = f.quantize8(w), f.quantize8(x)
    a64, w64 = quantize64(x)[0], quantize64(w)[0]
    for bias, gelu, dtype in ((b, True, bf), (b.to(bf), False, bf), (None, False, f32), (b.to(bf), True, f32)):
        print(f"  linear8 {rows} x {k} x {n} gelu {gelu} {dtype}", flush=True)
        y = f.linear8(x8, w8, bias, gelu=gelu, dtype=dtype)
        check_linear(y, a64, w64, bias, gelu)
        assert torch.equal(f.linear8(x, w8, bias, gelu=gelu, dtype=dtype), y)
    o = unaligned(torch.zeros((rows, n), dtype=f32, device=dev))
    assert torch.equal(f.linear8(x8, w8, b.to(bf), gelu=True, dtype=f32, out=o), y)


def test_blocks8_with_a_scale_of_nan(dev):
    """A scale byte of 255 stands for NaN: its run's values are, and what is made of them."""
    for rows in (40, 300):
        x8 = f.quantize8(tokens(gen_of(rows), rows, 300, bf, dev))
        w8 = f.quantize8(tokens(gen_of(5), 264, 300, bf, dev))
        dy = tokens(gen_of(6), rows, 264, bf, dev)
        x8.scales.view(torch.uint8)[7, 1] = 255
        v = f.dequantize8(x8).isnan()
        assert v[7, 128:256].all() and v.sum() == 128
        y = f.linear8(x8, w8).isnan()
        assert y[7].all() and y.sum() == 264
        for d in (dy, unaligned(dy)):
            dw = f.linear8_weight_grad(d, x8)[0].isnan()
            assert dw[:, 128:256].all() and dw.sum() == 128 * 264
        dx = f.layer_norm_backward(dy[:, :1].expand(rows, 300).contiguous(), x8, torch.ones((rows, 2), device=dev))[0].isnan()
        assert dx[7].all() and dx.sum() == 300


def test_linear8_of_rows_with_nan(dev):
    """A NaN token takes its row of y, a NaN weight its column; no other value."""
    _, x, w, b = linear_case(150, 300, 140, dev)
    clean = f.linear8(x, f.quantize8(w), b)
    x[7, 299], w[131, 0] = math.nan, math.inf
    y = f.linear8(x, f.quantize8(w), b)
    hit = torch.zeros_like(y, dtype=torch.bool)
    hit[7], hit[:, 131] = True, True
    assert torch.equal(y.isnan(), hit) and torch.equal(y[~hit], clean[~hit])


def test_linear8_past_32_bits(dev):
    """More than 2^32 bytes of 8-bit tokens: the last rows equal their own product, and their share of the weight gradient."""
    k = 16384
    rows = (1 << 32) // k + 300
    x8 = f.Blocks8(torch.zeros((rows, k), dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn),
                   torch.zeros((rows, k // RUN), dtype=torch.uint8, device=dev).view(torch.float8_e8m0fnu), k)
    g = gen_of(77)
    tail = f.quantize8(tokens(g, 200, k, bf, dev))
    x8.codes[-200:], x8.scales[-200:] = tail.codes, tail.scales
    w8 = f.quantize8((torch.randn((24, k), generator=g) / 128).to(bf).to(dev))
    y, ref = f.linear8(x8, w8, dtype=f32), f.linear8(tail, w8, dtype=f32)
    assert not y[:-200].any()
    within(y[-200:], ref.double(), 2 * product_off(values(tail), values(w8)), "tail")
    dy = torch.randn((rows, 24), generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(bf)
    dw, db = f.linear8_weight_grad(dy, x8)
    d64, a = dy[-200:].double(), values(tail)
    within(dw, d64.t() @ a, (rows + 8) * U * (d64.abs().t() @ a.abs()), "dweight")
    within(db, dy.double().sum(0), (rows + 8) * U * dy.double().abs().sum(0), "dbias")


@pytest.mark.parametrize("rows,k,n", LINEAR_SHAPES + [(1000, 136, 200), (5000, 256, 264), (40, 2304, 2000),
                                                      (129, 1000, 4200), (20000, 300, 520)])
def test_linear8_weight_grad(dev, rows, k, n):
    g, x, _, _ = linear_case(rows, k, n, dev)
    dy = torch.randn((rows, n), generator=g).to(bf).to(dev)
    x8, a = f.quantize8(x), quantize64(x)[0]
    want, mag = dy.double().t() @ a, dy.double().abs().t() @ a.abs()
    for dtype, d in ((f32, dy), (bf, dy), (bf, unaligned(dy))):
        print(f"  linear8_weight_grad {rows} x {k} x {n} {dtype}", flush=True)
        dw, db = f.linear8_weight_grad(d, x8, dtype)
        within(dw, want, ((rows + 8) * U * mag + HALF[dtype] * want.abs()) * (1 + 2.0 ** -7), "dweight")
        within(db, dy.double().sum(0), (rows + 8) * U * dy.double().abs().sum(0), "dbias")
        o = unaligned(torch.zeros((n, k), dtype=dtype, device=dev))
        got, none = f.linear8_weight_grad(d, x8, dtype, want_bias=False, out=o)
        assert got is o and none is None and torch.equal(o, dw)


@pytest.mark.parametrize("rows,k,n", [(9000, 3900, 4100), (9000, 1400, 5700)])
def test_linear8_weight_grad_of_many_tiles(dev, rows, k, n):
    """More tiles than workgroups run at once, or more than half as many, their tokens cut into parts all the same."""
    g = gen_of(rows, k)
    x8 = f.quantize8((torch.randn((rows, k), generator=g)).to(bf).to(dev))
    dy = torch.randn((rows, n), generator=g).to(bf).to(dev)
    dw, db = f.linear8_weight_grad(dy, x8)
    a = values(x8)[:, :k]
    within(dw, dy.double().t() @ a, (rows + 8) * U * (dy.double().abs().t() @ a.abs()) * (1 + 2.0 ** -7), "dweight")
    within(db, dy.double().sum(0), (rows + 8) * U * dy.double().abs().sum(0), "dbias")
    assert torch.equal(f.linear8_weight_grad(dy, x8, want_bias=False)[0], dw)


@pytest.mark.parametrize("rows,k,n", [(200, 300, 264), (50, 100, 130), (700, 300, 520)])
def test_linear8_weight_grad_of_infinities(dev, rows, k, n):
    """An infinity or NaN in dY takes its row of dW and its value of db; no other value."""
    g, x, _, _ = linear_case(rows, k, n, dev)
    dy = torch.randn((rows, n), generator=g).to(bf).to(dev)
    x8 = f.quantize8(x)
    for layout in (lambda t: t, unaligned):
        dw, db = f.linear8_weight_grad(layout(dy), x8)
        bad = dy.clone()
        bad[7, 16], bad[rows - 1, 40], bad[3, n - 1] = math.inf, math.nan, -math.inf
        gw, gb = f.linear8_weight_grad(layout(bad), x8)
        hit = torch.zeros(n, dtype=torch.bool, device=dev)
        hit[[16, 40, n - 1]] = True
        assert gb[16] == math.inf and gb[40].isnan() and gb[n - 1] == -math.inf
        assert torch.equal(gb[~hit], db[~hit]) and torch.equal(gw[~hit], dw[~hit])
        assert not gw[hit].isfinite().any()


def test_linear8_input_gradient(dev):
    """dx = linear8(dy, quantize8(W^T)) against the 8-bit values' product."""
    g, x, w, _ = linear_case(333, 520, 270, dev)
    dy = torch.randn((333, 270), generator=g).to(bf).to(dev)
    wt = w.t().contiguous()
    dx = f.linear8(dy, f.quantize8(wt), dtype=f32)
    check_linear(dx, quantize64(dy)[0], quantize64(wt)[0], None, False)


# ---- empty batches, streams, graphs, the chain ----------------------------------------------------------------------
def test_no_rows(dev):
    x = torch.zeros((0, 300), dtype=bf, device=dev)
    q = f.quantize8(x)
    assert q.shape == (0, 300) and f.dequantize8(q).shape == (0, 300)
    y, stats, x8 = f.layer_norm(x, want_stats=True, want_x8=True)
    assert y.shape == (0, 300) and stats.shape == (0, 2) and x8.rows == 0
    for kept in (x, x8):
        dx, dw, db = f.layer_norm_backward(x, kept, stats)
        assert dx.shape == (0, 300) and torch.equal(dw, torch.zeros(300, device=dev)) and torch.equal(db, dw)
    w8 = f.quantize8(torch.ones((40, 300), dtype=bf, device=dev))
    assert f.linear8(x, w8).shape == (0, 40) and f.linear8(q, w8, gelu=True, dtype=f32).shape == (0, 40)
    dw, db = f.linear8_weight_grad(torch.zeros((0, 40), dtype=bf, device=dev), q)
    assert torch.equal(dw, torch.zeros((40, 300), device=dev)) and torch.equal(db, torch.zeros(40, device=dev))


def training_pass(x, w, b, w8, w8t, nw, nb, dy, stream=None):
    """norm -> linear layer and back, everything kept in 8 bits"""
    y8, stats, x8 = f.layer_norm(x, nw, nb, want_stats=True, want_x8=True, quantized=True, stream=stream)
    z = f.linear8(y8, w8, b, stream=stream)
    dyn = f.linear8(dy, w8t, stream=stream)
    dw, db = f.linear8_weight_grad(dy, y8, stream=stream)
    dx, dnw, dnb = f.layer_norm_backward(dyn, x8, stats, nw, stream=stream)
    return z, dw, db, dx, dnw, dnb


def pass_inputs(dev, seed, rows=333, k=520, n=270):
    g, x, w, b = linear_case(rows + seed, k, n, dev)
    nw, nb = torch.randn(k, generator=g).to(dev), torch.randn(k, generator=g).to(dev)
    dy = torch.randn((rows + seed, n), generator=g).to(bf).to(dev)
    return [x, w, b, f.quantize8(w), f.quantize8(w.t().contiguous()), nw, nb, dy]


def test_training_pass_of_a_norm_and_a_linear_layer(dev):
    """The chain against the same chain of float64 plain forms; a step is held to its own tolerance on the operands that it was
    given, the steps before it having been checked."""
    x, w, b, w8, w8t, nw, nb, dy = pass_inputs(dev, 0)
    z, dw, db, dx, dnw, dnb = training_pass(x, w, b, w8, w8t, nw, nb, dy)
    y8, stats, x8 = f.layer_norm(x, nw, nb, want_stats=True, want_x8=True, quantized=True)
    y64 = norm64(x, nw, nb)[0]
    # off by half a step of e4m3, or a whole one where the fp32 value fell on the other side of a border
    within(values(y8)[:, :520], y64, 2.0 ** -3 * y64.abs() + 2.0 ** -16 * y64.abs().amax(1, keepdim=True), "y8")
    a = values(y8)[:, :520]
    check_linear(z, a, quantize64(w)[0], b, False)
    dyn = f.linear8(dy, w8t)
    check_linear(dyn, quantize64(dy)[0], quantize64(w.t().contiguous())[0], None, False)
    within(dw, dy.double().t() @ a, (333 + 8) * U * (dy.double().abs().t() @ a.abs()), "dw")
    check_norm_grad(dyn, quantize64(x)[0], stats, nw, dx, dnw, dnb)


def test_calls_on_two_streams_at_once(dev):
    """Passes of different inputs in turn on two side streams, neither waiting for the other: each the same as alone."""
    ins = [pass_inputs(dev, s) for s in (1, 2)]
    want = [training_pass(*i) for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev), torch.cuda.Stream(dev)]
    got = [[], []]
    for _ in range(6):
        for j in (0, 1):
            got[j].append(training_pass(*ins[j], stream=streams[j]))
    torch.cuda.synchronize()
    for j in (0, 1):
        for r in got[j]:
            assert all(torch.equal(p, q) for p, q in zip(r, want[j]))
    raw = f.quantize8(ins[0][0], stream=streams[0].cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(raw.codes.view(torch.uint8), f.quantize8(ins[0][0]).codes.view(torch.uint8))


def test_captured_passes_replay(dev):
    """Two graphs of a training pass, replayed in turn with new inputs and eager passes between: each replay equals the eager one."""
    ins = [pass_inputs(dev, s) for s in (3, 4)]
    for i in ins:
        training_pass(*i)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(training_pass(*i))
        graphs.append(g)
    for rep in range(3):
        for i, g, out in zip(ins, graphs, outs):
            print(f"  replay {rep}", flush=True)
            i[0].copy_(torch.randn_like(i[0].float()).to(bf))
            i[7].copy_(torch.randn_like(i[7].float()).to(bf))
            g.replay()
            torch.cuda.synchronize()
            want = training_pass(*i)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, want)), rep
