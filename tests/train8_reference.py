"""The 8-bit form, layer norm and the 8-bit linear layers in float64, written from their definitions without the package."""
import math

import torch

RUN = 128
U = 2.0 ** -24                                   # half a step of float32, relative
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def pow2(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def quantize64(x):
    """(values (rows, channels) float64, scale exponents (rows, runs)) of x in 8 bits."""
    x = x.double()
    rows, c = x.shape
    runs = -(-c // RUN)
    r = torch.nn.functional.pad(x, (0, runs * RUN - c)).reshape(rows, runs, RUN)
    fin = torch.isfinite(r)
    top = r.abs().masked_fill(~fin, 0).amax(-1, keepdim=True)
    part, power = torch.frexp(top / 448)
    e = torch.where(part == 0.5, power - 1, power)              # smallest e with top <= 448 * 2^e
    e = torch.where(top > 0, e, torch.full_like(e, -127)).clamp_min(-127)
    q = r.masked_fill(~fin, 0) / pow2(e)
    step = pow2((torch.frexp(q.abs())[1] - 1).clamp_min(-6) - 3)
    v = (torch.round(q / step) * step * pow2(e)).masked_fill(~fin, math.nan)
    return v.reshape(rows, -1)[:, :c], e[..., 0]


def norm64(x, w=None, b=None, eps=1e-6):
    """(y, mean, rstd)"""
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = ((x - mean).square().mean(1, keepdim=True) + eps).rsqrt()
    y = (x - mean) * rstd
    y = y if w is None else y * w.double()
    return (y if b is None else y + b.double()), mean, rstd


def norm_grad64(dy, x, stats, w=None):
    """(dx, dweight, dbias), and n"""
    dy, x, stats = dy.double(), x.double(), stats.double()
    n = (x - stats[:, :1]) * stats[:, 1:]
    g = dy if w is None else dy * w.double()
    dx = stats[:, 1:] * (g - g.mean(1, keepdim=True) - n * (g * n).mean(1, keepdim=True))
    return dx, (dy * n).sum(0), dy.sum(0), n


def gelu64(y):
    return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))


def within(got, want, tol, what=""):
    """Every |got - want| <= tol (a tensor), NaN exactly where `want` has it."""
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan()), what
    over = ((got - want).abs() - tol).nan_to_num(-1.0)
    bad = over > 0
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values are off by up to {float((got - want).abs()[bad].max()):.3e}"
