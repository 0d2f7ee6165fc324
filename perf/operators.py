"""The operators for training and serving the DiT's dense layers in 8 bits, as a pass of each is used and measured.

A case is a dict of plain values with a `kind`:

  norm         layer norm of (rows, channels) tokens, affine or not: y
  norm_train   a training pass through a layer norm: the forward pass keeps the rows' statistics and its input, as it is or
               (`keep8`) in 8 bits; the backward pass makes dx, dweight and dbias from what was kept
  checkpoint   an activation kept in 8 bits and brought back: the values that it stands for
  linear       y = x W^T + b, optionally GELU (tanh form): x (rows, inner) quantized in the call, W quantized beforehand
  norm_linear  the same product from tokens that a layer norm quantizes as it writes them
  weight_grad  dW = dY^T X and db = the sum of dY's rows, from X kept in 8 bits
  linear_train a training pass through a linear layer whose 8-bit input is also its checkpoint: y, dx, dW, db

8 bits: each run of 128 channels of a row (the last one padded with zeros) has a scale 2^e, the smallest (e >= -127) with
max |x| <= 448 * 2^e over the run's finite values, and each channel is the nearest e4m3 number to x / 2^e (ties to even);
what is not finite becomes NaN. Codes are float8_e4m3fn, (rows, 128 * runs); scales float8_e8m0fnu, one byte a run, rows
padded to a multiple of 4 bytes with zero bytes.

Sizes are the DiT block's: 1536 channels (12 heads of 128), FFN width 8960, 512 text tokens of 4096 features, 135 windows of
128 tokens a temporal slice at 1920 x 1152.
"""
import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-flashvsr-swift_amd")

EPS = 1e-6
RUN = 128
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _lib():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import fvsr_lcsa
    return fvsr_lcsa


def listed():
    return [
        # one time-embedding row: the latency of a norm call
        {"name": "norm 1 x 1536", "kind": "norm", "rows": 1, "channels": 1536, "dtype": "bf16", "affine": True},
        # norm3 of a steady 1920 x 1152 chunk (one temporal slice of tokens)
        {"name": "norm 17280 x 1536", "kind": "norm", "rows": 17280, "channels": 1536, "dtype": "bf16", "affine": True},
        # the same norm in training, its input kept in 8 bits
        {"name": "norm train 17280 x 1536", "kind": "norm_train", "rows": 17280, "channels": 1536, "dtype": "bf16",
         "affine": True, "keep8": True},
        # an odd width in fp32, the input kept as it is
        {"name": "norm train f32 2001 x 1003", "kind": "norm_train", "rows": 2001, "channels": 1003, "dtype": "f32",
         "affine": True, "keep8": False},
        # the FFN's hidden activations of a chunk, kept for the backward pass
        {"name": "checkpoint 17280 x 8960", "kind": "checkpoint", "rows": 17280, "channels": 8960, "dtype": "bf16"},
        # a ragged fp32 activation
        {"name": "checkpoint f32 333 x 4001", "kind": "checkpoint", "rows": 333, "channels": 4001, "dtype": "f32"},
        # the time projection: one row into the six modulation rows
        {"name": "linear 1 x 1536 x 9216", "kind": "linear", "rows": 1, "inner": 1536, "outer": 9216, "gelu": False},
        # the text embedding's first layer over a prompt
        {"name": "linear 512 x 4096 x 1536", "kind": "linear", "rows": 512, "inner": 4096, "outer": 1536, "gelu": True},
        # the FFN's second layer over a chunk
        {"name": "linear 17280 x 8960 x 1536", "kind": "linear", "rows": 17280, "inner": 8960, "outer": 1536,
         "gelu": False},
        # norm2 and the FFN's first layer over a chunk
        {"name": "norm linear 17280", "kind": "norm_linear", "rows": 17280, "inner": 1536, "outer": 8960, "gelu": True},
        # the weight gradient of the FFN's first layer over a chunk
        {"name": "weight grad 17280", "kind": "weight_grad", "rows": 17280, "inner": 1536, "outer": 8960},
        # a small layer with odd widths and a ragged batch of tokens, all of its training pass
        {"name": "linear train 777 x 523 x 270", "kind": "linear_train", "rows": 777, "inner": 523, "outer": 270},
    ]


def _spread(rng, low, high):
    """A whole number from low to high, uniform in its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm_train", "checkpoint", "linear", "norm_linear", "weight_grad", "linear_train"])
    rows = _spread(rng, 1, 17280)
    if kind in ("norm", "norm_train", "checkpoint"):
        c = {"kind": kind, "rows": rows, "channels": _spread(rng, 8, 8960), "dtype": rng.choice(["bf16", "bf16", "f32"])}
        if kind != "checkpoint":
            c["affine"] = rng.random() < 0.75
        if kind == "norm_train":
            c["keep8"] = rng.random() < 0.5
        return c
    inner, outer = _spread(rng, 32, 8960), _spread(rng, 32, 8960)
    if rng.random() < 0.5:   # widths of real layers are mostly whole runs
        inner = -(-inner // RUN) * RUN
    most = 17280 * 1536 * 8960 // (3 if kind == "linear_train" else 1)
    c = {"kind": kind, "rows": max(1, min(rows, most // (inner * outer))), "inner": inner, "outer": outer}
    if kind in ("linear", "norm_linear"):
        c["gelu"] = rng.random() < 0.5
    return c


# ----------------------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------------------
def _activations(gen, rows, channels, dtype):
    """Tokens as a transformer's residual stream has them: channels of different gains and means, a few outliers."""
    gain = torch.exp(0.5 * torch.randn(channels, generator=gen, device="cuda"))
    gain = torch.where(torch.rand(channels, generator=gen, device="cuda") < 0.01, 20 * gain, gain)
    mean = 0.3 * torch.randn(channels, generator=gen, device="cuda")
    return (torch.randn((rows, channels), generator=gen, device="cuda") * gain + mean).to(dtype)


def _normal(gen, shape, scale, dtype):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    rows, kind = case["rows"], case["kind"]
    if kind in ("norm", "norm_train", "checkpoint"):
        c, t = case["channels"], TYPES[case["dtype"]]
        s["x"] = _activations(gen, rows, c, t)
        if case.get("affine"):
            s["weight"] = 1 + _normal(gen, (c,), 0.1, torch.float32)
            s["bias"] = _normal(gen, (c,), 0.05, torch.float32)
        if kind == "norm_train":
            s["dy"] = _normal(gen, (rows, c), 1e-3, t)
        return s
    k, n, t = case["inner"], case["outer"], torch.bfloat16
    if kind == "weight_grad":
        s["x8"] = _plain_quantize(_activations(gen, rows, k, t))
        s["dy"] = _normal(gen, (rows, n), 1e-3, t)
        return s
    s["x"] = _activations(gen, rows, k, t)
    w = _normal(gen, (n, k), 1 / math.sqrt(k), t)
    s["w8"] = _plain_quantize(w)
    s["bias"] = _normal(gen, (n,), 0.05, torch.float32)
    if kind == "norm_linear":
        s["weight"] = 1 + _normal(gen, (k,), 0.1, torch.float32)
        s["shift"] = _normal(gen, (k,), 0.05, torch.float32)
    if kind == "linear_train":
        s["w8t"] = _plain_quantize(w.t().contiguous())
        s["dy"] = _normal(gen, (rows, n), 1e-3, t)
    return s


# ----------------------------------------------------------------------------------------------------------------------
# the plain forms, 32 bits
# ----------------------------------------------------------------------------------------------------------------------
def _runs(x):
    """(rows, channels) -> (rows, runs, 128), padded with zeros."""
    rows, c = x.shape
    g = -(-c // RUN)
    return torch.nn.functional.pad(x, (0, g * RUN - c)).reshape(rows, g, RUN)


def _plain_quantize(x):
    """(codes, scales, channels) of x."""
    rows, c = x.shape
    g = _runs(x.float())
    top = torch.where(torch.isfinite(g), g.abs(), 0.0).amax(-1)
    part, power = torch.frexp(top)                                   # top = part * 2^power, part in [0.5, 1)
    e = torch.where(part > 0.875, power - 8, power - 9)              # 448 = 0.875 * 2^9
    e = torch.where(top > 0, e, -127).clamp(min=-127)
    # 2^-e exactly (exp2 may be off in the last bit, which would move ties)
    inverse = (127 - e).to(torch.uint8).view(torch.float8_e8m0fnu).float()
    codes = (torch.where(torch.isfinite(g), g, math.nan) * inverse[..., None]).to(torch.float8_e4m3fn).reshape(rows, -1)
    n = g.shape[1]
    scales = torch.nn.functional.pad((127 + e).to(torch.uint8), (0, -n % 4)).view(torch.float8_e8m0fnu)
    return codes, scales, c


def _plain_values(q):
    codes, scales, c = q
    g = codes.shape[1] // RUN
    v = codes.float().reshape(codes.shape[0], g, RUN) * scales.float()[:, :g, None]
    return v.reshape(codes.shape[0], g * RUN)[:, :c]


def _plain_norm(x, weight, bias):
    """(y, the normed rows, 1 / standard deviation), all in 32 bits."""
    x = x.float()
    d = x - x.mean(-1, keepdim=True)
    inv = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS)
    n = d * inv
    return (n if weight is None else n * weight + bias), inv


def _plain_linear(a, w, bias, gelu):
    y = a @ w.t()
    if bias is not None:
        y = y + bias
    if gelu:
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return y


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "norm":
        return {"y": _plain_norm(s["x"], s.get("weight"), s.get("bias"))[0].to(s["x"].dtype)}
    if kind == "norm_train":
        x, dy, w = s["x"], s["dy"].float(), s.get("weight")
        y, inv = _plain_norm(x, w, s.get("bias"))
        kept = _plain_values(_plain_quantize(x)) if case["keep8"] else x.float()
        n = (kept - x.float().mean(-1, keepdim=True)) * inv
        g = dy if w is None else dy * w
        dx = inv * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
        out = {"y": y.to(x.dtype), "dx": dx.to(x.dtype)}
        if w is not None:
            out |= {"dweight": (dy * n).sum(0), "dbias": dy.sum(0)}
        return out
    if kind == "checkpoint":
        return {"x": _plain_values(_plain_quantize(s["x"])).to(s["x"].dtype)}
    if kind == "linear":
        a = _plain_values(_plain_quantize(s["x"]))
        return {"y": _plain_linear(a, _plain_values(s["w8"]), s["bias"], case["gelu"]).bfloat16()}
    if kind == "norm_linear":
        a = _plain_values(_plain_quantize(_plain_norm(s["x"], s["weight"], s["shift"])[0]))
        return {"y": _plain_linear(a, _plain_values(s["w8"]), s["bias"], case["gelu"]).bfloat16()}
    if kind == "weight_grad":
        dy = s["dy"].float()
        return {"dweight": dy.t() @ _plain_values(s["x8"]), "dbias": dy.sum(0)}
    a, dy = _plain_values(_plain_quantize(s["x"])), s["dy"].float()
    g = _plain_values(_plain_quantize(s["dy"]))
    return {"y": _plain_linear(a, _plain_values(s["w8"]), s["bias"], False).bfloat16(),
            "dx": _plain_linear(g, _plain_values(s["w8t"]), None, False).bfloat16(),
            "dweight": dy.t() @ a, "dbias": dy.sum(0)}


# ----------------------------------------------------------------------------------------------------------------------
# the framework's calls
# ----------------------------------------------------------------------------------------------------------------------
def _own(s):
    f = _lib()
    case = s["case"]
    kind = case["kind"]
    if kind == "norm":
        return {"y": f.layer_norm(s["x"], s.get("weight"), s.get("bias"), EPS)[0]}
    if kind == "norm_train":
        affine = case["affine"]
        y, stats, x8 = f.layer_norm(s["x"], s.get("weight"), s.get("bias"), EPS, want_stats=True, want_x8=case["keep8"])
        dx, dw, db = f.layer_norm_backward(s["dy"], x8 if case["keep8"] else s["x"], stats, s.get("weight"),
                                           want_params=affine)
        return {"y": y, "dx": dx} | ({"dweight": dw, "dbias": db} if affine else {})
    if kind == "checkpoint":
        return {"x": f.dequantize8(f.quantize8(s["x"]), s["x"].dtype)}
    if kind == "linear":
        return {"y": f.linear8(s["x"], f.Blocks8(*s["w8"]), s["bias"], gelu=case["gelu"])}
    if kind == "norm_linear":
        a = f.layer_norm(s["x"], s["weight"], s["shift"], EPS, quantized=True)[0]
        return {"y": f.linear8(a, f.Blocks8(*s["w8"]), s["bias"], gelu=case["gelu"])}
    if kind == "weight_grad":
        dw, db = f.linear8_weight_grad(s["dy"], f.Blocks8(*s["x8"]))
        return {"dweight": dw, "dbias": db}
    x8 = f.quantize8(s["x"])
    y = f.linear8(x8, f.Blocks8(*s["w8"]), s["bias"])
    dx = f.linear8(s["dy"], f.Blocks8(*s["w8t"]))
    dw, db = f.linear8_weight_grad(s["dy"], x8)
    return {"y": y, "dx": dx, "dweight": dw, "dbias": db}


def run(state):
    return _own(state) if own else _plain(state)


# ----------------------------------------------------------------------------------------------------------------------
# what a pass has to read, write and compute
# ----------------------------------------------------------------------------------------------------------------------
def work(case):
    kind, m = case["kind"], case["rows"]
    if kind in ("norm", "norm_train", "checkpoint"):
        c, es = case["channels"], 2 if case["dtype"] == "bf16" else 4
        params = 4 * c * (2 if case.get("affine") else 0)
        if kind == "norm":
            return {"bytes": 2 * m * c * es + params, "flops": 8 * m * c}
        if kind == "checkpoint":
            return {"bytes": 2 * m * c * es, "flops": 3 * m * c}
        return {"bytes": 4 * m * c * es + 2 * params, "flops": 24 * m * c}   # x, dy, y, dx; the weights and gradients
    k, n = case["inner"], case["outer"]
    runs = -(-k // RUN)
    weight = n * (k + runs)                                                  # 8-bit weights and their scales
    if kind == "weight_grad":
        return {"bytes": 2 * m * n + m * (k + runs) + 4 * n * k + 4 * n, "flops": 2 * m * n * k}
    if kind == "linear_train":
        back = k * (n + -(-n // RUN))
        return {"bytes": 4 * m * k + 4 * m * n + weight + back + 4 * n * k + 8 * n, "flops": 6 * m * n * k}
    return {"bytes": 2 * m * k + weight + 2 * m * n + 4 * n, "flops": 2 * m * n * k}


# ----------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ----------------------------------------------------------------------------------------------------------------------
def _two_to(e):
    """2^e in 64 bits, by its bits (a power function may be off in the last one)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _held64(x):
    """What x stands for after 8 bits: the definition, with half-to-even rounding of quotients by the step in 64 bits."""
    x = x.double()
    m, c = x.shape
    out = torch.empty_like(x)
    whole = c // RUN * RUN
    for part, width in ((slice(0, whole), RUN), (slice(whole, c), c - whole)):
        if width == 0 or part.start == part.stop:
            continue
        r = x[:, part].reshape(m, -1, width)
        ok = torch.isfinite(r)
        top = torch.where(ok, r.abs(), torch.zeros_like(r)).max(-1, keepdim=True).values
        part64, power = torch.frexp(top.clamp_min(1e-300) / 448)         # smallest e with top / 448 <= 2^e
        e = torch.where(part64 == 0.5, power - 1, power).clamp_min(-127)
        binade = torch.frexp(r.abs())[1] - 1 - e                         # of the quotient by the scale
        step = _two_to(binade.clamp_min(-6) - 3 + e)
        held = torch.round(r / step) * step
        out[:, part] = torch.where(ok, held, torch.full_like(held, math.nan)).reshape(m, -1)
    return out


def _decode64(q):
    codes, scales, c = q
    by = _two_to(scales.view(torch.uint8).to(torch.int64) - 127)
    return (codes.double() * by.repeat_interleave(RUN, 1)[:, :codes.shape[1]])[:, :c]


def _norm64(x, weight, bias):
    x = x.double()
    mean = x.sum(1) / x.shape[1]
    var = (x * x).sum(1) / x.shape[1] - mean * mean
    inv = (var + EPS) ** -0.5
    y = (x - mean[:, None]) * inv[:, None]
    if weight is not None:
        y = weight.double() * y + bias.double()
    return y, mean, inv


def _linear64(a, w, bias, gelu):
    y = torch.mm(a, w.t())
    if bias is not None:
        y += bias.double()
    if gelu:
        y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))   # (1 + tanh u) / 2 = sigmoid(2 u)
    return y


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        return {"y": _norm64(s["x"], s.get("weight"), s.get("bias"))[0]}
    if kind == "norm_train":
        w = s.get("weight")
        y, mean, inv = _norm64(s["x"], w, s.get("bias"))
        kept = _held64(s["x"]) if case["keep8"] else s["x"].double()
        n = (kept - mean[:, None]) * inv[:, None]
        dy = s["dy"].double()
        g = dy if w is None else dy * w.double()
        c = g.shape[1]
        dx = (g - (g.sum(1) / c)[:, None] - n * ((g * n).sum(1) / c)[:, None]) * inv[:, None]
        out = {"y": y, "dx": dx}
        if w is not None:
            out["dweight"], out["dbias"] = (dy * n).sum(0), dy.sum(0)
        return out
    if kind == "checkpoint":
        return {"x": _held64(s["x"])}
    if kind == "weight_grad":
        dy = s["dy"].double()
        return {"dweight": torch.mm(dy.t(), _decode64(s["x8"])), "dbias": dy.sum(0)}
    if kind == "norm_linear":
        # a rounding to 8 bits next to a border may fall either way by the norm's last bits: the norm in 32 bits, where the
        # operator rounds it, then everything in 64
        a = _held64(_norm64(s["x"], s["weight"], s["shift"])[0].float())
    else:
        a = _held64(s["x"])
    out = {"y": _linear64(a, _decode64(s["w8"]), s["bias"], case.get("gelu", False))}
    if kind == "linear_train":
        dy = s["dy"].double()
        out |= {"dx": _linear64(_held64(s["dy"]), _decode64(s["w8t"]), None, False),
                "dweight": torch.mm(dy.t(), a), "dbias": dy.sum(0)}
    return out
