"""The operators of the self-attention's training and serving path, as a pass of each is used and measured.

A case is a dict of plain values with a `kind`:

  rms            root-mean-square norm of (rows, channels) tokens, after the residual's addition where there is one: y, the sum
  rms8           the same with y in 8 bits, as the 8-bit linear layers read it: the values that it stands for, the sum
  rms_train      a training pass: y, the sum; then dx (the gradient of both addends) and dweight, from the gradients of y
                 and of the sum
  rotary         q and k turned by positions of one to three axes (time, height, width)
  rotary_train   the same, and the gradients turned back
  decode         one query a sequence (or a few) over a cache with room for `room` keys a sequence, `lengths` of them used
  prompt         attention over packed sequences of `lengths` tokens, causal or whole, the query heads in groups that share
                 one key and value head
  attend_train   a training pass: o, then dq, dk and dv

With s = x + residual, rounded to the tokens' type as the next layers read it: y = s / sqrt(mean(s^2) + eps) * weight. Pair i
of a head (channels 2 i and 2 i + 1, or, in halves, i and i + pairs) belongs to one axis and turns by that axis' position times
the pair's frequency, 10000^(-i / the axis' pairs); channels past the pairs stay. Query i of a sequence of m queries and n keys
sees all n, or, causal, the first i + 1 + n - m; a query that sees none gives zeros. In 8 bits a run of 128 channels has a scale
2^e, the smallest (e >= -127) with max |x| <= 448 * 2^e, and each channel the nearest e4m3 number to x / 2^e.

Sizes are the DiT block's (1536 channels, 12 heads of 128, 17280 tokens a temporal slice at 1920 x 1152, 43200 keys of five
latent frames), and generic ones around them.
"""
import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-flashvsr-swift_amd")

EPS = 1e-6
RUN = 128
THETA = 10000.0
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
MOST_PAIRS = 12 * 17280 * 17280      # visible (head, query, key) triples of the largest training pass


def _lib():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import fvsr_lcsa
    return fvsr_lcsa


def listed():
    return [
        # one token's row on its way through a block: the latency of a call
        {"name": "rms 1 x 1536", "kind": "rms", "rows": 1, "channels": 1536, "dtype": "bf16", "residual": True},
        # the norm before an 8-bit linear layer, over a chunk
        {"name": "rms to 8 bits 17280 x 1536", "kind": "rms8", "rows": 17280, "channels": 1536, "dtype": "bf16",
         "residual": True},
        # the same norm in training
        {"name": "rms train 17280 x 1536", "kind": "rms_train", "rows": 17280, "channels": 1536, "dtype": "bf16",
         "residual": True},
        # an odd width in fp32, without a residual
        {"name": "rms train f32 2001 x 1003", "kind": "rms_train", "rows": 2001, "channels": 1003, "dtype": "f32",
         "residual": False},
        # a chunk's q and k, at its (time, height, width) positions
        {"name": "rotary 17280 x 12 + 12", "kind": "rotary", "tokens": 17280, "heads": 12, "kv_heads": 12, "head_dim": 128,
         "axes": "22,21,21", "dtype": "bf16", "halves": False, "far": 1024},
        # an image's tokens in training, fp32, two axes, paired in halves, some channels not turned
        {"name": "rotary train f32 4001 x 9 + 3", "kind": "rotary_train", "tokens": 4001, "heads": 9, "kv_heads": 3,
         "head_dim": 80, "axes": "16,16", "dtype": "f32", "halves": True, "far": 100000},
        # one query over the keys of five latent frames: all of the card for 12 rows
        {"name": "decode 1 x 43200", "kind": "decode", "queries": 1, "room": 43200, "lengths": "43200", "heads": 12,
         "kv_heads": 2, "head_dim": 128},
        # a batch of sequences of very different lengths, one of them empty
        {"name": "decode 24 of up to 17280", "kind": "decode", "queries": 1, "room": 17280,
         "lengths": "17280,1,640,9001,128,15000,33,2047,12345,777,4096,16383,511,6000,1000,0,8192,3500,250,14000,129,7,10007,5120",
         "heads": 16, "kv_heads": 4, "head_dim": 128},
        # packed prompts of different lengths, causal, grouped heads
        {"name": "prompt causal 17280", "kind": "prompt", "lengths": "9001,1,2048,777,130,4099,31,1193", "causal": True,
         "heads": 12, "kv_heads": 4, "head_dim": 128},
        # small images side by side, every token seeing its own image
        {"name": "prompt 6 x 512", "kind": "prompt", "lengths": "512,512,512,512,512,512", "causal": False, "heads": 12,
         "kv_heads": 12, "head_dim": 128},
        # training on packed causal sequences, narrow heads in groups
        {"name": "attend train causal 8191", "kind": "attend_train", "lengths": "4097,2000,513,64,1500,17", "causal": True,
         "heads": 16, "kv_heads": 4, "head_dim": 64},
        # training on one temporal slice at 1920 x 1152: every token sees every other
        {"name": "attend train 17280", "kind": "attend_train", "lengths": "17280", "causal": False, "heads": 12,
         "kv_heads": 12, "head_dim": 128},
    ]


def _spread(rng, low, high):
    """A whole number from low to high, uniform in its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["rms", "rms8", "rms_train", "rotary", "rotary_train", "decode", "prompt", "attend_train"])
    if kind.startswith("rms"):
        return {"kind": kind, "rows": _spread(rng, 1, 17280), "channels": _spread(rng, 8, 8960),
                "dtype": rng.choice(["bf16", "bf16", "f32"]), "residual": rng.random() < 0.6}
    kv = rng.choice([1, 2, 3, 4, 6, 8])
    heads = {"heads": kv * rng.choice([1, 1, 2, 3, 4]), "kv_heads": kv}
    if kind.startswith("rotary"):
        d = 8 * rng.randint(2, 16)
        left, axes = d // 2, []
        for n in range(rng.randint(1, 3), 0, -1):
            axes.append(left // n - (rng.randint(0, 1) if left // n > 2 else 0))
            left -= axes[-1]
        return {"kind": kind, "tokens": _spread(rng, 1, 17280), **heads, "head_dim": d, "axes": ",".join(map(str, axes)),
                "dtype": rng.choice(["bf16", "bf16", "f32"]), "halves": rng.random() < 0.5, "far": _spread(rng, 16, 100000)}
    heads["head_dim"] = rng.choice([64, 64, 128, 128, 128, 8 * rng.randint(2, 16)])
    if kind == "decode":
        room = _spread(rng, 1, 43200)
        n = max(1, min(_spread(rng, 1, 64), 800000 // (room * kv)))
        lengths = [rng.randint(0, room) if rng.random() < 0.7 else _spread(rng, 1, room) for _ in range(n)]
        return {"kind": kind, "queries": rng.choice([1, 1, 1, 2, 5]), "room": room, "lengths": ",".join(map(str, lengths)), **heads}
    total, lengths = _spread(rng, 16, 17280), []
    while total > 0 and len(lengths) < 24:
        lengths.append(min(total, _spread(rng, 1, 17280)))
        total -= lengths[-1]
    causal = rng.random() < 0.6
    c = {"kind": kind, "lengths": ",".join(map(str, lengths)), "causal": causal, **heads}
    while _pairs(c) * c["heads"] * c["head_dim"] > MOST_PAIRS * 128 and len(lengths) > 1:
        lengths.remove(max(lengths))
        c["lengths"] = ",".join(map(str, lengths))
    while _pairs(c) * c["heads"] * c["head_dim"] > MOST_PAIRS * 128:
        lengths[0] //= 2
        c["lengths"] = str(lengths[0])
    return c


def _lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


def _pairs(case):
    """The visible (query, key) pairs of one head."""
    if case["kind"] == "decode":   # queries that see the keys up to their own, the last one all
        m = case["queries"]
        return sum(max(0, n - m + 1 + i) for n in _lengths(case) for i in range(m))
    return sum(n * (n + 1) // 2 if case["causal"] else n * n for n in _lengths(case))


# ----------------------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------------------
def _normal(gen, shape, scale, dtype):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _stream(gen, rows, channels, dtype):
    """Tokens as a transformer's residual stream has them: channels of different gains, a few outliers."""
    gain = torch.exp(0.5 * torch.randn(channels, generator=gen, device="cuda"))
    gain = torch.where(torch.rand(channels, generator=gen, device="cuda") < 0.01, 20 * gain, gain)
    return (torch.randn((rows, channels), generator=gen, device="cuda") * gain).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    s = {"case": case}
    if kind.startswith("rms"):
        rows, c, t = case["rows"], case["channels"], TYPES[case["dtype"]]
        s["x"] = _stream(gen, rows, c, t)
        s["residual"] = _stream(gen, rows, c, t) if case["residual"] else None
        s["weight"] = 1 + _normal(gen, (c,), 0.1, torch.float32)
        if kind == "rms_train":
            s["dy"] = _normal(gen, (rows, c), 1e-3, t)
            s["dsum"] = _normal(gen, (rows, c), 1e-3, t) if case["residual"] else None
        return s
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    if kind.startswith("rotary"):
        n, t = case["tokens"], TYPES[case["dtype"]]
        pairs = [int(a) for a in case["axes"].split(",")]
        # q, k and v come out of one projection: q and k are parts of its rows
        qkv = _normal(gen, (n, h + 2 * hk, d), 1.0, t)
        s["q"], s["k"] = qkv[:, :h], qkv[:, h:h + hk]
        s["axes"] = tuple(pairs)
        s["positions"] = torch.randint(0, case["far"], (len(pairs), n), generator=gen, device="cuda", dtype=torch.int32)
        s["frequencies"] = torch.cat([THETA ** (-torch.arange(p, dtype=torch.float64) / p) for p in pairs]).cuda()
        if kind == "rotary_train":
            s["dq"], s["dk"] = _normal(gen, (n, h, d), 1e-3, t), _normal(gen, (n, hk, d), 1e-3, t)
        return s
    lengths, b = _lengths(case), torch.bfloat16
    s["n"] = len(lengths)
    if kind == "decode":
        m, room = case["queries"], case["room"]
        s["q"] = _normal(gen, (len(lengths) * m, h, d), 1.5, b)
        s["k"], s["v"] = (_normal(gen, (len(lengths) * room, hk, d), 1.0, b) for _ in range(2))
        s["cu_q"] = m * torch.arange(len(lengths) + 1, dtype=torch.int32, device="cuda")
        s["cu_k"] = room * torch.arange(len(lengths) + 1, dtype=torch.int32, device="cuda")
        s["used"] = torch.tensor(lengths, dtype=torch.int32).cuda()
        return s
    total = sum(lengths)
    qkv = _normal(gen, (total, h + 2 * hk, d), 1.0, b)
    s["q"], s["k"], s["v"] = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    s["cu"] = torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32).cuda()
    if kind == "attend_train":
        s["do"] = _normal(gen, (total, h, d), 1e-3, b)
    return s


# ----------------------------------------------------------------------------------------------------------------------
# the plain forms, 32 bits
# ----------------------------------------------------------------------------------------------------------------------
def _plain_rms(s):
    """(the sum as it is kept, in 32 bits, 1 / root mean square, y)."""
    x = s["x"].float()
    if s["residual"] is not None:
        x = (x + s["residual"].float()).to(s["x"].dtype).float()
    inv = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x, inv, x * inv * s["weight"]


def _plain_held(x):
    """The values that x (rows, channels) stands for in 8 bits."""
    rows, c = x.shape
    g = torch.nn.functional.pad(x, (0, -c % RUN)).reshape(rows, -1, RUN)
    top = g.abs().amax(-1)
    part, power = torch.frexp(top)                                   # top = part * 2^power, part in [0.5, 1)
    e = torch.where(part > 0.875, power - 8, power - 9)              # 448 = 0.875 * 2^9
    e = torch.where(top > 0, e, -127).clamp(min=-127)
    to = lambda e: (127 + e).to(torch.uint8).view(torch.float8_e8m0fnu).float()[..., None]   # 2^e, exactly
    return ((g * to(-e)).to(torch.float8_e4m3fn).float() * to(e)).reshape(rows, -1)[:, :c]


def _plain_turn(x, positions, frequencies, axes, halves, back=False):
    """x (tokens, heads, channels) turned, or turned back; angles in 64 bits."""
    n = sum(axes)
    axis = torch.repeat_interleave(torch.arange(len(axes), device=x.device), torch.tensor(axes, device=x.device), output_size=n)
    angle = positions.double()[axis].t() * frequencies
    c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if back:
        s = -s
    f = x.float()
    a, b = (f[..., :n], f[..., n:2 * n]) if halves else (f[..., 0:2 * n:2], f[..., 1:2 * n:2])
    u, w = a * c - b * s, a * s + b * c
    turned = torch.cat([u, w], -1) if halves else torch.stack([u, w], -1).flatten(-2)
    return torch.cat([turned, f[..., 2 * n:]], -1).to(x.dtype)


def _plain_attend(q, k, v, causal):
    """(weights, o) of one sequence: q (heads, m, d), k and v (heads, n, d), in 32 bits."""
    m, n = q.shape[1], k.shape[1]
    s = torch.matmul(q, k.transpose(1, 2)) / math.sqrt(q.shape[2])
    if causal:
        s = s.masked_fill_(torch.ones(m, n, dtype=torch.bool, device=q.device).triu_(n - m + 1), -math.inf)
    p = s.sub_(s.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True))
    return p, torch.matmul(p, v)


def _heads(x, times=1):
    """(tokens, heads, d) in 32 bits as (heads * times, tokens, d), each head `times` times."""
    return x.float().transpose(0, 1).repeat_interleave(times, 0)


def _plain_decode(s):
    case = s["case"]
    m, room, h, hk, d = (case[x] for x in ("queries", "room", "heads", "kv_heads", "head_dim"))
    q = s["q"].float().view(s["n"], m, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(s["n"], hk, -1, d)
    k, v = (s[x].float().view(s["n"], room, hk, d).transpose(1, 2) for x in "kv")
    score = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(d)
    # query i of a sequence with n keys sees the first n - m + 1 + i
    most = s["used"][:, None] - m + 1 + torch.arange(m, device=q.device)
    seen = torch.arange(room, device=q.device) < most.repeat(1, h // hk)[:, None, :, None]
    top = score.masked_fill(~seen, -math.inf).amax(-1, keepdim=True).clamp_min(-1e30)
    p = torch.where(seen, torch.exp(score - top), 0.0)
    o = torch.matmul(p / p.sum(-1, keepdim=True).clamp_min(1e-30), v)
    return o.view(s["n"], hk, h // hk, m, d).permute(0, 3, 1, 2, 4).reshape(-1, h, d)


def _plain_packed(s):
    case = s["case"]
    g, d = case["heads"] // case["kv_heads"], case["head_dim"]
    train = "do" in s
    parts = []
    split = lambda x: torch.split(x, _lengths(case))
    for q, k, v, do in zip(*(split(s[x]) for x in "qkv"), split(s["do"] if train else s["q"])):
        q, k, v = _heads(q), _heads(k, g), _heads(v, g)
        p, o = _plain_attend(q, k, v, case["causal"])
        if not train:
            parts.append((o,))
            continue
        do = _heads(do)
        dv = torch.matmul(p.transpose(1, 2), do)
        ds = torch.matmul(do, v.transpose(1, 2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).div_(math.sqrt(d))
        dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(1, 2), q)
        del p, ds
        parts.append((o, dq, dk.view(-1, g, *dk.shape[1:]).sum(1), dv.view(-1, g, *dv.shape[1:]).sum(1)))
    return [torch.cat(x, 1).transpose(0, 1).bfloat16().contiguous() for x in zip(*parts)]


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind.startswith("rms"):
        t = s["x"].dtype
        x, inv, y = _plain_rms(s)
        out = {"y": _plain_held(y).bfloat16() if kind == "rms8" else y.to(t)}
        if s["residual"] is not None:
            out["sum"] = x.to(t)
        if kind == "rms_train":
            dy, n = s["dy"].float(), x * inv
            g = dy * s["weight"]
            dx = inv * (g - n * (g * n).mean(-1, keepdim=True))
            if s["dsum"] is not None:
                dx = dx + s["dsum"].float()
            out |= {"dx": dx.to(t), "dweight": (dy * n).sum(0)}
        return out
    if kind.startswith("rotary"):
        how = (s["positions"], s["frequencies"], s["axes"], case["halves"])
        out = {"q": _plain_turn(s["q"], *how), "k": _plain_turn(s["k"], *how)}
        if kind == "rotary_train":
            out |= {"dq": _plain_turn(s["dq"], *how, back=True), "dk": _plain_turn(s["dk"], *how, back=True)}
        return out
    if kind == "decode":
        return {"o": _plain_decode(s).bfloat16()}
    return dict(zip(("o", "dq", "dk", "dv"), _plain_packed(s)))


# ----------------------------------------------------------------------------------------------------------------------
# the framework's calls
# ----------------------------------------------------------------------------------------------------------------------
def _own(s):
    f = _lib()
    case = s["case"]
    kind = case["kind"]
    if kind.startswith("rms"):
        y, total, rstd = f.rms_norm(s["x"], s["weight"], EPS, residual=s["residual"], want_stats=kind == "rms_train",
                                    quantized=kind == "rms8")
        out = {"y": f.dequantize8(y) if kind == "rms8" else y}
        if s["residual"] is not None:
            out["sum"] = total
        if kind == "rms_train":
            kept = s["x"] if total is None else total
            out["dx"], out["dweight"] = f.rms_norm_backward(s["dy"], kept, rstd, s["weight"], dsum=s["dsum"])
        return out
    if kind.startswith("rotary"):
        how = (s["positions"], s["frequencies"], s["axes"])
        q, k = f.rotary(s["q"], s["k"], *how, halves=case["halves"])
        out = {"q": q, "k": k}
        if kind == "rotary_train":
            out["dq"], out["dk"] = f.rotary_backward(s["dq"], s["dk"], *how, halves=case["halves"])
        return out
    if kind == "decode":
        return {"o": f.packed_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=True, used_k=s["used"])[0]}
    causal = case["causal"]
    o, lse = f.packed_attention(s["q"], s["k"], s["v"], s["cu"], causal=causal, want_lse=kind == "attend_train")
    if kind == "prompt":
        return {"o": o}
    dq, dk, dv = f.packed_attention_backward(s["do"], s["q"], s["k"], s["v"], o, lse, s["cu"], causal=causal)
    return {"o": o, "dq": dq, "dk": dk, "dv": dv}


def run(state):
    return _own(state) if own else _plain(state)


# ----------------------------------------------------------------------------------------------------------------------
# what a pass has to read, write and compute
# ----------------------------------------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind.startswith("rms"):
        m, c, es = case["rows"], case["channels"], 2 if case["dtype"] == "bf16" else 4
        r = 1 if case["residual"] else 0
        if kind == "rms_train":   # x, residual, y, sum; dy, dsum, dx; the weight and its gradient
            return {"bytes": (4 + 3 * r) * m * c * es + 8 * c, "flops": 14 * m * c}
        return {"bytes": (1 + 2 * r) * m * c * es + m * c * (2 if kind == "rms8" else es) + 4 * c, "flops": 6 * m * c}
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    if kind.startswith("rotary"):
        n, axes = case["tokens"], [int(a) for a in case["axes"].split(",")]
        times = 2 if kind == "rotary_train" else 1
        es = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": times * 2 * n * (h + hk) * d * es + 4 * len(axes) * n + 8 * sum(axes),
                "flops": times * n * (6 * sum(axes) * (h + hk) + 20 * sum(axes))}
    keys = sum(_lengths(case))
    if kind == "decode":
        rows = len(_lengths(case)) * case["queries"]
        return {"bytes": 4 * rows * h * d + 4 * keys * hk * d, "flops": 4 * _pairs(case) * h * d}
    if kind == "prompt":
        return {"bytes": 4 * keys * h * d + 4 * keys * hk * d, "flops": 4 * _pairs(case) * h * d}
    # q, k, v, do read; o, dq, dk, dv written; two products forward, five back
    return {"bytes": 8 * keys * h * d + 8 * keys * hk * d, "flops": 14 * _pairs(case) * h * d}


# ----------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ----------------------------------------------------------------------------------------------------------------------
def _two_to(e):
    """2^e in 64 bits, by its bits (a power function may be off in the last one)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _held64(x):
    """What x stands for after 8 bits: the definition, with half-to-even rounding of quotients by the step in 64 bits."""
    m, c = x.shape
    r = torch.zeros((m, -(-c // RUN) * RUN), dtype=torch.float64, device=x.device)
    r[:, :c] = x
    r = r.view(m, -1, RUN)
    top = r.abs().max(-1, keepdim=True).values
    part, power = torch.frexp(top.clamp_min(1e-300) / 448)               # smallest e with top / 448 <= 2^e
    e = torch.where(part == 0.5, power - 1, power).clamp_min(-127)
    binade = torch.frexp(r.abs())[1] - 1 - e                             # of the quotient by the scale
    step = _two_to(binade.clamp_min(-6) - 3 + e)
    return (torch.round(r / step) * step).view(m, -1)[:, :c]


def _turn64(x, positions, case, sign):
    """The rotation as a product of complex numbers."""
    pairs = [int(a) for a in case["axes"].split(",")]
    n, cos, sin = sum(pairs), [], []
    for a, p in enumerate(pairs):
        i = torch.arange(p, dtype=torch.float64, device=x.device)
        angle = torch.outer(positions[a].double(), torch.exp(-math.log(THETA) * i / p))
        cos.append(torch.cos(angle))
        sin.append(sign * torch.sin(angle))
    by = torch.complex(torch.cat(cos, 1), torch.cat(sin, 1))[:, None]
    x = x.double()
    first = torch.arange(n, device=x.device) if case["halves"] else 2 * torch.arange(n, device=x.device)
    second = first + (n if case["halves"] else 1)
    turned = torch.complex(x[..., first], x[..., second]) * by
    out = x.clone()
    out[..., first], out[..., second] = turned.real, turned.imag
    return out


def _attend64(q, k, v, seen, do=None):
    """(o, dq, dk, dv) of one head: q (m, d), k and v (n, d); seen (m,): how many keys each query sees."""
    scale = q.shape[1] ** -0.5
    s = torch.mm(q, k.t()) * scale
    hide = torch.arange(k.shape[0], device=q.device) >= seen[:, None]
    p = torch.exp(s - torch.logsumexp(s.masked_fill(hide, -math.inf), 1, keepdim=True))
    p = p.masked_fill(hide, 0)
    o = torch.mm(p, v)
    if do is None:
        return (o,)
    dp = torch.mm(do, v.t())
    ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
    return o, torch.mm(ds, k), torch.mm(ds.t(), q), torch.mm(p.t(), do)


def _attention64(s):
    case = s["case"]
    g = case["heads"] // case["kv_heads"]
    decode = case["kind"] == "decode"
    out = [torch.zeros(x.shape, dtype=torch.float64, device=x.device) for x in (s["q"], s["q"], s["k"], s["v"])]
    at = 0
    for i, n in enumerate(_lengths(case)):
        m = case["queries"] if decode else n
        rows = slice(i * m, i * m + m) if decode else slice(at, at + n)
        keys = slice(i * case["room"], i * case["room"] + n) if decode else rows
        at += n
        seen = n - m + 1 + torch.arange(m, device="cuda") if decode or case["causal"] else torch.full((m,), n, device="cuda")
        for h in range(case["heads"]):
            q, k, v = s["q"][rows, h].double(), s["k"][keys, h // g].double(), s["v"][keys, h // g].double()
            got = _attend64(q, k, v, seen, s["do"][rows, h].double() if "do" in s else None) if n else ()
            for to, r, hh, x in zip(out, (rows, rows, keys, keys), (h, h, h // g, h // g), got):
                to[r, hh] += x
    return dict(zip(("o", "dq", "dk", "dv"), out if "do" in s else out[:1]))


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind.startswith("rms"):
        t = s["x"].dtype
        x = s["x"].double()
        if s["residual"] is not None:
            x = (x + s["residual"].double()).to(t).double()   # as it is kept
        inv = ((x ** 2).sum(1) / x.shape[1] + EPS) ** -0.5
        w = s["weight"].double()
        y = x * inv[:, None] * w
        # a rounding to 8 bits next to a border may fall either way by the norm's last bits: it is of the norm in 32 bits
        out = {"y": _held64(y.float().double()) if kind == "rms8" else y}
        if s["residual"] is not None:
            out["sum"] = s["x"].double() + s["residual"].double()
        if kind == "rms_train":
            dy = s["dy"].double()
            g = dy * w * inv[:, None]
            dx = g - x * ((g * x).sum(1) * inv ** 2 / x.shape[1])[:, None]
            out |= {"dx": dx if s["dsum"] is None else dx + s["dsum"].double(), "dweight": (dy * x * inv[:, None]).sum(0)}
        return out
    if kind.startswith("rotary"):
        out = {x: _turn64(s[x], s["positions"], case, 1) for x in ("q", "k")}
        if kind == "rotary_train":
            out |= {x: _turn64(s[x], s["positions"], case, -1) for x in ("dq", "dk")}
        return out
    return _attention64(s)
