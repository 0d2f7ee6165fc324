"""Training and serving the self-attention: norms of the residual stream, rotary positions, attention over packed sequences.

  rms_norm / rms_norm_backward                  norm after the residual's addition, in the tokens' type or in 8 bits
  rotary / rotary_backward                      q and k turned by positions of one to three axes (time, height, width)
  packed_attention / packed_attention_backward  causal or whole attention, grouped heads, sequences of any lengths; with few
                                                queries a sequence (single tokens over a cache) the keys are split
  rotary_frequencies, grid_positions            what rotary takes, for a model's axes and a grid of tokens

A training pass from one projection's rows to the next, and back:

  qkv = linear(...).view(L, H + 2 Hk, D); q, k = rotary(qkv[:, :H], qkv[:, H:H + Hk], positions, frequencies, axes)
  o, lse = packed_attention(q, k, qkv[:, H + Hk:], cu, causal=True, want_lse=True)
  dq, dk, dv = packed_attention_backward(do, q, k, qkv[:, H + Hk:], o, lse, cu, causal=True)
  dq, dk = rotary_backward(dq, dk, positions, frequencies, axes)

Rows are (L, C), heads (L, H, D), either with a leading batch of 1, on a HIP device. As in train8.py the calls keep no state,
take their temporaries from torch's allocator on the stream they run on (the current one, or `stream`), overlap and are
captured into graphs, and are plain functions: gradients are asked for by name, and a tensor that requires one is refused
where autograd records, as is one that carries a tangent. An `out` must not overlap what the call reads, but where it says so.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
import struct
import threading

import torch
from torch.autograd import forward_ad

from . import Context, _abi
from ._abi import DTYPE_F32, Heads, Packed, lib
from .train8 import Blocks8, _CODE, _check, _current, _detached, _kind, _no_tangents, _out, _out8, _p, _p8, _param, _params, _raw_stream, _refuse, _same

__all__ = ["rms_norm", "rms_norm_backward", "rotary", "rotary_backward", "rotary_frequencies", "grid_positions",
           "packed_attention", "packed_attention_backward"]

_BF16 = (torch.bfloat16,)
_FLOATS = (torch.float32, torch.bfloat16)
_Tensor = torch.Tensor
_recording = torch.is_grad_enabled
_empty_like = torch.empty_like   # a third faster than new_empty; of rows and heads it gives rows and heads, channels innermost


def _unbatched(x, name: str, dims: int):
    if x.dim() == dims + 1:
        if x.shape[0] != 1:
            _refuse(name, "batch 1 only (flatten the batch into the tokens)", _abi.ERR_UNSUPPORTED)
        x = x[0]
    if x.dim() != dims:
        _refuse(name, f"expected {dims} dimensions, got {tuple(x.shape)}")
    return x


def _tensor(x, name: str, dtypes, dims: int):
    """x, a tensor of one of these types that autograd does not wait for, without a leading batch of 1."""
    if not isinstance(x, _Tensor):
        _kind(x, name, _Tensor)
    if x.dtype not in dtypes:
        _refuse(name, f"unsupported dtype {x.dtype} ({' or '.join(str(d)[6:] for d in dtypes)})")
    if x.requires_grad and _recording():
        _detached(x, name)
    return x if x.dim() == dims else _unbatched(x, name, dims)


def _device(first, name: str, *more) -> int:
    """The index of the HIP device of the first operand, which the others (None: skipped) share. Checked after every shape, before a
    pointer reaches the library."""
    if forward_ad._current_level >= 0:
        _no_tangents((first, name), *more)
    if not first.is_cuda:
        _refuse(name, f"expected a tensor on a HIP device, got {first.device}")
    index = first.get_device()
    for t, n in more:
        if t is not None and (t.get_device() if isinstance(t, _Tensor) else t.codes.get_device()) != index:
            _refuse(n, f"expected a tensor on {first.device}, got {t.device}")
    return index


def _handle(index: int):
    found = Context._by_device.get(index)
    return (Context.get(index) if found is None else found).handle


# ----------------------------------------------------------------------------------------------------------------------
# root-mean-square norm
# ----------------------------------------------------------------------------------------------------------------------
def _rows(x, name: str):
    """((L, C) rows of contiguous channels, L, C, elements between rows): a part of a wider tensor's rows, maybe."""
    x = _tensor(x, name, _FLOATS, 2)
    rows, c = x.shape
    if x.is_contiguous() and c > 0:
        return x, rows, c, c
    if c < 1 or (c > 1 and x.stride(1) != 1) or (rows > 1 and x.stride(0) < c):
        _refuse(name, f"expected (L, C) rows of contiguous channels, got {tuple(x.shape)} with strides {x.stride()}")
    return x, rows, c, (x.stride(0) if rows > 1 else c)


def _plain(w, c: int) -> bool:
    """Whether a weight is what _param gives of it, seen at a third of its time."""
    return isinstance(w, _Tensor) and w.dtype is torch.float32 and w.shape == (c,) and w.is_contiguous() and not w.requires_grad


def _like(x, name: str, rows: int, c: int, dtype):
    """A contiguous (rows, c) operand or output of this type, or None."""
    if x is None or (isinstance(x, _Tensor) and x.dtype is dtype and x.dim() == 2 and x.shape == (rows, c) and x.is_contiguous()
                     and not x.requires_grad):
        return x
    return _out(x, name, (rows, c), dtype)


def rms_norm(x: torch.Tensor, weight=None, eps: float = 1e-6, residual=None, want_stats: bool = False, quantized: bool = False,
             stream=None, out=None, out_sum=None):
    """(y, total, rstd): total = x + residual, rounded to their dtype (None without a residual: x itself is what was normed);
    y = total * rstd * weight, rstd = 1 / sqrt(mean(total^2) + eps) over each row's channels, in 32 bits, rounded once to x's
    dtype; with `quantized`, y is a Blocks8 made from the 32-bit values. rstd, (rows) float32, is what rms_norm_backward reads
    (None unless wanted). x: (L, C), its rows at any distance; weight: (C), float32 or bfloat16. `out_sum` may be x or residual,
    `out` x or residual where the other is not."""
    if stream is not None:
        with _current(stream, x):
            return rms_norm(x, weight, eps, residual, want_stats, quantized, out=out, out_sum=out_sum)
    x2, rows, c, stride = _rows(x, "x")
    dtype = x2.dtype
    w = weight if _plain(weight, c) else _param(weight, "weight", c)
    r = _like(residual, "residual", rows, c, dtype)
    if r is None and out_sum is not None:
        _refuse("out_sum", "there is no sum without a residual")
    s = _like(out_sum, "out_sum", rows, c, dtype)
    y = _out8(out, "out", (rows, c)) if quantized else _like(out, "out", rows, c, dtype)
    dev = _device(x2, "x", (w, "weight"), (r, "residual"), (y, "out"), (s, "out_sum"))
    kind = DTYPE_F32
    if w is not None and w.dtype is not torch.float32:
        kind, w, _ = _params(dtype, w)
    total, result = out_sum, out
    if r is not None and s is None:
        total = s = _empty_like(residual)
    rstd = x.new_empty(rows, dtype=torch.float32) if want_stats else None
    yp = yc = ys = None
    if quantized:
        if y is None:
            result = y = Blocks8.empty(rows, c, x2.device)
        yc, ys = _p8(y)
    else:
        if y is None:
            result = y = _empty_like(x) if stride == c else x.new_empty(x.shape)
        yp = y.data_ptr()
        if s is out_sum is not None and yp == s.data_ptr() and rows:
            _refuse("out", "the norm and the sum need memory of their own")
    rc = lib.fvsr_rms_norm(_handle(dev), _CODE[dtype], x2.data_ptr(), stride, _p(r), rows, c, float(eps), kind, _p(w), yp, yc, ys, _p(s),
                           _p(rstd), _raw_stream(dev))
    if rc:
        _check(rc, "fvsr_rms_norm")
    return result, total, rstd


_grad_workspace = functools.lru_cache(256)(lib.fvsr_rms_norm_backward_workspace)


def rms_norm_backward(dy: torch.Tensor, total: torch.Tensor, rstd: torch.Tensor, weight=None, dsum=None,
                      want_weight: bool = True, stream=None, out=None):
    """(dx, dweight) of rms_norm; dx is the gradient of x and of the residual alike. total: the sum that it returned, or the x that
    it normed; rstd: what it returned; weight: the one that it was given; dsum: the gradient that reached the sum from elsewhere
    (the rest of the residual stream). dweight, float32 (C), is summed in a fixed order (None without `want_weight`). `out` may be
    dy or dsum itself."""
    if stream is not None:
        with _current(stream, dy):
            return rms_norm_backward(dy, total, rstd, weight, dsum, want_weight, out=out)
    d2, rows, c, stride = _rows(dy, "dy")
    dtype = d2.dtype
    if stride != c:
        _refuse("dy", "expected a contiguous tensor")
    t2, n, m, stride = _rows(total, "total")
    if (n, m) != (rows, c) or t2.dtype is not dtype:
        _same("total", t2.shape, (rows, c), t2.dtype, dtype)
    if not isinstance(rstd, _Tensor) or rstd.shape != (rows,) or rstd.dtype is not torch.float32:
        _same("rstd", _kind(rstd, "rstd", _Tensor).shape, (rows,), rstd.dtype, torch.float32)
    _detached(rstd, "rstd")
    if not rstd.is_contiguous():
        _refuse("rstd", "expected a contiguous tensor")
    w = weight if _plain(weight, c) else _param(weight, "weight", c)
    ds = _like(dsum, "dsum", rows, c, dtype)
    o = _like(out, "out", rows, c, dtype)
    dev = _device(d2, "dy", (t2, "total"), (rstd, "rstd"), (w, "weight"), (ds, "dsum"), (o, "out"))
    kind = DTYPE_F32
    if w is not None and w.dtype is not torch.float32:
        kind, w, _ = _params(dtype, w)
    dx = out
    if o is None:
        dx = o = _empty_like(dy)
    dw = ws = None
    nbytes = 0
    if want_weight:
        nbytes = _grad_workspace(rows, c)
        dw = _empty_like(w) if kind == DTYPE_F32 and w is not None and w.dim() == 1 else dy.new_empty(c, dtype=torch.float32)
        ws = dy.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    rc = lib.fvsr_rms_norm_backward(_handle(dev), _CODE[dtype], d2.data_ptr(), t2.data_ptr(), stride, rstd.data_ptr(), _p(ds), rows,
                                    c, kind, _p(w), o.data_ptr(), _p(dw), _p(ws), nbytes, _raw_stream(dev))
    if rc:
        _check(rc, "fvsr_rms_norm_backward")
    return dx, dw


# ----------------------------------------------------------------------------------------------------------------------
# heads
# ----------------------------------------------------------------------------------------------------------------------
class _Structs(threading.local):
    """A thread's memory for the structs of one call, which the library reads before it returns: filled by struct.pack_into, at a
    tenth of the time that ctypes' fields take."""
    views = [struct.Struct("@" + n * "Piqq") for n in range(9)]
    packed = struct.Struct("@PPPiqqiif")

    def __init__(self):
        self.memory = C.create_string_buffer(1024)
        self.at = [C.addressof(self.memory) + C.sizeof(Heads) * i for i in range(9)]
        self.seqs = C.addressof(self.memory) + 640

    def heads(self, *x):
        """The addresses of the structs of these heads, as _heads gives them."""
        fields = []
        for t, _, h, _, ts, hs in x:
            fields += (t.data_ptr(), h, ts, hs)
        self.views[len(x)].pack_into(self.memory, 0, *fields)
        return self.at[:len(x)]

    def sequences(self, *fields) -> int:
        self.packed.pack_into(self.memory, 640, *fields)
        return self.seqs


_structs = _Structs()
assert all(s.size == n * C.sizeof(Heads) <= 640 for n, s in enumerate(_Structs.views)) and _Structs.packed.size <= C.sizeof(Packed) <= 384


def _heads(x, name: str, dtypes):
    """((L, H, D) heads of contiguous channels, L, H, D, elements between tokens, between heads): heads and tokens at any distance
    (parts of one projection's rows)."""
    if not isinstance(x, _Tensor) or x.dim() != 3 or x.dtype not in dtypes or x.requires_grad:
        x = _tensor(x, name, dtypes, 3)
    n, h, d = x.shape
    if x.is_contiguous() and h > 0 and d > 0:
        return x, n, h, d, h * d, d
    ts, hs, cs = x.stride()
    if h < 1 or d < 1 or (d > 1 and cs != 1):
        _refuse(name, f"expected (L, H, D) heads of contiguous channels, got {tuple(x.shape)} with strides {x.stride()}")
    return x, n, h, d, (ts if n > 1 else h * d), (hs if h > 1 else d)


def _made(x, heads):
    """New heads like x, whose `heads` _heads has given, as it gives them."""
    o = _empty_like(x)
    _, n, h, d, ts, hs = heads
    if ts == h * d and hs == d and x.is_contiguous():
        return o, n, h, d, ts, hs
    ts, hs, cs = o.stride()[-3:]
    if cs != 1:   # of windows that overlap, the dimension with the shortest stride is innermost
        o = x.new_empty(x.shape)
        ts, hs = h * d, d
    return o, n, h, d, (ts if n > 1 else h * d), (hs if h > 1 else d)


def _out_heads(out, name: str, n: int, h: int, d: int, dtype):
    """A caller's output of heads, as _heads gives it: no two elements at one address."""
    o = _heads(out, name, (dtype,))
    _same(name, o[0].shape, (n, h, d))
    ts, hs = (o[4] if n > 1 else 1 << 62), (o[5] if h > 1 else 1 << 62)
    if not (hs >= d and ts >= d and (n == 1 or h == 1 or ts >= (h - 1) * hs + d or hs >= (n - 1) * ts + d)):
        _refuse(name, f"rows that overlap: {tuple(o[0].shape)} with strides {o[0].stride()}")
    return o


# ----------------------------------------------------------------------------------------------------------------------
# rotary positions
# ----------------------------------------------------------------------------------------------------------------------
def rotary_frequencies(axes, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """(sum of axes) float64: pair i of an axis with p pairs turns by theta^(-i / p) radians a position. The DiT's axes are
    (22, 21, 21): time, height, width."""
    f = [theta ** (-torch.arange(int(p), dtype=torch.float64) / int(p)) for p in axes]
    return torch.cat(f).to(device)


def grid_positions(f: int, h: int, w: int, t0: int = 0, device="cuda") -> torch.Tensor:
    """(3, f * h * w) int32: time (from t0 on), row and column of each token of a grid in natural (f, h, w) order."""
    t, y, x = (torch.arange(a, a + n, dtype=torch.int32, device=device) for a, n in ((t0, f), (0, h), (0, w)))
    return torch.stack([g.reshape(-1) for g in torch.meshgrid(t, y, x, indexing="ij")])


def rotary(q: torch.Tensor, k, positions: torch.Tensor, frequencies: torch.Tensor, axes, halves: bool = False, stream=None,
           out=None):
    """(q', k'): q (L, H, D) and k (L, Hk, D), or None, float32 or bfloat16, with each head's pair i turned by
    positions[axis of i] * frequencies[i] radians: (a, b) becomes (a cos - b sin, a sin + b cos). Pairs are neighbours, (2 i,
    2 i + 1), or with `halves` (i, pairs + i); channels past the pairs are copied. positions: (axes, L), int32 or int64;
    frequencies: (pairs) float64; axes: the pairs of each of one to three axes. Angles in 64 bits, the rest in 32, rounded once.
    `out`: a pair of tensors for the results, which may be q and k themselves."""
    return _turn(q, k, positions, frequencies, axes, halves, stream, out, 0)


def rotary_backward(dq: torch.Tensor, dk, positions: torch.Tensor, frequencies: torch.Tensor, axes, halves: bool = False,
                    stream=None, out=None):
    """The gradients of q and k from those of rotary's results: turned back. Arguments as there."""
    return _turn(dq, dk, positions, frequencies, axes, halves, stream, out, 1)


@functools.lru_cache(64)
def _axes(axes: tuple):
    """(number of axes, pairs, the pairs of each as the library reads them) of whole numbers."""
    if not 1 <= len(axes) <= 3 or min(axes) < 0 or sum(axes) < 1:
        raise ValueError
    return len(axes), sum(axes), struct.pack(f"{len(axes)}i", *axes)


def _turn(q, k, positions, frequencies, axes, halves, stream, out, back):
    if stream is not None:
        with _current(stream, q):
            return _turn(q, k, positions, frequencies, axes, halves, None, out, back)
    q3 = _heads(q, "q", _FLOATS)
    _, n, h, d, _, _ = q3
    dtype = q3[0].dtype
    k3 = None
    if k is not None:
        k3 = _heads(k, "k", (dtype,))
        if k3[1] != n or k3[3] != d:
            _refuse("k", f"expected {n} tokens and {d} channels a head as q has, got {tuple(k3[0].shape)}")
    try:
        axes = tuple(axes)
        whole = tuple(map(int, axes))   # plain numbers: what the cache knows them by
        if whole != axes:
            raise ValueError
        count, pairs, packed = _axes(whole)
    except (TypeError, ValueError, OverflowError, struct.error):
        count, pairs = 0, 0
    if not count or 2 * pairs > d or d % 2:
        _refuse("axes", f"expected 1 to 3 axes of 1 to {d // 2} pairs together, got {axes} for {d} channels")
    wide = _kind(positions, "positions", _Tensor).dtype is torch.int64
    if not wide and positions.dtype is not torch.int32:
        _refuse("positions", f"unsupported dtype {positions.dtype} (int32 or int64)")
    if positions.shape != (count, n) and not (count == 1 and positions.shape == (n,)):
        _refuse("positions", f"expected ({count}, {n}), got {tuple(positions.shape)}")
    if not isinstance(frequencies, _Tensor) or frequencies.shape != (pairs,) or frequencies.dtype is not torch.float64:
        _same("frequencies", _kind(frequencies, "frequencies", _Tensor).shape, (pairs,), frequencies.dtype, torch.float64)
    _detached(frequencies, "frequencies")
    if not (positions.is_contiguous() and frequencies.is_contiguous()):
        _refuse("positions", "expected contiguous positions and frequencies")
    oq = ok = yq = yk = None
    if out is not None:
        if not isinstance(out, (tuple, list)) or len(out) != 2:
            _refuse("out", "expected a pair of tensors (or None), for q and k")
        oq, ok = out
        if ok is not None and k3 is None:
            _refuse("out", "there is no k to write")
        yq = None if oq is None else _out_heads(oq, "out", n, h, d, dtype)
        yk = None if ok is None else _out_heads(ok, "out", n, k3[2], d, dtype)
        if n and yq and yk and yq[0].data_ptr() == yk[0].data_ptr():
            _refuse("out", "q's and k's results need memory of their own")
    dev = _device(q3[0], "q", (k3 and k3[0], "k"), (positions, "positions"), (frequencies, "frequencies"), (yq and yq[0], "out"),
                  (yk and yk[0], "out"))
    if yq is None:
        yq = _made(q, q3)
        oq = yq[0]
    if k3 is None:
        (a, b), e, f = _structs.heads(q3, yq), None, None
    else:
        if yk is None:
            yk = _made(k, k3)
            ok = yk[0]
        a, b, e, f = _structs.heads(q3, yq, k3, yk)
    rc = lib.fvsr_rotary(_handle(dev), _CODE[dtype], a, b, e, f, n, d, positions.data_ptr(), wide, frequencies.data_ptr(), count, packed,
                         bool(halves), back, _raw_stream(dev))
    if rc:
        _check(rc, "fvsr_rotary")
    return oq, ok


# ----------------------------------------------------------------------------------------------------------------------
# attention over packed sequences
# ----------------------------------------------------------------------------------------------------------------------
def _aligned(x) -> bool:
    """Whether the kernels can read heads as they lie: 16-byte aligned rows."""
    return not (x[0].data_ptr() & 15 or x[4] & 7 or x[5] & 7)


def _ready(x):
    """Heads as the kernels read them: as they lie, or a copy."""
    if _aligned(x):
        return x
    _, n, h, d, _, _ = x
    return x[0].clone(memory_format=torch.contiguous_format), n, h, d, h * d, d


def _offsets(cu, name: str, n=None):
    if not isinstance(cu, _Tensor) or cu.dtype is not torch.int32:
        _refuse(name, f"unsupported dtype {_kind(cu, name, _Tensor).dtype} (int32)")
    m = cu.numel()
    if cu.dim() != 1 or not cu.is_contiguous() or (m < 2 if n is None else m != n):
        _refuse(name, f"expected {'at least 2' if n is None else n} contiguous offsets, got {tuple(cu.shape)}")
    return m


def _sequences(q, k, v, cu_q, cu_k, used_k, scale):
    """(q, k, v, as _heads gives them, cu_k, offsets, scale), checked."""
    q, k, v = _heads(q, "q", _BF16), _heads(k, "k", _BF16), _heads(v, "v", _BF16)
    n, h, d = q[1:4]
    if d % 8 or d > 128:
        _refuse("q", f"{d} channels a head: a multiple of 8, at most 128, is needed", _abi.ERR_UNSUPPORTED)
    if k[3] != d or h % k[2]:
        _refuse("k", f"expected heads of {d} channels that divide q's {h}, got {tuple(k[0].shape)}")
    if v[1:4] != k[1:4]:
        _same("v", v[0].shape, k[0].shape)
    m = _offsets(cu_q, "cu_q")
    if cu_k is None:
        if k[1] != n:
            _refuse("k", f"expected q's {n} tokens where there is no cu_k, got {k[1]}")
        cu_k = cu_q
    else:
        _offsets(cu_k, "cu_k", m)
    if used_k is not None:
        _offsets(used_k, "used_k", m - 1)
    if scale is None:
        scale = d ** -0.5
    else:
        scale = float(scale)
        if not (scale > 0 and math.isfinite(scale)):
            _refuse("scale", f"expected a positive finite number, got {scale}")
    return q, k, v, cu_k, m, scale


def _out_ready(out, name: str, like):
    o = _out_heads(out, name, *like[1:4], like[0].dtype)
    if not _aligned(o):
        _refuse(name, "expected 16-byte aligned rows")
    return o


@functools.lru_cache(256)
def _workspace(backward: bool, sequences: int, tokens_q: int, tokens_k: int, channels: int, causal: bool, heads: int, kv_heads: int) -> int:
    p = Packed(None, None, None, sequences, tokens_q, tokens_k, channels, causal, 1.0)
    size = lib.fvsr_packed_attention_backward_workspace if backward else lib.fvsr_packed_attention_workspace
    return size(C.byref(p), heads, kv_heads)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, cu_k=None, causal: bool = False,
                     scale=None, used_k=None, want_lse: bool = False, stream=None, out=None):
    """(o, lse): o (Lq, H, D) = softmax(scale q k^T) v within each sequence, from bfloat16 q (Lq, H, D), k and v (Lk, Hk, D), D a
    multiple of 8 up to 128; query heads g * h .. g * h + g - 1, g = H / Hk, share key head h. Sequence b has the queries cu_q[b] ..
    cu_q[b + 1] - 1 and the keys cu_k[b] .. cu_k[b + 1] - 1 (cu_q's without cu_k), of which the first used_k[b] count where used_k is
    given (a cache with room); all int32, read on the device when the kernels run. Query i of m sees all n keys, or, `causal`, the
    first i + 1 + n - m: a query over a cache that holds its own key is causal. One that sees none gives zeros. scale: 1 / sqrt(D)
    unless given. lse: (H, Lq) float32, log(sum(exp(scores))), which packed_attention_backward reads (None unless wanted). Rows of no
    sequence are zeros, in an `out` as they were, and -inf in lse. Operands may be parts of wider rows; parts that are not 16-byte aligned
    are copied first."""
    if stream is not None:
        with _current(stream, q):
            return packed_attention(q, k, v, cu_q, cu_k, causal, scale, used_k, want_lse, out=out)
    q3, k3, v3, ck, m, scale = _sequences(q, k, v, cu_q, cu_k, used_k, scale)
    o3 = None if out is None else _out_ready(out, "out", q3)
    dev = _device(q3[0], "q", (k3[0], "k"), (v3[0], "v"), (cu_q, "cu_q"), (ck, "cu_k"), (used_k, "used_k"), (o3 and o3[0], "out"))
    n, h, d = q3[1:4]
    o = out
    if o3 is None:
        o3 = _made(q, q3)
        o = o3[0]
    lse = q.new_empty((h, n), dtype=torch.float32) if want_lse else None
    nbytes = _workspace(False, m - 1, n, k3[1], d, bool(causal), h, k3[2])
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    q3, k3, v3 = _ready(q3), _ready(k3), _ready(v3)
    clear = 1 if out is None else _abi.CLEAR_LSE if want_lse else 0   # a new lse has -inf for rows of no sequence either way
    st = _structs
    p = st.sequences(cu_q.data_ptr(), ck.data_ptr(), 0 if used_k is None else used_k.data_ptr(), m - 1, n, k3[1], d, bool(causal), scale)
    rc = lib.fvsr_packed_attention(_handle(dev), p, *st.heads(q3, k3, v3, o3), _p(lse), clear, _p(ws), nbytes, _raw_stream(dev))
    if rc:
        _check(rc, "fvsr_packed_attention")
    return o, lse


def packed_attention_backward(do: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor,
                              lse: torch.Tensor, cu_q: torch.Tensor, cu_k=None, causal: bool = False, scale=None, used_k=None,
                              stream=None, out=None):
    """(dq, dk, dv) of packed_attention from the gradient of its o, its operands and its results. dk and dv are summed over the query
    heads that share them, in a fixed order. Keys that no query sees have gradients of zero. `out`: three tensors for the results
    (parts of one projection's gradient, say); rows of no sequence are left as they were there, and zeros otherwise."""
    if stream is not None:
        with _current(stream, q):
            return packed_attention_backward(do, q, k, v, o, lse, cu_q, cu_k, causal, scale, used_k, out=out)
    q3, k3, v3, ck, m, scale = _sequences(q, k, v, cu_q, cu_k, used_k, scale)
    n, h, d = q3[1:4]
    g3, o3 = _heads(do, "do", _BF16), _heads(o, "o", _BF16)
    for x, name in ((g3, "do"), (o3, "o")):
        if x[1:4] != q3[1:4]:
            _same(name, x[0].shape, q3[0].shape)
    if not isinstance(lse, _Tensor) or lse.shape != (h, n) or lse.dtype is not torch.float32:
        _same("lse", _kind(lse, "lse", _Tensor).shape, (h, n), lse.dtype, torch.float32)
    _detached(lse, "lse")
    if not lse.is_contiguous():
        _refuse("lse", "expected a contiguous tensor")
    made = (None, None, None)
    if out is not None:
        if not isinstance(out, (tuple, list)) or len(out) != 3 or any(x is None for x in out):
            _refuse("out", "expected three tensors, for dq, dk and dv")
        out = tuple(out)
        made = [_out_ready(x, "out", like) for x, like in zip(out, (q3, k3, v3))]
        at = [x[0].data_ptr() for x in made if x[1]]
        if len(set(at)) < len(at):
            _refuse("out", "the gradients need memory of their own")
    dev = _device(q3[0], "q", (k3[0], "k"), (v3[0], "v"), (g3[0], "do"), (o3[0], "o"), (lse, "lse"), (cu_q, "cu_q"), (ck, "cu_k"),
                  (used_k, "used_k"), *((x and x[0], "out") for x in made))
    grads = out
    if out is None:
        made = _made(q, q3), _made(k, k3), _made(v, v3)
        grads = tuple(x[0] for x in made)
    nbytes = _workspace(True, m - 1, n, k3[1], d, bool(causal), h, k3[2])
    ws = q.new_empty(nbytes, dtype=torch.uint8)
    g3, q3, k3, v3, o3 = _ready(g3), _ready(q3), _ready(k3), _ready(v3), _ready(o3)
    st = _structs
    p = st.sequences(cu_q.data_ptr(), ck.data_ptr(), 0 if used_k is None else used_k.data_ptr(), m - 1, n, k3[1], d, bool(causal), scale)
    a = st.heads(g3, q3, k3, v3, o3, *made)
    rc = lib.fvsr_packed_attention_backward(_handle(dev), p, *a[:5], lse.data_ptr(), *a[5:], out is None, ws.data_ptr(), nbytes,
                                            _raw_stream(dev))
    if rc:
        _check(rc, "fvsr_packed_attention_backward")
    return grads
