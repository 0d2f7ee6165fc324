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
where autograd records. An `out` must not overlap what the call reads, but where it says so.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _abi
from ._abi import FVSRError, Heads, Packed, lib
from .train8 import (Blocks8, _CODE, _check, _ctx, _current, _detached, _kind, _one_device, _out, _out8, _p, _p8, _param,
                     _params, _raw_stream, _refuse, _same)

__all__ = ["rms_norm", "rms_norm_backward", "rotary", "rotary_backward", "rotary_frequencies", "grid_positions",
           "packed_attention", "packed_attention_backward"]

_BF16 = (torch.bfloat16,)


# ----------------------------------------------------------------------------------------------------------------------
# root-mean-square norm
# ----------------------------------------------------------------------------------------------------------------------
def _rows(x, name: str) -> torch.Tensor:
    """(L, C) rows of contiguous channels, at any distance from each other (a part of a wider tensor's rows)."""
    if _kind(x, name, torch.Tensor).dtype not in _CODE:
        _refuse(name, f"unsupported dtype {x.dtype} (float32 or bfloat16)")
    _detached(x, name)
    x = _unbatched(x, name, 2)
    if x.shape[1] < 1 or (x.shape[1] > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        _refuse(name, f"expected (L, C) rows of contiguous channels, got {tuple(x.shape)} with strides {x.stride()}")
    return x


def _unbatched(x, name: str, dims: int):
    if x.dim() == dims + 1:
        if x.shape[0] != 1:
            _refuse(name, "batch 1 only (flatten the batch into the tokens)", _abi.ERR_UNSUPPORTED)
        x = x[0]
    if x.dim() != dims:
        _refuse(name, f"expected {dims} dimensions, got {tuple(x.shape)}")
    return x


def _row_stride(x) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


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
    x2 = _rows(x, "x")
    rows, c = x2.shape
    weight = _param(weight, "weight", c)
    r = _out(residual, "residual", (rows, c), x2.dtype)
    if r is None and out_sum is not None:
        _refuse("out_sum", "there is no sum without a residual")
    s = _out(out_sum, "out_sum", (rows, c), x2.dtype)
    y = _out8(out, "out", (rows, c)) if quantized else _out(out, "out", (rows, c), x2.dtype)
    dev = _one_device(x2, "x", (weight, "weight"), (r, "residual"), (out, "out"), (s, "out_sum"))
    kind, w, _ = _params(x2.dtype, weight)
    total = out_sum
    if r is not None and s is None:
        total = s = torch.empty(x.shape, dtype=x.dtype, device=dev)
    rstd = torch.empty(rows, dtype=torch.float32, device=dev) if want_stats else None
    result = out
    if quantized:
        if result is None:
            result = Blocks8.empty(rows, c, dev)
        yp, (yc, ys) = None, _p8(result)
    else:
        if y is None:
            result = y = torch.empty(x.shape, dtype=x.dtype, device=dev)
        if s is not None and y.data_ptr() == s.data_ptr() and rows:
            _refuse("out", "the norm and the sum need memory of their own")
        yp, yc, ys = y.data_ptr(), None, None
    _check(lib.fvsr_rms_norm(_ctx(dev), _CODE[x2.dtype], x2.data_ptr(), _row_stride(x2), _p(r), rows, c, float(eps), kind, _p(w),
                             yp, yc, ys, _p(s), _p(rstd), _raw_stream(dev.index)), "fvsr_rms_norm")
    return result, total, rstd


def rms_norm_backward(dy: torch.Tensor, total: torch.Tensor, rstd: torch.Tensor, weight=None, dsum=None,
                      want_weight: bool = True, stream=None, out=None):
    """(dx, dweight) of rms_norm; dx is the gradient of x and of the residual alike. total: the sum that it returned, or the x that
    it normed; rstd: what it returned; weight: the one that it was given; dsum: the gradient that reached the sum from elsewhere
    (the rest of the residual stream). dweight, float32 (C), is summed in a fixed order (None without `want_weight`). `out` may be
    dy or dsum itself."""
    if stream is not None:
        with _current(stream, dy):
            return rms_norm_backward(dy, total, rstd, weight, dsum, want_weight, out=out)
    d2 = _rows(dy, "dy")
    if not d2.is_contiguous():
        _refuse("dy", "expected a contiguous tensor")
    rows, c = d2.shape
    t2 = _rows(total, "total")
    _same("total", t2.shape, (rows, c), t2.dtype, d2.dtype)
    _same("rstd", _kind(rstd, "rstd", torch.Tensor).shape, (rows,), rstd.dtype, torch.float32)
    _detached(rstd, "rstd")
    if not rstd.is_contiguous():
        _refuse("rstd", "expected a contiguous tensor")
    weight = _param(weight, "weight", c)
    ds = _out(dsum, "dsum", (rows, c), d2.dtype)
    o = _out(out, "out", (rows, c), d2.dtype)
    dev = _one_device(d2, "dy", (t2, "total"), (rstd, "rstd"), (weight, "weight"), (ds, "dsum"), (o, "out"))
    kind, w, _ = _params(d2.dtype, weight)
    dx = torch.empty(dy.shape, dtype=dy.dtype, device=dev) if o is None else o
    dw = ws = None
    nbytes = 0
    if want_weight:
        nbytes = lib.fvsr_rms_norm_backward_workspace(rows, c)
        dw = torch.empty(c, dtype=torch.float32, device=dev)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _check(lib.fvsr_rms_norm_backward(_ctx(dev), _CODE[d2.dtype], d2.data_ptr(), t2.data_ptr(), _row_stride(t2), rstd.data_ptr(),
                                      _p(ds), rows, c, kind, _p(w), dx.data_ptr(), _p(dw), _p(ws), nbytes, _raw_stream(dev.index)),
           "fvsr_rms_norm_backward")
    return (dx if out is None else out), dw


# ----------------------------------------------------------------------------------------------------------------------
# heads
# ----------------------------------------------------------------------------------------------------------------------
def _heads(x, name: str, dtypes) -> torch.Tensor:
    """(L, H, D) with contiguous channels; heads and tokens at any distance (parts of one projection's rows)."""
    if _kind(x, name, torch.Tensor).dtype not in dtypes:
        _refuse(name, f"unsupported dtype {x.dtype} ({' or '.join(str(d)[6:] for d in dtypes)})")
    _detached(x, name)
    x = _unbatched(x, name, 3)
    if x.shape[1] < 1 or x.shape[2] < 1 or (x.shape[2] > 1 and x.stride(2) != 1):
        _refuse(name, f"expected (L, H, D) heads of contiguous channels, got {tuple(x.shape)} with strides {x.stride()}")
    return x


def _out_heads(out, name: str, like: torch.Tensor):
    """A caller's output of heads (or None): no two elements at one address."""
    if out is None:
        return None
    o = _heads(out, name, (like.dtype,))
    _same(name, o.shape, like.shape)
    n, h, d = o.shape
    ts, hs = (o.stride(0) if n > 1 else 1 << 62), (o.stride(1) if h > 1 else 1 << 62)
    if not (hs >= d and (n == 1 or h == 1 or ts >= (h - 1) * hs + d or hs >= (n - 1) * ts + d) and ts >= d):
        _refuse(name, f"rows that overlap: {tuple(o.shape)} with strides {o.stride()}")
    return o


def _view(x) -> Heads:
    n, h, d = x.shape
    return Heads(x.data_ptr(), h, x.stride(0) if n > 1 else h * d, x.stride(1) if h > 1 else d)


def _ref(view):
    return None if view is None else C.byref(view)


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


def _turn(q, k, positions, frequencies, axes, halves, stream, out, back):
    if stream is not None:
        with _current(stream, q):
            return _turn(q, k, positions, frequencies, axes, halves, None, out, back)
    q3 = _heads(q, "q", tuple(_CODE))
    k3 = None if k is None else _heads(k, "k", (q3.dtype,))
    n, _, d = q3.shape
    if k3 is not None and (k3.shape[0], k3.shape[2]) != (n, d):
        _refuse("k", f"expected {n} tokens and {d} channels a head as q has, got {tuple(k3.shape)}")
    try:
        axes = tuple(int(p) for p in axes)
    except (TypeError, ValueError):
        _refuse("axes", "expected the pairs of each axis")
    if not 1 <= len(axes) <= 3 or min(axes) < 0 or not 1 <= sum(axes) <= d // 2 or d % 2:
        _refuse("axes", f"expected 1 to 3 axes of 1 to {d // 2} pairs together, got {axes} for {d} channels")
    if _kind(positions, "positions", torch.Tensor).dtype not in (torch.int32, torch.int64):
        _refuse("positions", f"unsupported dtype {positions.dtype} (int32 or int64)")
    if tuple(positions.shape) != (len(axes), n) and not (len(axes) == 1 and tuple(positions.shape) == (n,)):
        _refuse("positions", f"expected ({len(axes)}, {n}), got {tuple(positions.shape)}")
    _same("frequencies", _kind(frequencies, "frequencies", torch.Tensor).shape, (sum(axes),), frequencies.dtype, torch.float64)
    _detached(frequencies, "frequencies")
    if not (positions.is_contiguous() and frequencies.is_contiguous()):
        _refuse("positions", "expected contiguous positions and frequencies")
    oq, ok = out if out is not None else (None, None)
    if ok is not None and k3 is None:
        _refuse("out", "there is no k to write")
    yq, yk = _out_heads(oq, "out", q3), None if k3 is None else _out_heads(ok, "out", k3)
    dev = _one_device(q3, "q", (k3, "k"), (positions, "positions"), (frequencies, "frequencies"), (yq, "out"), (yk, "out"))
    if yq is None:
        oq = torch.empty(q.shape, dtype=q.dtype, device=dev)
        yq = oq.view(q3.shape)
    if k3 is not None and yk is None:
        ok = torch.empty(k.shape, dtype=k.dtype, device=dev)
        yk = ok.view(k3.shape)
    a, b = _view(q3), _view(yq)
    e, f = (None, None) if k3 is None else (_view(k3), _view(yk))
    _check(lib.fvsr_rotary(_ctx(dev), _CODE[q3.dtype], C.byref(a), C.byref(b), _ref(e), _ref(f), n, d, positions.data_ptr(),
                           positions.dtype == torch.int64, frequencies.data_ptr(), len(axes), (C.c_int32 * len(axes))(*axes),
                           bool(halves), back, _raw_stream(dev.index)), "fvsr_rotary")
    return oq, ok


# ----------------------------------------------------------------------------------------------------------------------
# attention over packed sequences
# ----------------------------------------------------------------------------------------------------------------------
def _aligned(x):
    """x, or a copy of it, as the kernels read it: 16-byte aligned rows."""
    n, h, _ = x.shape
    if x.data_ptr() & 15 or (n > 1 and x.stride(0) & 7) or (h > 1 and x.stride(1) & 7):
        return x.clone(memory_format=torch.contiguous_format)
    return x


def _offsets(cu, name: str, n=None):
    if _kind(cu, name, torch.Tensor).dtype != torch.int32:
        _refuse(name, f"unsupported dtype {cu.dtype} (int32)")
    if cu.dim() != 1 or not cu.is_contiguous() or (cu.numel() < 2 if n is None else cu.numel() != n):
        _refuse(name, f"expected {'at least 2' if n is None else n} contiguous offsets, got {tuple(cu.shape)}")
    return cu


def _sequences(q, k, v, cu_q, cu_k, used_k, scale):
    """(q, k, v, cu_k, scale), checked."""
    q, k, v = _heads(q, "q", _BF16), _heads(k, "k", _BF16), _heads(v, "v", _BF16)
    d = q.shape[2]
    if d % 8 or d > 128:
        _refuse("q", f"{d} channels a head: a multiple of 8, at most 128, is needed", _abi.ERR_UNSUPPORTED)
    if k.shape[2] != d or q.shape[1] % k.shape[1]:
        _refuse("k", f"expected heads of {d} channels that divide q's {q.shape[1]}, got {tuple(k.shape)}")
    _same("v", v.shape, k.shape)
    _offsets(cu_q, "cu_q")
    if cu_k is None:
        if k.shape[0] != q.shape[0]:
            _refuse("k", f"expected q's {q.shape[0]} tokens where there is no cu_k, got {k.shape[0]}")
        cu_k = cu_q
    else:
        _offsets(cu_k, "cu_k", cu_q.numel())
    if used_k is not None:
        _offsets(used_k, "used_k", cu_q.numel() - 1)
    scale = 1 / math.sqrt(d) if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        _refuse("scale", f"expected a positive finite number, got {scale}")
    return q, k, v, cu_k, scale


def _out_aligned(out, name: str, like):
    o = _out_heads(out, name, like)
    if o is not None and _aligned(o) is not o:
        _refuse(name, "expected 16-byte aligned rows")
    return o


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, cu_k=None, causal: bool = False,
                     scale=None, used_k=None, want_lse: bool = False, stream=None, out=None):
    """(o, lse): o (Lq, H, D) = softmax(scale q k^T) v within each sequence, from bfloat16 q (Lq, H, D), k and v (Lk, Hk, D), D a
    multiple of 8 up to 128; query heads g * h .. g * h + g - 1, g = H / Hk, share key head h. Sequence b has the queries cu_q[b] ..
    cu_q[b + 1] - 1 and the keys cu_k[b] .. cu_k[b + 1] - 1 (cu_q's without cu_k), of which the first used_k[b] count where used_k is
    given (a cache with room); all int32, read on the device when the kernels run. Query i of m sees all n keys, or, `causal`, the
    first i + 1 + n - m: a query over a cache that holds its own key is causal. One that sees none gives zeros. scale: 1 / sqrt(D)
    unless given. lse: (H, Lq) float32, log(sum(exp(scores))), which packed_attention_backward reads (None unless wanted). Rows of no
    sequence are zeros, in an `out` as they were. Operands may be parts of wider rows; parts that are not 16-byte aligned
    are copied first."""
    if stream is not None:
        with _current(stream, q):
            return packed_attention(q, k, v, cu_q, cu_k, causal, scale, used_k, want_lse, out=out)
    q3, k3, v3, ck, scale = _sequences(q, k, v, cu_q, cu_k, used_k, scale)
    o3 = _out_aligned(out, "out", q3)
    dev = _one_device(q3, "q", (k3, "k"), (v3, "v"), (cu_q, "cu_q"), (ck, "cu_k"), (used_k, "used_k"), (o3, "out"))
    q3, k3, v3 = _aligned(q3), _aligned(k3), _aligned(v3)
    n, h, d = q3.shape
    o = out
    if o3 is None:
        o = torch.empty(q.shape, dtype=q.dtype, device=dev)
        o3 = o.view(n, h, d)
    lse = torch.empty(h, n, dtype=torch.float32, device=dev) if want_lse else None
    p = Packed(cu_q.data_ptr(), ck.data_ptr(), _p(used_k), cu_q.numel() - 1, n, k3.shape[0], d, bool(causal), scale)
    hk = k3.shape[1]
    nbytes = lib.fvsr_packed_attention_workspace(C.byref(p), h, hk)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    a, b, c, e = _view(q3), _view(k3), _view(v3), _view(o3)
    _check(lib.fvsr_packed_attention(_ctx(dev), C.byref(p), C.byref(a), C.byref(b), C.byref(c), C.byref(e), _p(lse), out is None,
                                     _p(ws), nbytes, _raw_stream(dev.index)), "fvsr_packed_attention")
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
    q3, k3, v3, ck, scale = _sequences(q, k, v, cu_q, cu_k, used_k, scale)
    g3, o3 = _heads(do, "do", _BF16), _heads(o, "o", _BF16)
    _same("do", g3.shape, q3.shape)
    _same("o", o3.shape, q3.shape)
    n, h, d = q3.shape
    _same("lse", _kind(lse, "lse", torch.Tensor).shape, (h, n), lse.dtype, torch.float32)
    _detached(lse, "lse")
    if not lse.is_contiguous():
        _refuse("lse", "expected a contiguous tensor")
    outs = (None, None, None) if out is None else tuple(out)
    if len(outs) != 3 or (out is not None and any(x is None for x in outs)):
        _refuse("out", "expected three tensors, for dq, dk and dv")
    views = [_out_aligned(x, "out", like) for x, like in zip(outs, (q3, k3, v3))]
    dev = _one_device(q3, "q", (k3, "k"), (v3, "v"), (g3, "do"), (o3, "o"), (lse, "lse"), (cu_q, "cu_q"), (ck, "cu_k"),
                      (used_k, "used_k"), *((x, "out") for x in views))
    if out is None:
        outs = tuple(torch.empty(x.shape, dtype=x.dtype, device=dev) for x in (q, k, v))
        views = [x.view(y.shape) for x, y in zip(outs, (q3, k3, v3))]
    q3, k3, v3, g3, o3 = (_aligned(x) for x in (q3, k3, v3, g3, o3))
    p = Packed(cu_q.data_ptr(), ck.data_ptr(), _p(used_k), cu_q.numel() - 1, n, k3.shape[0], d, bool(causal), scale)
    nbytes = lib.fvsr_packed_attention_backward_workspace(C.byref(p), h, k3.shape[1])
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    given = [_view(x) for x in (g3, q3, k3, v3, o3)]
    made = [_view(x) for x in views]
    _check(lib.fvsr_packed_attention_backward(_ctx(dev), C.byref(p), *map(C.byref, given), lse.data_ptr(), *map(C.byref, made),
                                              out is None, _p(ws), nbytes, _raw_stream(dev.index)),
           "fvsr_packed_attention_backward")
    return outs
