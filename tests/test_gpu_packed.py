"""The packed operators against float64 plain forms (tests/packed_reference.py, which derives attention's tolerances).

Others, per value, with U = 2^-24 and h half a step of the output's type:
  rms norm: a sum over a row adds at most 32 squares in a lane, then over 64 lanes and 16 waves: below 64 U of itself, rstd below 40 U
      with its root and quotient; y below (h + 48 U) |y|; the sum is one addition in 32 bits (exact for bfloat16 but where exponents
      are more than 16 apart) and one rounding: equal to torch's
  its gradient: n is off by 2 U |n|, mean(g n) by 70 U of the mean of magnitudes: dx below 80 U rstd (|g| + |n| mean|g n|) + h |dx|
      + U |dsum|; dweight: at most rows / 512 + 8 values in a lane, 16 teams, 32 blocks' parts in a thread, 16 threads: below
      (rows / 512 + 80) U of the sum of magnitudes
  rotary: an angle's fraction of a turn is exact to 2^-25 turns (rounded to 32 bits below half a turn): 2^-22.3 radians; sine and
      cosine 4 U more; products and sums 3 U: below (|a| + |b|) 2^-21 + h |result|
"""
import ctypes
import math
import threading

import pytest
import torch

import fvsr_lcsa as f
from fvsr_lcsa import _abi
from packed_reference import H, U, attention64, rms64, rms_grad64, turn64, within
from train8_reference import RUN, quantize64

pytestmark = pytest.mark.gpu
bf, f32 = torch.bfloat16, torch.float32


def gen_of(*seed):
    return torch.Generator().manual_seed(hash(seed) % (1 << 31))


def randn(gen, shape, dev, dtype=bf, scale=1.0):
    return (torch.randn(shape, generator=gen) * scale).to(dtype).to(dev)


def cu_of(lengths, dev, start=0):
    at = [start]
    for n in lengths:
        at.append(at[-1] + n)
    return at, torch.tensor(at, dtype=torch.int32, device=dev)


# ---- rms norm ------------------------------------------------------------------------------------------------------------
def stream_of(gen, rows, c, dtype, dev):
    x = torch.randn((rows, c), generator=gen) * torch.exp(torch.randn(c, generator=gen))
    if c > 3:
        x[:, 3] *= 30
    if rows > 2:
        x[1] = 0
    return x.to(dtype).to(dev)


@pytest.mark.parametrize("dtype", [bf, f32])
@pytest.mark.parametrize("rows,c", [(1, 1), (3, 7), (5, 8), (65, 64), (17, 128), (4, 129), (33, 520), (9, 1003), (130, 1536), (3, 2047),
                                    (5, 4096), (2, 6000), (3, 8192), (2, 8961), (2, 16384), (3, 1026), (4, 1004), (3, 10), (4, 13), (3, 4102),
                                    (7, 9214), (600, 9), (1100, 8195)])
def test_rms_norm_and_gradient(dev, dtype, rows, c):
    g = gen_of(rows, c)
    x, r, dy, ds = (stream_of(g, rows, c, dtype, dev) for _ in range(4))
    for res in (None, r):
        for w in (None, torch.randn(c, generator=g).to(dev), torch.randn(c, generator=g).to(bf).to(dev)):
            y, total, rstd = f.rms_norm(x, w, 1e-6, residual=res, want_stats=True)
            t64, y64, r64 = rms64(x.cpu(), None if res is None else res.cpu(), None if w is None else w.cpu(), 1e-6)
            assert y.dtype == dtype and (total is None) == (res is None)
            if res is not None:
                assert torch.equal(total.cpu().double(), t64)
            within(rstd, r64, 40 * U * r64, "rstd")
            within(y, y64, (H[dtype] + 48 * U) * y64.abs() + 1e-44, "y")
            kept = x if res is None else total
            for more in (None, ds):
                dx, dw = f.rms_norm_backward(dy, kept, rstd, w, dsum=more)
                want, w64, size, wsize = rms_grad64(dy.cpu(), t64, rstd.cpu(), None if w is None else w.cpu(), None if more is None else more.cpu())
                tol = 80 * U * size + H[dtype] * want.abs() + (0 if more is None else U * more.cpu().double().abs()) + 1e-44
                within(dx, want, tol * (1 + H[dtype]), "dx")
                within(dw, w64, (rows / 512 + 80) * U * wsize, "dweight")
                again = f.rms_norm_backward(dy, kept, rstd, w, dsum=more)
                assert torch.equal(again[0], dx) and torch.equal(again[1], dw)
                assert f.rms_norm_backward(dy, kept, rstd, w, dsum=more, want_weight=False)[1] is None


@pytest.mark.parametrize("rows,c", [(1, 8), (40, 64), (5, 129), (33, 1536), (7, 2500)])
def test_rms_norm_in_8_bits(dev, rows, c):
    g = gen_of(rows, c, 8)
    x, r = (stream_of(g, rows, c, bf, dev) for _ in range(2))
    w = torch.randn(c, generator=g).to(dev)
    q, total, _ = f.rms_norm(x, w, residual=r, quantized=True)
    _, y64, _ = rms64(x.cpu(), r.cpu(), w.cpu(), 1e-6)
    held, e = quantize64(y64)
    # a value next to a border may fall to the neighbouring code: a step of e4m3 is 2^-3 of a value, 2^-9 of the scale below its normals
    step = torch.maximum(held.abs() / 8, torch.ldexp(torch.ones(1, dtype=torch.float64), e.repeat_interleave(RUN, 1)[:, :c] - 9))
    got = f.dequantize8(q, f32).cpu().double()
    assert ((got - held).abs() <= 2 * step).all()
    assert ((got != held).double().mean()) <= 1e-3 + 2 / got.numel()   # borders met: 48 U of 2^-4 a value, a run's scale, both rare
    assert not q.codes.view(torch.uint8)[:, c:].any() and not q.scales.view(torch.uint8)[:, e.shape[1]:].any()
    assert torch.equal(total.double(), (x.double() + r.double()).to(bf).double())


def test_rms_norm_of_wide_rows_in_place_and_empty(dev):
    g = gen_of("wide")
    qkv = randn(g, (50, 3 * 1536 + 5), dev)
    part = qkv[:, 1536:1536 + 1540]
    y, _, rstd = f.rms_norm(part, want_stats=True)
    y2, _, rstd2 = f.rms_norm(part.contiguous(), want_stats=True)
    assert torch.equal(y, y2) and torch.equal(rstd, rstd2)
    dy = randn(g, (50, 1540), dev)
    a, b = f.rms_norm_backward(dy, part, rstd), f.rms_norm_backward(dy, part.contiguous(), rstd)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    x, r = randn(g, (9, 300), dev), randn(g, (9, 300), dev)
    want, total, _ = f.rms_norm(x, residual=r)
    x1, r1 = x.clone(), r.clone()
    got = f.rms_norm(x1, residual=r1, out=x1, out_sum=r1)
    assert got[0] is x1 and got[1] is r1 and torch.equal(x1, want) and torch.equal(r1, total)
    d1 = dy.clone()
    assert torch.equal(f.rms_norm_backward(d1, part, rstd, out=d1)[0], a[0])
    e = torch.empty((0, 256), dtype=bf, device=dev)
    y, t, s = f.rms_norm(e, residual=e, want_stats=True)
    dx, dw = f.rms_norm_backward(e, t, s)
    assert y.shape == (0, 256) and dx.shape == (0, 256) and torch.equal(dw, torch.zeros(256, device=dev))
    assert f.rms_norm(x[None])[0].shape == (1, 9, 300)


def test_rms_norm_of_rows_that_are_not_finite(dev):
    x = randn(gen_of("inf"), (6, 200), dev)
    x[1, 7], x[2, 199], x[3] = math.inf, math.nan, 0
    y, _, rstd = f.rms_norm(x, eps=0.0, want_stats=True)
    assert torch.isfinite(y[[0, 4, 5]]).all() and y[2].isnan().all()
    assert y[1, 7].isnan() and not y[1, :7].any() and y[3].isnan().all()
    q = f.rms_norm(x, eps=0.0, quantized=True)[0]
    assert not q.codes.view(torch.uint8)[:, 200:].any()
    dx, _ = f.rms_norm_backward(x, x, rstd)
    assert torch.isfinite(dx[[0, 4, 5]]).all()


# ---- rotary --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [bf, f32])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("n,h,hk,d,axes,far", [(1, 12, 2, 128, (22, 21, 21), 1024), (5, 3, 1, 16, (8,), 10), (33, 4, 4, 64, (16, 16), 500),
                                               (7, 2, 0, 80, (16, 17), 10 ** 6), (100, 9, 3, 104, (25, 27), 2 ** 31 - 1),
                                               (3, 5, 1, 6, (1,), 3), (19, 20, 4, 30, (0, 11, 2), 77), (2100, 2, 1, 256, (40, 40, 40), 9000), (3, 1, 1, 1024, (512,), 50),
                                               (2, 2, 1, 1022, (3, 200, 307), 2 ** 20), (9, 2, 1, 12, (6,), 50), (9, 3, 1, 20, (3, 4), 50),
                                               (5, 4, 2, 44, (9, 10), 1000), (6, 9, 9, 72, (33,), 100), (40, 3, 2, 18, (2, 3, 4), 9), (300, 5, 5, 72, (17, 15), 60)])
def test_rotary_and_gradient(dev, dtype, halves, n, h, hk, d, axes, far):
    g = gen_of(n, h, d, halves)
    qkv = randn(g, (n, h + 2 * hk + 1, d), dev, dtype)
    q, k = qkv[:, :h], qkv[:, h:h + hk] if hk else None
    pos = torch.randint(0, far, (len(axes), n), generator=g)
    freq = torch.cat([10000.0 ** (-torch.arange(p, dtype=torch.float64) / max(p, 1)) for p in axes])
    for dt in (torch.int32, torch.int64):
        how = (pos.to(dt).to(dev), freq.to(dev), axes, halves)
        for fn, back in ((f.rotary, False), (f.rotary_backward, True)):
            got = fn(q, k, *how)
            for x, y in zip((q, k), got):
                if x is None:
                    assert y is None
                    continue
                want = turn64(x.cpu(), pos, freq, axes, halves, back)
                size = torch.zeros_like(want)
                m = sum(axes)
                first = torch.arange(m) if halves else 2 * torch.arange(m)
                second = first + (m if halves else 1)
                xx = x.cpu().double().abs()
                size[..., first] = size[..., second] = xx[..., first] + xx[..., second]
                assert y.is_contiguous() and y.dtype == dtype
                within(y, want, size * 2.0 ** -21 + H[dtype] * want.abs(), "turned")
                assert torch.equal(y[..., 2 * m:], x[..., 2 * m:])
    keep = qkv.clone()
    got = f.rotary(q, k, *how)
    assert torch.equal(qkv, keep)
    same = f.rotary(q, k, *how, out=(q, k))
    assert same[0] is q and torch.equal(q, got[0]) and (k is None or torch.equal(k, got[1]))
    assert torch.equal(qkv[:, h + hk:], keep[:, h + hk:])


@pytest.mark.parametrize("dtype", [bf, f32])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("d,pairs", [(16, 5), (80, 33), (24, 8), (72, 33)])
def test_rotary_of_channels_that_are_not_finite(dev, dtype, halves, d, pairs):
    """Channels past the pairs are copied whatever they hold, and a pair's values stay in the pair."""
    g = gen_of("not finite", d, pairs, halves)
    n, m = 7, 2 * pairs
    q, pos = randn(g, (n, 3, d), dev, dtype), torch.randint(0, 50, (n,), generator=g, dtype=torch.int32).to(dev)
    freq = f.rotary_frequencies((pairs,), device=dev)
    want = f.rotary(q, None, pos, freq, (pairs,), halves)[0]
    q[:, 1, m:] = math.inf
    q[:, 1, m::2] = math.nan
    got = f.rotary(q, None, pos, freq, (pairs,), halves)[0]
    assert torch.equal(got[..., :m], want[..., :m])
    assert torch.equal(got[..., m:].view(torch.int16 if dtype == bf else torch.int32), q[..., m:].view(torch.int16 if dtype == bf else torch.int32))
    same = q.clone()
    f.rotary(same, None, pos, freq, (pairs,), halves, out=(same, None))
    assert torch.equal(same[..., :m], want[..., :m])
    i = pairs - 1
    a, b = (i, i + pairs) if halves else (2 * i, 2 * i + 1)
    q[:, 1, a] = math.nan
    got = f.rotary(q, None, pos, freq, (pairs,), halves)[0]
    rest = [c for c in range(m) if c not in (a, b)]
    assert got[:, 1, [a, b]].isnan().all() and torch.equal(got[:, 1, rest], want[:, 1, rest])


def test_rotary_is_the_fused_epilogues(dev):
    """The positions and axes of the DiT: rotary of normed q against the fused epilogue's, which keeps its tables in float32."""
    fr, hh, ww, heads = 2, 8, 8, 2
    g = gen_of("fused")
    q, k, v = (randn(g, (fr * hh * ww, heads * 128), dev) for _ in range(3))
    wq = torch.ones(heads * 128, dtype=bf, device=dev)
    eq, ek, _ = f.qkv_epilogue(q, k, v, fr, hh, ww, heads, 3, wq, wq)
    pos, freq = f.grid_positions(fr, hh, ww, 3, dev), f.rotary_frequencies((22, 21, 21), device=dev)
    nq, nk = (f.rms_norm(x, wq)[0].view(-1, heads, 128) for x in (q, k))
    rq, rk = f.rotary(nq, nk, pos, freq, (22, 21, 21))
    for a, b in ((eq, rq), (ek, rk)):
        b = f.window_partition(b.reshape(-1, heads * 128), fr, hh, ww)
        # both round the norm and the result to bfloat16; the norms may differ by a step (2^-7), in either channel of a pair
        assert ((a.double() - b.double()).abs() <= 2.0 ** -6 * 1.5 * (1 + b.double().abs().amax(1, keepdim=True) / 4)).all()
        assert (a != b).double().mean() < 0.05


def test_rotary_of_no_tokens(dev):
    e = torch.empty((0, 4, 64), dtype=bf, device=dev)
    freq = f.rotary_frequencies((32,), device=dev)
    a, b = f.rotary(e, e[:, :1], torch.empty(0, dtype=torch.int32, device=dev), freq, (32,))
    assert a.shape == (0, 4, 64) and b.shape == (0, 1, 64)


# ---- attention -----------------------------------------------------------------------------------------------------------
def check_attention(dev, lengths_q, lengths_k, h, hk, d, causal, used=None, train=True, scale=None, start=0, tail=0, strided=False, seed=0):
    g = gen_of(tuple(lengths_q), h, hk, d, causal, seed)
    cq, cu_q = cu_of(lengths_q, dev, start)
    lq = cq[-1] + tail
    if lengths_k is None:
        ck, cu_k, lk = None, None, lq
    else:
        ck, cu_k = cu_of(lengths_k, dev, start)
        lk = ck[-1] + tail
    wide = 8 if strided else 0
    q = randn(g, (lq, h + wide, d), dev, scale=1.5)[:, :h]
    k, v = (randn(g, (lk, hk + wide, d), dev)[:, :hk] for _ in range(2))
    do = randn(g, (lq, h, d), dev)
    us = None if used is None else torch.tensor(used, dtype=torch.int32, device=dev)
    how = dict(causal=causal, scale=scale)
    ref = attention64(q, k, v, cq, ck, used=used, do=do if train else None, **how)
    o, lse = f.packed_attention(q, k, v, cu_q, cu_k, used_k=us, want_lse=True, **how)
    within(o, ref["o"], ref["tol_o"], "o")
    within(lse, ref["lse"], ref["tol_lse"], "lse")
    o2, none = f.packed_attention(q, k, v, cu_q, cu_k, used_k=us, **how)
    assert none is None and torch.equal(o, o2)
    mark = torch.full_like(o, 7.0)
    f.packed_attention(q, k, v, cu_q, cu_k, used_k=us, out=mark, **how)
    inside = torch.zeros(lq, dtype=torch.bool)
    inside[cq[0]:cq[-1]] = True
    assert torch.equal(mark[inside.to(dev)], o[inside.to(dev)]) and (mark[~inside.to(dev)] == 7).all()
    if not train:
        return
    grads = f.packed_attention_backward(do, q, k, v, o, lse, cu_q, cu_k, used_k=us, **how)
    for n, x in zip(("dq", "dk", "dv"), grads):
        within(x, ref[n], ref["tol_" + n], n)
    again = f.packed_attention_backward(do, q, k, v, o, lse, cu_q, cu_k, used_k=us, **how)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    marks = [torch.full((x.shape[0], x.shape[1] + 8, d), 7.0, dtype=bf, device=dev)[:, :x.shape[1]] for x in grads]
    f.packed_attention_backward(do, q, k, v, o, lse, cu_q, cu_k, used_k=us, out=marks, **how)
    for m, x, c in zip(marks, grads, (cq, ck or cq, ck or cq)):
        rows = torch.zeros(x.shape[0], dtype=torch.bool, device=dev)
        rows[c[0]:c[-1]] = True
        assert torch.equal(m[rows], x[rows]) and (m[~rows] == 7).all()


def workspace(lengths_q, lengths_k, h, hk, d, causal):
    """Bytes of workspace of a forward call, where the keys are split over the workgroups."""
    packed = _abi.Packed(0, 0, None, len(lengths_q), sum(lengths_q), sum(lengths_k), d, int(causal), 1.0)
    return _abi.lib.fvsr_packed_attention_workspace(ctypes.byref(packed), h, hk)


LENGTHS = [[1], [2, 1, 3], [31, 32, 33], [128], [129, 0, 127, 1], [300, 64], [5, 257, 0, 0, 40, 128, 31]]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("h,hk,d", [(1, 1, 64), (4, 2, 128), (3, 1, 40), (2, 2, 80), (4, 1, 8)])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_packed_attention_and_gradient(dev, lengths, h, hk, d, causal):
    check_attention(dev, lengths, None, h, hk, d, causal)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,lk", [([1], [1]), ([1], [700]), ([3, 1], [2, 1]), ([200, 5], [90, 400]), ([64, 0, 30], [0, 50, 31]),
                                   ([260], [131]), ([131], [300]), ([1] * 70, list(range(70)))], ids=str)
def test_packed_attention_of_other_keys(dev, lq, lk, causal):
    check_attention(dev, lq, lk, 4, 2, 64, causal, strided=True)
    check_attention(dev, lq, lk, 2, 2, 128, causal, used=[max(0, n - 7) for n in lk])


@pytest.mark.parametrize("causal", [False, True])
def test_packed_attention_rows_of_no_sequence(dev, causal):
    for lengths in ([40, 100], [1, 1, 1], [0, 130], [300]):
        check_attention(dev, lengths, None, 2, 1, 64, causal, start=150, tail=200)
        check_attention(dev, lengths, None, 4, 2, 128, causal, start=5, tail=1)


@pytest.mark.parametrize("n", [62, 63, 64, 65, 130])
def test_packed_attention_of_many_sequences(dev, n):
    """Around the number that a wave's lanes hold, and past it."""
    check_attention(dev, [40 + i % 3 for i in range(n)], None, 4, 1, 64, True)
    check_attention(dev, [i % 4 for i in range(n)], [i % 7 for i in range(n)], 2, 2, 128, False)


def test_packed_attention_scales(dev):
    check_attention(dev, [70, 33], None, 2, 1, 64, True, scale=1.0)      # sharp weights
    check_attention(dev, [70, 33], None, 2, 1, 64, False, scale=1e-4)
    check_attention(dev, [1, 1], [900, 40], 2, 1, 128, True, scale=2.0, train=False)


@pytest.mark.parametrize("h,hk,d", [(12, 2, 128), (1, 1, 64), (16, 16, 24), (40, 1, 128)])
@pytest.mark.parametrize("m", [1, 2, 5])
def test_single_tokens_over_a_cache(dev, h, hk, d, m):
    g = gen_of(h, hk, d, m)
    room = 2500
    lengths = [2500, 0, 1, 31, 32, 33, 700, 2047, 3, 1200]
    n = len(lengths)
    q = randn(g, (n * m, h, d), dev, scale=1.5)
    k, v = (randn(g, (n * room, hk, d), dev) for _ in range(2))
    cq, ck = [m * i for i in range(n + 1)], [room * i for i in range(n + 1)]
    args = [torch.tensor(x, dtype=torch.int32, device=dev) for x in (cq, ck, lengths)]
    # what a cache holds past its used part is whatever it was
    for i, u in enumerate(lengths):
        k[i * room + u:(i + 1) * room] = math.nan
        v[i * room + u:(i + 1) * room] = math.inf
    ref = attention64(q, k, v, cq, ck, True, used=lengths)
    o, lse = f.packed_attention(q, k, v, args[0], args[1], causal=True, used_k=args[2], want_lse=True)
    within(o, ref["o"], ref["tol_o"], "o")
    within(lse, ref["lse"], ref["tol_lse"], "lse")


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("h,hk,d", [(4, 2, 128), (3, 1, 64), (16, 1, 40)])
@pytest.mark.parametrize("lq,lk", [([2], [700]), ([131], [5000]), ([200, 5], [90, 9000]), ([3, 1, 40], [2, 1, 9000]),
                                   ([64, 0, 30], [0, 9000, 31]), ([33, 32, 1], [3000, 4001, 2990])], ids=str)
def test_few_queries_over_long_keys(dev, lq, lk, h, hk, d, causal):
    """Calls whose keys are split over the workgroups: sizes that have a workspace."""
    assert workspace(lq, lk, h, hk, d, causal)
    check_attention(dev, lq, lk, h, hk, d, causal, train=h == 4, strided=True)
    check_attention(dev, lq, lk, h, hk, d, causal, train=False, start=150, tail=200, used=[max(0, n - 40) for n in lk])


@pytest.mark.parametrize("n", [62, 63, 64, 65, 130])
def test_few_queries_of_many_sequences(dev, n):
    lq, lk = [i % 3 for i in range(n)], [(i * 379) % 1500 for i in range(n)]
    for more in (0, 1500):      # either way, and split
        lk = [k + more for k in lk]
        assert workspace(lq, lk, 4, 1, 64, True) or not more
        check_attention(dev, lq, lk, 4, 1, 64, True, train=False)
        check_attention(dev, lq, lk, 2, 2, 128, False, train=False, used=[k // 2 for k in lk])


def test_hundreds_of_sequences(dev):
    """More than a workgroup has threads: blocks that look for their sequence, and the split walk that counts its tiles."""
    check_attention(dev, [i % 4 for i in range(700)], None, 2, 1, 64, True)
    check_attention(dev, [(i * 7) % 40 for i in range(300)], [(i * 11) % 50 for i in range(300)], 2, 2, 128, True, start=3, tail=5)
    lq, lk = [i % 2 for i in range(700)], [(i * 379) % 1500 + 100 for i in range(700)]
    assert workspace(lq, lk, 2, 1, 64, True)
    check_attention(dev, lq, lk, 2, 1, 64, True, train=False)


def test_few_queries_and_keys_that_are_not_finite(dev):
    """Where the keys are split: an infinity or NaN in the keys and values of one token, of a sequence before or past the used keys."""
    g = gen_of("split nan")
    lq, room, used, h, hk, d = [2, 40, 3], [1000, 5000, 800], [1000, 4900, 790], 4, 2, 64
    assert workspace(lq, room, h, hk, d, True)
    (cq, cu_q), (ck, cu_k) = cu_of(lq, dev), cu_of(room, dev)
    us = torch.tensor(used, dtype=torch.int32, device=dev)
    q = randn(g, (cq[-1], h, d), dev)
    k, v = (randn(g, (ck[-1], hk, d), dev) for _ in range(2))
    ref = attention64(q, k, v, cq, ck, True, used=used)
    for i, n in enumerate(used):
        k[ck[i] + n:ck[i + 1]] = math.nan
        v[ck[i] + n:ck[i + 1]] = math.inf
    for value in (math.inf, math.nan):
        for x in (k, v):
            keep = x.clone()
            x[ck[1] + used[1] - 20] = value      # queries 20 .. 39 of the second sequence see it
            o, lse = f.packed_attention(q, k, v, cu_q, cu_k, causal=True, used_k=us, want_lse=True)
            blind = [i for i in range(cq[-1]) if not cq[1] + 20 <= i < cq[2]]
            within(o[blind], ref["o"][blind], ref["tol_o"][blind], "o")
            within(lse[:, blind], ref["lse"][:, blind], ref["tol_lse"][:, blind], "lse")
            if x is v or value != math.inf:      # a key's infinity may leave a weight of zero
                assert not torch.isfinite(o[cq[1] + 20:cq[2]]).flatten(1).all(1).any()
            x.copy_(keep)


def test_long_sequences(dev):
    check_attention(dev, [2100], None, 2, 1, 128, True)
    check_attention(dev, [1500, 900], None, 2, 1, 64, False)
    check_attention(dev, [1], [20000], 6, 1, 128, True, train=False)


@pytest.mark.parametrize("d,lq,lk,used", [(64, [2100], [3400], None), (128, [2100], [3400], None), (64, [2100, 2049], [1700, 1601], [1690, 1555]),
                                          (40, [2100], [3330], [3300])])
def test_blocks_of_keys_left_for_a_last_round(dev, d, lq, lk, used):
    """dK and dV where the queries of the last blocks of keys are cut into parts, and no others'."""
    h, sel = 40, [0, 17, 39]
    bytes_of = lambda h, causal: _abi.lib.fvsr_packed_attention_backward_workspace(
        ctypes.byref(_abi.Packed(0, 0, None, len(lq), sum(lq), sum(lk), d, causal, 1.0)), h, h)
    parts = bytes_of(h, 0) - bytes_of(h, 1)
    assert 0 < parts < 2 * 4 * sum(lk) * h * d
    g = gen_of("last round", d, len(lq))
    (cq, cu_q), (ck, cu_k) = cu_of(lq, dev), cu_of(lk, dev)
    us = None if used is None else torch.tensor(used, dtype=torch.int32, device=dev)
    q, do = (randn(g, (cq[-1], h, d), dev) for _ in range(2))
    k, v = (randn(g, (ck[-1], h, d), dev) for _ in range(2))
    o, lse = f.packed_attention(q, k, v, cu_q, cu_k, used_k=us, want_lse=True)
    got = f.packed_attention_backward(do, q, k, v, o, lse, cu_q, cu_k, used_k=us)
    ref = attention64(*(x[:, sel] for x in (q, k, v)), cq, ck, used=used, do=do[:, sel])
    for n, x in zip(("dq", "dk", "dv"), got):
        within(x[:, sel], ref[n], ref["tol_" + n], n)
    again = f.packed_attention_backward(do, q, k, v, o, lse, cu_q, cu_k, used_k=us)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    # a few heads by themselves: cut otherwise, or not at all, and off by what the bounds allow each
    few = f.packed_attention_backward(*(x[:, sel] for x in (do, q, k, v, o)), lse[sel], cu_q, cu_k, used_k=us)
    for n, x in zip(("dq", "dk", "dv"), few):
        within(x, ref[n], ref["tol_" + n], n)


def test_offsets_past_32_bits(dev):
    """A cache whose rows lie more than 2^32 bytes from its first: the last of its sequences."""
    n, stride = 600, 1 << 22
    big = torch.empty(n * stride + 128, dtype=bf, device=dev)     # 5 GB
    k = big.as_strided((n, 1, 128), (stride, 128, 1))
    g = gen_of("far")
    k.copy_(randn(g, (n, 1, 128), dev))
    q = randn(g, (130, 2, 128), dev)
    _, cu_q = cu_of([130], dev)
    _, cu_k = cu_of([n], dev)
    ref = attention64(q, k, k, [0, 130], [0, n], True)
    within(f.packed_attention(q, k, k, cu_q, cu_k, causal=True)[0], ref["o"], ref["tol_o"])
    _, c1 = cu_of([1], dev)
    ref = attention64(q[:1], k, k, [0, 1], [0, n], True)
    within(f.packed_attention(q[:1], k, k, c1, cu_k, causal=True)[0], ref["o"], ref["tol_o"])


@pytest.mark.parametrize("m", [2, 200])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_what_a_query_does_not_see_does_not_reach_it(dev, m, value):
    """An infinity or NaN in K, V, q or dO of one token reaches what sees it, and nothing else."""
    g = gen_of("nan", m)
    h, hk, d, at = 4, 2, 64, m // 2 + m // 5
    q, do = (randn(g, (m, h, d), dev) for _ in range(2))
    k, v = (randn(g, (m, hk, d), dev) for _ in range(2))
    cq, cu = cu_of([m], dev)
    ref = attention64(q, k, v, cq, causal=True, do=do)
    before, after = slice(0, at), slice(at + 1, m)
    for name, x in (("k", k), ("v", v), ("q", q), ("do", do)):
        a = {"q": q, "k": k, "v": v, "do": do}
        a[name] = x.clone()
        a[name][at] = value
        o, lse = f.packed_attention(a["q"], a["k"], a["v"], cu, causal=True, want_lse=True)
        within(o[before], ref["o"][before], ref["tol_o"][before], name)
        if name in ("q", "do"):
            within(o[after], ref["o"][after], ref["tol_o"][after], name)
        assert not torch.isfinite(o[at]).all() or name == "do"
        dq, dk, dv = f.packed_attention_backward(a["do"], a["q"], a["k"], a["v"], o, lse, cu, causal=True)
        within(dq[before], ref["dq"][before], ref["tol_dq"][before], name)
        if name in ("q", "do"):      # one row's: reaches the keys it sees
            within(dq[after], ref["dq"][after], ref["tol_dq"][after], name)
            within(dk[after], ref["dk"][after], ref["tol_dk"][after], name)
            within(dv[after], ref["dv"][after], ref["tol_dv"][after], name)
            assert not torch.isfinite(dk[:at + 1]).all() or not torch.isfinite(dv[:at + 1]).all()


def test_offsets_that_leave_the_tensors_or_fall_write_nothing_outside(dev):
    """Bad offsets are taken into the tensors' range: what comes out is of no use, but the guard rows around stay."""
    g = gen_of("bad")
    whole = torch.full((400, 2, 64), 7.0, dtype=bf, device=dev)
    q = randn(g, (200, 2, 64), dev)
    for cu in ([0, 500], [-50, 100, 99999], [0, 150, 20, 200], [2 ** 31 - 1, -2 ** 31]):
        c = torch.tensor(cu, dtype=torch.int32, device=dev)
        o, lse = f.packed_attention(q, q, q, c, causal=True, want_lse=True, out=whole[100:300])
        f.packed_attention_backward(q, q, q, q, o, lse, c, causal=True)
        torch.cuda.synchronize()
        assert (whole[:100] == 7).all() and (whole[300:] == 7).all()


def test_unaligned_and_overlapping_views_are_read(dev):
    g = gen_of("view")
    flat = randn(g, (60 * 2 * 64 + 4,), dev)
    q = flat[4:].view(60, 2, 64)                       # 8-byte aligned
    k = randn(g, (60, 1, 64), dev).expand(60, 2, 64)   # one head read as two
    cq, cu = cu_of([60], dev)
    ref = attention64(q, k, k, cq, causal=True)
    within(f.packed_attention(q, k, k, cu, causal=True)[0], ref["o"], ref["tol_o"])
    assert f.packed_attention(q[None], k[None], k[None], cu)[0].shape == (1, 60, 2, 64)
    # heads that lie one behind another, a lone token far from the next, no stride at all
    q, k = randn(g, (4, 60, 64), dev).transpose(0, 1), randn(g, (2, 60, 64), dev).transpose(0, 1)
    ref = attention64(q, k, k, cq, causal=True, do=q)
    o, lse = f.packed_attention(q, k, k, cu, causal=True, want_lse=True)
    within(o, ref["o"], ref["tol_o"])
    for name, x in zip(("dq", "dk", "dv"), f.packed_attention_backward(q, q, k, k, o, lse, cu, causal=True)):
        within(x, ref[name], ref["tol_" + name], name)
    far = torch.empty((2, 1 << 24), dtype=bf, device=dev)
    lone = far.as_strided((1, 4, 64), (1 << 24, 64, 1))
    lone.copy_(randn(g, (1, 4, 64), dev))
    _, c1 = cu_of([1], dev)
    assert torch.equal(f.packed_attention(lone, lone, lone, c1)[0], lone)
    freq, pos = f.rotary_frequencies((32,), device=dev), torch.arange(60, dtype=torch.int32, device=dev)
    a, b = f.rotary(q, k, pos, freq, (32,))
    c, d = f.rotary(q.contiguous(), k.contiguous(), pos, freq, (32,))
    assert torch.equal(a, c) and torch.equal(b, d)
    for n in (1, 40, 45):   # one token read as many: rows past the last are not zeros
        one, do = randn(g, (1, 2, 64), dev).expand(n, 2, 64), randn(g, (1, 2, 64), dev).expand(n, 2, 64)
        cq, cu = cu_of([n], dev)
        for causal in (False, True):
            ref = attention64(one, one, one, cq, causal=causal, do=do)
            o, lse = f.packed_attention(one, one, one, cu, causal=causal, want_lse=True)
            within(o, ref["o"], ref["tol_o"])
            for name, x in zip(("dq", "dk", "dv"), f.packed_attention_backward(do, one, one, one, o, lse, cu, causal=causal)):
                within(x, ref[name], ref["tol_" + name], name)


def test_no_tokens(dev):
    e = torch.empty((0, 4, 64), dtype=bf, device=dev)
    cu = torch.zeros(3, dtype=torch.int32, device=dev)
    o, lse = f.packed_attention(e, e[:, :2], e[:, :2], cu, want_lse=True)
    assert o.shape == e.shape and lse.shape == (4, 0)
    assert all(x.shape[0] == 0 for x in f.packed_attention_backward(e, e, e[:, :2], e[:, :2], o, lse, cu))
    q = torch.ones((3, 4, 64), dtype=bf, device=dev)
    o, lse = f.packed_attention(q, e[:, :2], e[:, :2], torch.tensor([0, 1, 3], dtype=torch.int32, device=dev), cu, want_lse=True)
    assert not o.any() and (lse == -math.inf).all()
    cu_q = torch.tensor([0, 1, 3], dtype=torch.int32, device=dev)
    dq, dk, dv = f.packed_attention_backward(q, q, e[:, :2], e[:, :2], o, lse, cu_q, cu)      # no keys
    assert not dq.any() and dk.shape == dv.shape == (0, 2, 64)
    dq, dk, dv = f.packed_attention_backward(e, e, q[:, :2], q[:, :2], e, lse[:, :0], cu, cu_q)      # no queries
    assert dq.shape == e.shape and not dk.any() and not dv.any()


@pytest.mark.parametrize("nq", [1, 200])
@pytest.mark.parametrize("h", [1, 40])
def test_keys_whose_scores_are_all_minus_infinity(dev, nq, h):
    """An infinity in the first keys that gives them no weight, in tiles that are seen whole: as if they were not there."""
    g = gen_of("minus", nq, h)
    n, blind = 1500, 70
    q, (k, v) = randn(g, (nq, h, 64), dev), (randn(g, (n, 1, 64), dev) for _ in range(2))
    q[..., 5] = q[..., 5].abs() + 0.1
    _, cu_q = cu_of([nq], dev)
    _, cu_k = cu_of([n], dev)
    ref = attention64(q, k[blind:], v[blind:], [0, nq], [0, n - blind])
    k[:blind, :, 5] = -math.inf
    o, lse = f.packed_attention(q, k, v, cu_q, cu_k, want_lse=True)
    within(o, ref["o"], ref["tol_o"], "o")
    within(lse, ref["lse"], ref["tol_lse"], "lse")


# ---- together, as they are used ------------------------------------------------------------------------------------------
class Pass:
    """Norm with the residual, projection, norms of q and k, positions, attention, and all the way back."""

    def __init__(self, dev, lengths, h=4, hk=2, d=64):
        g = gen_of("pass", tuple(lengths))
        n, c = sum(lengths), h * d
        self.h, self.hk, self.d = h, hk, d
        self.x, self.res, self.do, self.dsum = (randn(g, (n, c), dev) for _ in range(4))
        self.w = 1 + 0.1 * torch.randn(c, generator=g).to(dev)
        self.wh = 1 + 0.1 * torch.randn(d, generator=g).to(dev)
        self.proj = randn(g, (c, (h + 2 * hk) * d), dev, scale=c ** -0.5)
        self.axes = (d // 4 - 5, 5, d // 4)
        self.pos = torch.randint(0, 200, (3, n), generator=g, dtype=torch.int32).to(dev)
        self.freq = f.rotary_frequencies(self.axes, device=dev)
        self.lengths, (self.cq, self.cu) = lengths, cu_of(lengths, dev)

    def run(self):
        n, h, hk, d = self.x.shape[0], self.h, self.hk, self.d
        y, total, rstd = f.rms_norm(self.x, self.w, residual=self.res, want_stats=True)
        qkv = (y @ self.proj).view(n, h + 2 * hk, d)
        qk = qkv[:, :h + hk].reshape(-1, d)
        nq, _, rs = f.rms_norm(qk, self.wh, want_stats=True)
        nqk = nq.view(n, h + hk, d)
        q, k = f.rotary(nqk[:, :h], nqk[:, h:], self.pos, self.freq, self.axes)
        v = qkv[:, h + hk:]
        o, lse = f.packed_attention(q, k, v, self.cu, causal=True, want_lse=True)
        back = torch.empty((n, h + 2 * hk, d), dtype=bf, device=self.x.device)
        f.packed_attention_backward(self.do.view(n, h, d), q, k, v, o, lse, self.cu, causal=True,
                                    out=(back[:, :h], back[:, h:h + hk], back[:, h + hk:]))
        f.rotary_backward(back[:, :h], back[:, h:h + hk], self.pos, self.freq, self.axes, out=(back[:, :h], back[:, h:h + hk]))
        dqk, dwh = f.rms_norm_backward(back[:, :h + hk].reshape(-1, d), qk, rs, self.wh)
        back[:, :h + hk] = dqk.view(n, h + hk, d)
        dx, dw = f.rms_norm_backward(back.view(n, -1) @ self.proj.t(), total, rstd, self.w, dsum=self.dsum)
        return o, dx, dw, dwh, total

    def want(self):
        """The same in float64 by autograd, from formulas."""
        n, h, hk, d = self.x.shape[0], self.h, self.hk, self.d
        x = (self.x.double() + self.res.double()).to(bf).double().cpu().requires_grad_()
        w, wh = (t.double().cpu().requires_grad_() for t in (self.w, self.wh))
        norm = lambda t, w: t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w
        qkv = (norm(x, w) @ self.proj.double().cpu()).view(n, h + 2 * hk, d)
        qk = turn64(norm(qkv[:, :h + hk], wh), self.pos.cpu(), self.freq.cpu(), self.axes, False)
        out = []
        for a, m in zip(self.cq, self.lengths):
            r = slice(a, a + m)
            k, v = (t.repeat_interleave(h // hk, 1).transpose(0, 1) for t in (qk[r, h:], qkv[r, h + hk:]))
            s = qk[r, :h].transpose(0, 1) @ k.transpose(1, 2) / math.sqrt(d)
            s = s.masked_fill(torch.ones(m, m, dtype=torch.bool).triu(1), -math.inf)
            out.append((torch.softmax(s, -1) @ v).transpose(0, 1))
        o = torch.cat(out)
        (o * self.do.double().cpu().view(n, h, d)).sum().add((x * self.dsum.double().cpu()).sum()).backward()
        return o.detach(), x.grad, w.grad, wh.grad


def test_a_training_pass(dev):
    p = Pass(dev, [70, 1, 130, 33])
    got, want = p.run(), p.want()
    for name, a, b in zip(("o", "dx", "dw", "dwh"), got, want):
        a = a.double().cpu()
        # the path rounds to bfloat16 nine times (norm, projection, norm, positions, o; dq/dk/dv, back, norm, projection), each off by
        # at most 2^-8 of its size, and P and dS once each: 11 roundings; their size against the result's is at most 4 here in the
        # root mean square (products of random rows do not cancel more)
        assert float((a - b).norm() / b.norm()) <= 11 * 4 * 2.0 ** -8, name


def test_a_training_pass_captured_and_replayed(dev):
    """One graph, its inputs written anew between the replays, with eager passes between them, and a second graph of its own."""
    with torch.no_grad():
        p, other = Pass(dev, [70, 1, 130, 33]), Pass(dev, [64, 200])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            p.run(), other.run()
        torch.cuda.current_stream().wait_stream(side)
        graphs = []
        for x in (p, other):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                held = x.run()
            graphs.append((gr, held))
        for i in range(3):
            p.x.copy_(randn(gen_of("replay", i), p.x.shape, dev))
            if i == 2:   # other lengths in the same total: the graph follows the offsets
                p.cu.copy_(torch.tensor([0, 100, 101, 200, 234], dtype=torch.int32))
            graphs[1][0].replay()
            graphs[0][0].replay()
            torch.cuda.synchronize()
            for x, (_, held) in zip((p, other), graphs):
                assert all(torch.equal(a, b) for a, b in zip(held, x.run())), i


def test_single_tokens_captured_and_on_another_stream(dev):
    g = gen_of("serve")
    room, n = 900, 5
    q = randn(g, (n, 8, 128), dev)
    k, v = (randn(g, (n * room, 2, 128), dev) for _ in range(2))
    cu_q = torch.arange(n + 1, dtype=torch.int32, device=dev)
    used = torch.tensor([1, 400, 0, 899, 33], dtype=torch.int32, device=dev)
    call = lambda **kw: f.packed_attention(q, k, v, cu_q, room * cu_q, causal=True, used_k=used, **kw)[0]
    ck = room * cu_q
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = [f.packed_attention(q, k, v, cu_q, ck, causal=True, used_k=used, stream=side)[0] for _ in range(2)]
    more = call()   # beside them, on this stream
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got) and torch.equal(more, want)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        o, _ = f.packed_attention(q, k, v, cu_q, ck, causal=True, used_k=used)
    for i in range(3):
        used += 1
        gr.replay()
        torch.cuda.synchronize()
        ref = attention64(q, k, v, list(range(n + 1)), [room * j for j in range(n + 1)], True, used=used.tolist())
        within(o, ref["o"], ref["tol_o"], str(i))
        assert torch.equal(o, call())


def test_calls_of_several_threads(dev):
    """Threads with streams of their own, at the same time."""
    g = gen_of("threads")
    q, do = (randn(g, (300, 4, 64), dev) for _ in range(2))
    k, v = (randn(g, (300, 2, 64), dev) for _ in range(2))
    x, w = randn(g, (300, 256), dev), torch.ones(256, device=dev)
    cu = [torch.tensor(c, dtype=torch.int32, device=dev) for c in ([0, 300], [0, 1, 200, 300])]
    freq, pos = f.rotary_frequencies((32,), device=dev), torch.arange(300, dtype=torch.int32, device=dev)

    def once(i):
        a, b = f.rotary(q, k, pos + i, freq, (32,))
        o, lse = f.packed_attention(a, b, v, cu[i % 2], causal=True, want_lse=True)
        grads = f.packed_attention_backward(do, a, b, v, o, lse, cu[i % 2], causal=True)
        y, _, rstd = f.rms_norm(x, w, residual=x, want_stats=True)
        return (a, b, o, lse, *grads, y, *f.rms_norm_backward(y, x, rstd, w))

    want, wrong = [once(i) for i in range(4)], []
    torch.cuda.synchronize()

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = once(i)
                torch.cuda.current_stream().synchronize()
                wrong.extend(i for a, b in zip(got, want[i]) if not torch.equal(a, b))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_whatever_a_workspace_holds(dev):
    """Temporaries from memory full of NaN: nothing is read before it is written."""
    g = gen_of("workspace")
    (_, c1), (_, ck), (_, c2) = cu_of([1, 2, 40], dev), cu_of([3000, 1, 4000], dev), cu_of([2000, 500, 60], dev)
    q, k = randn(g, (43, 4, 128), dev), randn(g, (7001, 2, 128), dev)
    x, y = randn(g, (2560, 4, 64), dev), randn(g, (2560, 1, 64), dev)
    r, w = randn(g, (700, 640), dev), torch.ones(640, device=dev)

    def run():
        o, lse = f.packed_attention(x, y, y, c2, causal=True, want_lse=True)
        n, _, rstd = f.rms_norm(r, w, want_stats=True)
        return (*f.packed_attention(q, k, k, c1, ck, causal=True, want_lse=True), o, *f.packed_attention_backward(x, x, y, y, o, lse, c2, causal=True),
                *f.rms_norm_backward(n, r, rstd, w))

    want = run()
    torch.cuda.synchronize()
    for size in (1 << 18, 1 << 22, 1 << 25, 1 << 27):
        held = [torch.full((size // 4,), math.nan, device=dev) for _ in range(4)]
        del held
        assert all(torch.equal(a, b) for a, b in zip(run(), want))


def test_norm_to_8_bits_into_a_linear_layer(dev):
    g = gen_of("serve8")
    x, r = (randn(g, (130, 512), dev) for _ in range(2))
    w8 = f.quantize8(randn(g, (256, 512), dev, scale=512 ** -0.5))
    w = 1 + 0.1 * torch.randn(512, generator=g).to(dev)
    a, total, _ = f.rms_norm(x, w, residual=r, quantized=True)
    y = f.linear8(a, w8)
    want = f.dequantize8(a, f32).double() @ f.dequantize8(w8, f32).double().t()
    size = f.dequantize8(a, f32).double().abs() @ f.dequantize8(w8, f32).double().abs().t()
    within(y, want, 2.0 ** -8 * want.abs() + size * 2.0 ** -7)
