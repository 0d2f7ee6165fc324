"""Calls of the packed operators at the edges of what their documentation allows: the packed pass' rings at their shortest, views that
overlap, rows of no sequence, very large scores and values, offsets that fall. Against the float64 forms of tests/packed_reference.py."""
import ctypes
import math
import zlib

import pytest
import torch

import fvsr_lcsa as f
from packed_reference import attention64, within

pytestmark = pytest.mark.gpu
bf = torch.bfloat16


def gen_of(*seed):
    return torch.Generator().manual_seed(zlib.crc32(repr(seed).encode()))


def randn(gen, shape, dev, dtype=bf, scale=1.0):
    return (torch.randn(shape, generator=gen) * scale).to(dtype).to(dev)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("keys", [128, 130, 160, 256])
def test_the_first_tile_is_read_before_its_place_is_filled_again(dev, d, keys):
    """Whole attention over four tiles of keys and a few more: the walk's first step requests the fifth tile, or zeros, into the first
    one's place. Many blocks, many times: the same bits, and the formula's values."""
    g = gen_of("ring", d, keys)
    m, h = 1152, 48
    q, k, v = (randn(g, (n, h, d), dev, scale=s) for n, s in ((m, 1.5), (keys, 1.0), (keys, 1.0)))
    cu_q, cu_k = (torch.tensor([0, n], dtype=torch.int32, device=dev) for n in (m, keys))
    o, lse = f.packed_attention(q, k, v, cu_q, cu_k, want_lse=True)
    for _ in range(20):
        again = f.packed_attention(q, k, v, cu_q, cu_k, want_lse=True)
        assert torch.equal(again[0], o) and torch.equal(again[1], lse)
    sel = [0, 23, 47]
    ref = attention64(q[:, sel], k[:, sel], v[:, sel], [0, m], [0, keys])
    within(o[:, sel], ref["o"], ref["tol_o"], "o")
    within(lse[sel], ref["lse"], ref["tol_lse"], "lse")


@pytest.mark.parametrize("dtype", [bf, torch.float32])
@pytest.mark.parametrize("shape,strides", [((4, 2, 8), (16, 1, 1)), ((4, 2, 8), (1, 16, 1)), ((9, 3, 8), (2, 1, 1)), ((1, 4, 8), (1, 1, 1)),
                                           ((40, 1, 64), (1, 1, 1)), ((5, 4, 64), (0, 1, 1))])
def test_windows_that_overlap_are_read(dev, dtype, shape, strides):
    """Heads, or tokens, one element apart: results have their own layout, with the channels innermost."""
    g = gen_of("windows", shape, strides)
    n, h, d = shape
    x = randn(g, (4096,), dev, dtype).as_strided(shape, strides)
    own = x.contiguous()
    freq, pos = f.rotary_frequencies((d // 2,), device=dev), torch.arange(n, dtype=torch.int32, device=dev)
    for call in (f.rotary, f.rotary_backward):
        for a, b in zip(call(x, x, pos, freq, (d // 2,)), call(own, own, pos, freq, (d // 2,))):
            assert a.stride(-1) == 1 and torch.equal(a, b)
    if dtype != bf:
        return
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    o, lse = f.packed_attention(x, x, x, cu, causal=True, want_lse=True)
    want, wlse = f.packed_attention(own, own, own, cu, causal=True, want_lse=True)
    assert o.stride(-1) == 1 and torch.equal(o, want) and torch.equal(lse, wlse)
    got = f.packed_attention_backward(x, x, x, x, o, lse, cu, causal=True)
    for a, b in zip(got, f.packed_attention_backward(own, own, own, own, want, wlse, cu, causal=True)):
        assert a.stride(-1) == 1 and torch.equal(a, b)


@pytest.mark.parametrize("lengths,keys", [([40, 100], [40, 100]), ([700], [700]), ([1, 2], [3000, 4000]), ([3] * 70, [200] * 70)], ids=str)
def test_lse_of_rows_of_no_sequence_is_minus_infinity_beside_a_callers_output(dev, lengths, keys):
    """`out` keeps the rows of no sequence, an lse made by the call has -inf there, whatever its memory held."""
    g = gen_of("lse", lengths)
    start, tail, h, hk, d = 150, 200, 4, 2, 64
    at = [start + sum(lengths[:i]) for i in range(len(lengths) + 1)]
    ak = [sum(keys[:i]) for i in range(len(keys) + 1)]
    n = at[-1] + tail
    q, k, v = randn(g, (n, h, d), dev), randn(g, (ak[-1], hk, d), dev), randn(g, (ak[-1], hk, d), dev)
    cu_q, cu_k = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (at, ak))
    o, lse = f.packed_attention(q, k, v, cu_q, cu_k, want_lse=True)
    outside = torch.ones(n, dtype=torch.bool, device=dev)
    outside[at[0]:at[-1]] = False
    assert (lse[:, outside] == -math.inf).all() and not o[outside].any()
    mark = torch.full_like(o, 7.0)
    held = [torch.full((h, n), 7.0, device=dev) for _ in range(8)]      # what the next allocations of this size will hold
    torch.cuda.synchronize()
    del held
    for _ in range(4):
        out, lse2 = f.packed_attention(q, k, v, cu_q, cu_k, want_lse=True, out=mark)
        assert out is mark and torch.equal(lse2, lse)
        assert (mark[outside] == 7).all() and torch.equal(mark[~outside], o[~outside])
    mark.fill_(7)
    assert f.packed_attention(q, k, v, cu_q, cu_k, out=mark)[1] is None
    assert (mark[outside] == 7).all() and torch.equal(mark[~outside], o[~outside])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("m,n,causal", [(900, 700, False), (300, 700, False), (300, 300, True), (1, 6000, False), (20, 50, True)])
def test_large_values_stay_finite(dev, d, m, n, causal):
    """Values near 2^108 under weights that grow by 2^30 from one tile of keys to a later one: the sums on the way stay in range."""
    g = gen_of("large", d, m, n)
    h = 12 if m == 900 else 2      # no split of the keys, and a split, and neither
    q, k, v = randn(g, (m, h, d), dev), randn(g, (n, 1, d), dev), randn(g, (n, 1, d), dev, scale=2.0 ** 108)
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[2 * n // 3 + 8::97, :, 0] = 20.0 * d ** 0.5 / 8.0
    cu_q, cu_k = (torch.tensor([0, x], dtype=torch.int32, device=dev) for x in (m, n))
    ref = attention64(q, k, v, [0, m], [0, n], causal)
    assert torch.isfinite(ref["o"]).all()
    o, lse = f.packed_attention(q, k, v, cu_q, cu_k, causal=causal, want_lse=True)
    within(o, ref["o"], ref["tol_o"], "o")
    within(lse, ref["lse"], ref["tol_lse"], "lse")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("m,n,causal", [(900, 700, False), (300, 300, True), (1, 3000, False), (2, 2, True)])
def test_small_values_keep_their_precision(dev, d, m, n, causal):
    """Values near 2^-112: products with the smallest unnormalised weights that count are below fp32's normal numbers. An addition there is
    off by 2^-150 at most, and a row's sum of weights is 2^-20 or more: n 2^-130 beside the other errors."""
    g = gen_of("small", d, m, n)
    h = 12 if m == 900 else 2
    q, k, v = randn(g, (m, h, d), dev, scale=1.5), randn(g, (n, 1, d), dev), randn(g, (n, 1, d), dev, scale=2.0 ** -112)
    cu_q, cu_k = (torch.tensor([0, x], dtype=torch.int32, device=dev) for x in (m, n))
    ref = attention64(q, k, v, [0, m], [0, n], causal)
    o, lse = f.packed_attention(q, k, v, cu_q, cu_k, causal=causal, want_lse=True)
    within(o, ref["o"], ref["tol_o"] + n * 2.0 ** -130, "o")
    within(lse, ref["lse"], ref["tol_lse"], "lse")


@pytest.mark.parametrize("nq", [1, 300])
@pytest.mark.parametrize("d", [64, 128])
def test_weights_that_round_above_two_keep_their_gradient(dev, nq, d):
    """Scores from 2^26 to 2^27, where a weight comes back from lse off by e^8 either way: it is held to 2^0.5, and dK loses no term. Each
    sequence's queries see two keys of the same score (weights of a half) among others of none; dV shows the weight w that the pass
    used, since dV of a key is w dO, and dK is w (dP - delta) q scale."""
    seqs, keys = 128, 160
    a = (1 + torch.arange(seqs) / 128).to(bf)                            # exact scores: q is a everywhere, k a power of two
    q = a[:, None, None].expand(seqs, 1, d).repeat_interleave(nq, 0).to(dev)
    k = torch.zeros((seqs, keys, 1, d), dtype=bf)
    k[:, [40, 100]] = 2.0 ** 26 / d
    v = torch.zeros((seqs, keys, 1, d), dtype=bf)
    v[:, 40], v[:, 100] = 1.0, -1.0
    k, v = (x.view(-1, 1, d).to(dev) for x in (k, v))
    do = torch.zeros((seqs, nq, 1, d), dtype=bf)
    do[:, 0] = 1.0                                                       # one query of a sequence
    do = do.view(-1, 1, d).to(dev)
    cu_q, cu_k = (n * torch.arange(seqs + 1, dtype=torch.int32, device=dev) for n in (nq, keys))
    o, lse = f.packed_attention(q, k, v, cu_q, cu_k, scale=1.0, want_lse=True)
    assert not o.any()                                                   # a half of 1 and a half of -1
    _, dk, dv = f.packed_attention_backward(do, q, k, v, o, lse, cu_q, cu_k, scale=1.0)
    w = dv.view(seqs, keys, d)[:, 40, 0].double().cpu()
    got = dk.view(seqs, keys, d)[:, 40, 0].double().cpu() / (d * a.double())      # dP = d, delta = 0
    assert (w > 1.4).any() and (w < 0.1).any() and w.max() < 1.42        # both sides are met
    # dV and dK are rounded to bfloat16, w to 10 bits on its way and to bfloat16 for the product: 2^-8 each
    assert ((got - w).abs() <= 2.0 ** -6 * w).all(), (w, got)


@pytest.mark.parametrize("n,offsets,cache", [
    (200, [[0, 500], [-50, 100, 99999], [0, 150, 20, 200], [2 ** 31 - 1, -2 ** 31]], None),                 # blocks one behind another
    (1500, [[0, 99999], [-7, 1499, 300, 1500], [1500, 0], [700, 2 ** 31 - 1]], None),                        # in slots
    (300, [[(i * 97) % 331 - 15 for i in range(65)], [300 - 4 * i for i in range(76)], [0] * 64 + [2 ** 31 - 1]], None),   # of many sequences
    (6, [[0, 99], [5, 1, 6], [-3, 2, 1, 2 ** 31 - 1]], 9000),                                                # the keys split
], ids=["dense", "slots", "many", "split"])
def test_offsets_that_fall_or_leave_the_tensors_write_between_the_guards(dev, n, offsets, cache):
    """Offsets are taken into the tensors' range: results are of no use, but every row outside an output stays, the gradients' too."""
    g = gen_of("guards", n)
    h, hk, d, room = 4, 2, 64, cache or n
    q, k = randn(g, (n, h, d), dev), randn(g, (room, hk, d), dev)

    def guarded(like):
        whole = torch.full((like.shape[0] + 300, *like.shape[1:]), 7.0, dtype=bf, device=dev)
        return whole, whole[150:150 + like.shape[0]]

    for cu in offsets:
        c = torch.tensor(cu, dtype=torch.int32, device=dev)
        ck = c if cache is None else torch.tensor([x * 1000 % 2 ** 31 for x in cu], dtype=torch.int32, device=dev)
        if cache:
            p = f._abi.Packed(None, None, None, len(cu) - 1, n, room, d, 1, 1.0)
            assert f._abi.lib.fvsr_packed_attention_workspace(ctypes.byref(p), h, hk) > 0
        for used in (None, [(-1) ** i * 40 * i for i in range(len(cu) - 1)], [2 ** 31 - 1] * (len(cu) - 1)):
            us = None if used is None else torch.tensor(used, dtype=torch.int32, device=dev)
            for causal in (False, True):
                how = dict(causal=causal, used_k=us)
                wholes, outs = zip(*(guarded(x) for x in (q, q, k, k)))
                o, lse = f.packed_attention(q, k, k, c, ck, want_lse=True, out=outs[0], **how)
                f.packed_attention_backward(q, q, k, k, o, lse, c, ck, out=outs[1:], **how)
                torch.cuda.synchronize()
                for w in wholes:
                    assert (w[:150] == 7).all() and (w[-150:] == 7).all()
