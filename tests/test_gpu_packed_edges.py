"""Calls of the packed operators at the edges of what their documentation allows: the packed pass' rings at their shortest, views that
overlap, rows of no sequence, very large scores and values, offsets that fall. Against the float64 forms of tests/packed_reference.py."""
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
