"""Plain float64 forms of the packed operators, and how far a kernel may be from them.

U = 2^-24 is half a step of float32, relative; H[dtype] half a step of an output's type.
"""
import math

import torch

U = 2.0 ** -24
H = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def within(got, want, tol, what=""):
    """|got - want| <= tol, elementwise, and NaN and infinities where they are wanted."""
    got, want, tol = got.double().cpu(), want.double().cpu(), tol.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)), what
    assert torch.equal(got[~fine].nan_to_num(7e77), want[~fine].nan_to_num(7e77)), what
    off = (got - want).abs()[fine] - tol.expand_as(want)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, (what, float(off.max()), float((got - want)[fine].abs().max()))


def rms64(x, residual, weight, eps):
    """(total, y, rstd)"""
    t = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    t = t.double()
    rstd = 1 / torch.sqrt((t * t).mean(-1) + eps)
    y = t * rstd[:, None]
    return t, (y if weight is None else y * weight.double()), rstd


def rms_grad64(dy, total, rstd, weight, dsum):
    """(dx, dweight, and the sums of magnitudes that bound their errors)"""
    dy, n = dy.double(), total.double() * rstd.double()[:, None]
    g = dy if weight is None else dy * weight.double()
    m2, a2 = (g * n).mean(-1, keepdim=True), (g * n).abs().mean(-1, keepdim=True)
    r = rstd.double()[:, None]
    dx = r * (g - n * m2)
    size = r * (g.abs() + n.abs() * a2)
    if dsum is not None:
        dx = dx + dsum.double()
    return dx, (dy * n).sum(0), size, (dy * n).abs().sum(0)


def turn64(x, positions, frequencies, axes, halves, back=False):
    """x (L, H, D) turned by products of complex numbers."""
    n = sum(axes)
    axis = torch.tensor([a for a, p in enumerate(axes) for _ in range(p)])
    angle = positions.double().reshape(len(axes), -1)[axis].t() * frequencies.double()
    by = torch.polar(torch.ones_like(angle), -angle if back else angle)[:, None]
    first = torch.arange(n) if halves else 2 * torch.arange(n)
    second = first + (n if halves else 1)
    x = x.double()
    z = torch.complex(x[..., first], x[..., second]) * by
    out = x.clone()
    out[..., first], out[..., second] = z.real, z.imag
    return out


def spans(cu_q, cu_k, used):
    """(first query, queries, first key, keys) of each sequence."""
    cu_k = cu_q if cu_k is None else cu_k
    for b in range(len(cu_q) - 1):
        n = cu_k[b + 1] - cu_k[b]
        yield cu_q[b], cu_q[b + 1] - cu_q[b], cu_k[b], n if used is None else min(used[b], n)


def attention64(q, k, v, cu_q, cu_k=None, causal=False, scale=None, used=None, do=None):
    """A dict of o, lse (and dq, dk, dv) with `tol_` bounds, on the CPU; cu_q, cu_k and used are lists. Rows of no sequence: zeros,
    -inf.

    What a kernel may be off by. A score is a sum of D exact products in 32 bits, times the scale: D + 2 roundings of at most U of
    B = scale sum |q||k|. An exponential's argument is rounded once more in its size (below B + |lse| + 32), and the instruction is
    off by 2 U: the exponential is off by e = U ((D + 4) B + 2 (|lse| + 32)) of itself. P is rounded to bfloat16 for the product
    with V (2^-8), sums of n terms add n U, and o is rounded: 2^-8 |o| + (2^-8 + 2 e + (n + 8) U) sum p |v|. lse: e + (n + 8) U
    + 4 U |lse|. Backward, p comes from the lse: off by 2 e + (n + 12) U =: f. dP is off by (D + 2) U sum |do||v|, delta by sum
    |do| (what o is off by) and (D + 2) U of its size; dS by p times these two and (f + 2^-8) of itself; each product by (n + 2) U
    of its terms' sum, and 2^-8 of its result.
    """
    q, k, v = (x.double().cpu() for x in (q, k, v))
    lq, h, d = q.shape
    group = h // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    r = {"o": torch.zeros_like(q), "lse": torch.full((h, lq), -math.inf, dtype=torch.float64), "tol_o": torch.zeros_like(q),
         "tol_lse": torch.zeros(h, lq, dtype=torch.float64)}
    if do is not None:
        do = do.double().cpu()
        for n, x in (("dq", q), ("dk", k), ("dv", v)):
            r[n], r["tol_" + n] = torch.zeros_like(x), torch.zeros_like(x)
    b8 = 2.0 ** -8
    for q0, m, k0, n in spans(cu_q, cu_k, used):
        if m == 0 or n == 0:
            continue
        i, j = torch.arange(m)[:, None], torch.arange(n)[None]
        seen = (j < i + 1 + n - m) if causal else torch.ones(m, n, dtype=torch.bool)
        none = ~seen.any(1)
        for x in range(h):
            qq, kk, vv = q[q0:q0 + m, x], k[k0:k0 + n, x // group], v[k0:k0 + n, x // group]
            s = (qq @ kk.t() * scale).masked_fill(~seen, -math.inf)
            big = (scale * qq.abs() @ kk.abs().t()).masked_fill(~seen, 0).amax(1)
            lse = torch.logsumexp(s, 1)
            p = torch.where(seen, torch.exp(s - lse.nan_to_num(0, 0, 0)[:, None]), 0.0)
            # a key that a row does not see does not count, whatever it holds
            only = lambda w, y: torch.stack([(w[a][seen[a]][:, None] * y[seen[a]]).sum(0) for a in range(m)]) \
                if not torch.isfinite(y).all() else w @ y
            o, av = only(p, vv), only(p, vv.abs())
            e = U * ((d + 4) * big + 2 * (lse.abs().nan_to_num(0, 0, 0) + 32))
            tol_o = b8 * o.abs() + (b8 + 2 * e + (n + 8) * U)[:, None] * av
            r["o"][q0:q0 + m, x], r["tol_o"][q0:q0 + m, x] = o.masked_fill(none[:, None], 0), tol_o.masked_fill(none[:, None], 0)
            r["lse"][x, q0:q0 + m] = lse
            r["tol_lse"][x, q0:q0 + m] = (e + (n + 8) * U + 4 * U * lse.abs()).nan_to_num(0, 0, 0)
            if do is None:
                continue
            dd = do[q0:q0 + m, x]
            f = (2 * e + (n + 12) * U)[:, None]
            dp = dd @ vv.t()
            delta = (p * dp.masked_fill(~seen, 0)).sum(1, keepdim=True)
            ds = torch.where(seen, p * (dp - delta), 0.0)
            off_dp = (d + 2) * U * (dd.abs() @ vv.abs().t())
            off_delta = (dd.abs() * (tol_o + (d + 2) * U * o.abs())).sum(1, keepdim=True)
            off_ds = p * (off_dp + off_delta) + (f + b8) * ds.abs()
            off_p = (f + b8) * p
            r["dq"][q0:q0 + m, x] = scale * (ds @ kk)
            r["tol_dq"][q0:q0 + m, x] = scale * (off_ds @ kk.abs() + (n + 2) * U * (ds.abs() @ kk.abs()))
            r["dk"][k0:k0 + n, x // group] += scale * (ds.t() @ qq)
            r["tol_dk"][k0:k0 + n, x // group] += scale * (off_ds.t() @ qq.abs() + (group * m + 2) * U * (ds.abs().t() @ qq.abs()))
            r["dv"][k0:k0 + n, x // group] += p.t() @ dd
            r["tol_dv"][k0:k0 + n, x // group] += off_p.t() @ dd.abs() + (group * m + 2) * U * (p.t() @ dd.abs())
    if do is not None:
        for n in ("dq", "dk", "dv"):
            # 2^-8 of the result as it is: off by what it may be off by
            r["tol_" + n] = r["tol_" + n] * (1 + b8) + b8 * r[n].abs()
    return r
