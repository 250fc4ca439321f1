"""Plain 64-bit forms of the paged-cache operators, and the error bounds that the kernels'
roundings allow (each bound is arithmetic on the operator's formula, no measured slack).

u(t) = torch.finfo(t).eps / 2 is the largest relative rounding error of type t.

Append: one rotated element is two products and a sum in fp32 (each off by at most 2^-24 of
its result), then one rounding to the output's type: u*|y| + 2^-22*(|x1| + |x2|), plus half the
type's smallest subnormal where the result is below its normal range.

Attention: products of two 16-bit values are exact in fp32; a sum of n terms in the MMA's fp32
accumulators is off by at most n*2^-23 of the sum of magnitudes (2^-23 instead of 2^-24: the
tensor cores may truncate). So a score is off by ds = scale * D * 2^-23 * sum|q||k|, a weight
2^(s-m) by a factor within ds + |s-m|*2^-23 + 2^-21 (exp2f and its rounded argument), and by
the rounding of P in front of the second product. Weighted sums over n keys add n*2^-22, once
for P.V and once for the sum of P. With A = sum p|v| / sum p this bounds the output by
A * 2 * (that), plus one rounding of the result to its type.
"""
import math

import torch


def u(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """Half the distance between neighbours below the normal range."""
    return {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float8_e4m3fn: 2.0 ** -10}[t]


def rotate64(x, cos, sin, interleaved):
    """x [T,H,D] turned by cos, sin [T, R/2] (fp64 inside), and |x1|+|x2| for the bound."""
    x = x.double()
    y, mag = x.clone(), x.abs()
    r = 2 * cos.shape[-1]
    c, s = cos.double()[:, None], sin.double()[:, None]
    i1 = torch.arange(0, r, 2) if interleaved else torch.arange(0, r // 2)
    i2 = i1 + 1 if interleaved else i1 + r // 2
    a, b = x[..., i1], x[..., i2]
    y[..., i1], y[..., i2] = a * c - b * s, b * c + a * s
    mag[..., i1] = mag[..., i2] = a.abs() + b.abs()
    return y, mag


def attend64(q, k, v, seen, scale, p_round, out):
    """q [n,g,d], k and v [m,d], seen [n,m] -> (o [n,g,d], bound on its error, lse [n,g],
    bound); p_round is the relative rounding of P that the kernel is allowed."""
    q, k, v = q.double(), k.double(), v.double()
    n, g, d = q.shape
    m = k.shape[0]
    if m == 0:
        z = torch.zeros_like(q)
        return z, z, torch.full((n, g), -math.inf, dtype=torch.float64, device=q.device), z[..., 0]
    s = torch.einsum("ngd,md->ngm", q, k) * scale
    ds = scale * d * 2.0 ** -23 * torch.einsum("ngd,md->ngm", q.abs(), k.abs())
    s = s.masked_fill(~seen[:, None], -math.inf)
    ds = ds.masked_fill(~seen[:, None], 0.0)
    top = s.amax(-1, keepdim=True)
    some = seen.any(-1)[:, None, None]
    ref = torch.where(some, top, torch.zeros_like(top))
    p = (s - ref).exp().masked_fill(~seen[:, None], 0.0)
    l = p.sum(-1, keepdim=True)
    o = torch.einsum("ngm,md->ngd", p, v.masked_fill(~seen.any(0)[:, None], 0.0)) / l
    o = torch.where(some, o, torch.zeros_like(o))
    mag = torch.where(some, torch.einsum("ngm,md->ngd", p, v.abs().masked_fill(~seen.any(0)[:, None], 0.0)) / l,
                      torch.zeros_like(o))
    # Weights far below the largest carry larger argument errors but count for p only.
    arg = ds + ((s - ref).abs() * 2.0 ** -23).masked_fill(~seen[:, None], 0.0)
    worst = torch.where(some, ((arg * p).sum(-1, keepdim=True) / l + ds.amax(-1, keepdim=True)), torch.zeros_like(l))
    each = torch.where(some, torch.einsum("ngm,md->ngd", arg * p, v.abs()) / l, torch.zeros_like(o))
    rel = 2 * (2.0 ** -21 + m * 2.0 ** -22) + p_round
    bound = 2 * each + mag * (2 * worst + rel) + u(out) * o.abs() + tiny(out)
    lse = torch.where(some, top + l.log(), torch.full_like(l, -math.inf))[..., 0]
    lse_bound = 2 * worst[..., 0] + rel + 2.0 ** -22 * torch.where(some[..., 0], lse.abs(), torch.zeros_like(lse))
    return o, bound, lse, lse_bound


def gather_pages(pool, row, length):
    """Rows 0..length-1 of every head of one sequence: [Hkv, length, D] in fp32."""
    size = pool.shape[2]
    pages = row[: -(-length // size)].long()
    if pool.dtype == torch.float8_e4m3fn:
        x = pool.view(torch.uint8)[pages].view(pool.dtype).float()
    else:
        x = pool[pages].float()
    return x.transpose(0, 1).reshape(pool.shape[1], -1, pool.shape[3])[:, :length]


def check(got, want, bound, what=""):
    got = got.double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf), f"{what}: infinity in other places"
    assert torch.equal(got[inf], want[inf]), f"{what}: infinity of other sign"
    fine = ~(nan | inf)
    over = (got[fine] - want[fine]).abs() / bound.expand_as(want)[fine].clamp_min(1e-300)
    if over.numel():
        assert float(over.max()) <= 1.0, f"{what}: error {float(over.max()):.3g} of its bound"
