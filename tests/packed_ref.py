"""64-bit references of the packed-row operators and the bounds that their
outputs keep. u = 2^-24 is half a step of binary32, 2^-11 of binary16."""
import math

import torch

U32, U16 = 2.0 ** -24, 2.0 ** -11


def attend(q, k, v, seen, rows_f16, cache_f16, scale=None):
    """q [n, heads, hd], k and v [len, kv heads, hd] (CPU, any type); row i sees
    the first seen[i] positions. Returns (output, bound) in 64 bits.

    The weight of position j is off by a factor 1 + eta_j, |eta_j| <= eta:
      scores: a sum of hd products in matrix instructions, whose additions may cut
        off (a whole step, 2 u, each); binary32 rows on a binary16 cache have q in
        two binary16 parts, off by 2^-22 of an element and 2^-39 of the largest;
      exponent: the scaled difference to the maximum, three roundings of terms no
        larger than 2 max |s| log2(e), and the exponential, two steps.
    The output is off by at most (2 eta + weights' rounding + n additions) of
    sum_j p_j |v_j|, and its own rounding. Weights: binary16 rows round them to
    binary16 (2^-11, and 2^-31 of the largest where they are tiny), binary32 rows
    on a binary16 cache to two parts (2^-22, and 2^-38 of the largest). Where the
    rounded weights are also summed, sum p (1 + d) v / sum p (1 + d) is off by
    sum p d (v - out) <= max |d| (sum p |v| + |out|)."""
    q, k, v = q.double(), k.double(), v.double()
    n, heads, hd = q.shape
    rep = heads // k.shape[1]
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    length = k.shape[0]
    if length == 0:
        return out, tol
    there = torch.arange(length)[None] < torch.as_tensor(seen)[:, None]
    for h in range(heads):
        kh, vh = k[:, h // rep], v[:, h // rep]
        s = (q[:, h] @ kh.T) * scale
        mag = (q[:, h].abs() @ kh.abs().T) * scale
        if cache_f16 and not rows_f16:
            part = 2.0 ** -22 * mag + 2.0 ** -39 * q[:, h].abs().amax(-1, keepdim=True) * kh.abs().sum(-1)[None] * scale
        else:
            part = 0.0
        s = s.masked_fill(~there, -math.inf)
        mag = (2 * hd * U32 * mag + part).masked_fill(~there, 0.0)
        top = s.amax(-1, keepdim=True).clamp(min=-1e300)
        p = torch.exp(s - top)
        total = p.sum(-1, keepdim=True)
        p = p / total.clamp(min=1e-300)
        big = torch.where(there, s.abs(), 0.0).amax(-1, keepdim=True)
        eta = mag.amax(-1, keepdim=True) + 6 * U32 * 2 * big + 4 * U32
        if rows_f16:
            weight, floor = U16, 2.0 ** -31
        elif cache_f16:
            weight, floor = 2.0 ** -22, 2.0 ** -38
        else:
            weight, floor = 0.0, 0.0
        steps = torch.as_tensor(seen).double()[:, None].clamp(max=length) * 2 * U32 + 16 * U32
        pv = p @ vh.abs()
        out[:, h] = p @ vh
        tol[:, h] = (2 * eta + weight + steps) * pv + weight * out[:, h].abs() + floor / total.clamp(min=1e-300) * (there.double() @ vh.abs()) \
            + (U16 if rows_f16 else U32) * out[:, h].abs() + 1e-30
        if rows_f16:
            tol[:, h] += 2.0 ** -25   # half a step of binary16's smallest values
    return out, tol


def normed_rotated(x, gamma, cs, eps, out_f16):
    """x [rows, heads, hd], cs [rows, hd / 2, 2]; (output, bound) in 64 bits.

    The sum of squares is off by (hd + 1) u at most, its root by half of that,
    the quotient, products and two-term sum by a few u more."""
    x, cs = x.double(), cs.double()
    hd = x.shape[-1]
    if gamma is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gamma.double()
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    out = torch.cat([a * c - b * s, a * s + b * c], -1)
    size = torch.cat([(a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()], -1)
    rel = ((hd + 1) / 2 + 8) * U32 if gamma is not None else 2 * U32
    tol = rel * size + (U16 if out_f16 else U32) * (out.abs() + rel * size) + (2.0 ** -25 if out_f16 else 1e-40)
    return out, tol


def check(got, want, tol, what=""):
    got = got.detach().double().cpu()
    off = (got - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((off / tol)[bad].max()), torch.nonzero(bad)[:4].tolist())
