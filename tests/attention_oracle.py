"""Plain 64-bit attention and rotary positions, and the error a correct
kernel may make, for the GPU parity tests."""
from __future__ import annotations

import math

import torch

# Unit roundoff of each output type.
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# Half the spacing of the type's subnormals.
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def attend(q, k, v, first, causal, window, scale):
    """q [rows][hq][d] at positions first, first + 1, ... over k, v [keys][hkv][d], in 64 bits.
    Masked keys are left out by indexing, so what they hold cannot matter.

    Returns (out, lse, tol_out, tol_lse).  The tolerances follow from the types: with u the
    type's unit roundoff, a 32-bit product of d terms is off by at most g = (d + 2) 2^-24
    scale sum|q||k|; a weight exp(s - m) by 2 g + u / 16 (its exponential's own error) and by u
    when it is rounded to the type for the product with v (and the sum of weights by as much, if
    it is taken over the rounded ones), plus half a subnormal; sums of n
    terms in 32 bits by n 2^-24; and the output by u of itself."""
    dtype = q.dtype
    u, tiny = UNIT[dtype], TINY[dtype]
    q, k, v = q.double(), k.double(), v.double()
    rows, hq, d = q.shape
    keys, hkv, _ = k.shape
    out = torch.zeros_like(q)
    tol = torch.full_like(q, tiny)
    lse = torch.full((rows, hq), -math.inf, dtype=torch.float64, device=q.device)
    tol_lse = torch.zeros_like(lse)
    for r in range(rows):
        place = first + r
        lo = max(0, place - window + 1) if window else 0
        hi = min(keys, place + 1) if causal else keys
        if hi <= lo:
            continue
        n = hi - lo
        kk = k[lo:hi].repeat_interleave(hq // hkv, dim=1)
        vv = v[lo:hi].repeat_interleave(hq // hkv, dim=1)
        s = torch.einsum("hd,jhd->hj", q[r], kk) * scale
        g = (torch.einsum("hd,jhd->hj", q[r].abs(), kk.abs()).amax(dim=1) * abs(scale) *
             (d + 2) * 2.0 ** -24)
        m = s.amax(dim=1, keepdim=True)
        p = torch.exp(s - m)
        l = p.sum(dim=1, keepdim=True)
        o = torch.einsum("hj,jhd->hd", p / l, vv)
        a = torch.einsum("hj,jhd->hd", p / l, vv.abs())
        out[r] = o
        lse[r] = (m + l.log())[:, 0]
        eps = (2 * g + u / 16 + (n + d) * 2.0 ** -24)[:, None]
        tol[r] += 1.05 * (u * o.abs() + (2 * u + 2 * eps) * a +
                          tiny * vv.abs().sum(dim=0) / l)
        tol_lse[r] = 2 * g + u / 16 + (n + 8) * 2.0 ** -24 + lse[r].abs() * 2.0 ** -22
    return out, lse, tol, tol_lse


def rotate(x, positions, rot, layout, freq, amplitude=1.0):
    """x [tokens][heads][d] in 64 bits; freq [rot/2] radians a position."""
    x = x.double().clone()
    if rot == 0:
        return x
    angle = positions.double()[:, None] * freq.to(x.device)
    c, s = angle.cos()[:, None] * amplitude, angle.sin()[:, None] * amplitude
    first, second = ((slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else
                     (slice(0, rot, 2), slice(1, rot, 2)))
    a, b = x[..., first].clone(), x[..., second].clone()
    x[..., first], x[..., second] = a * c - b * s, a * s + b * c
    return x


def rotary_tolerance(x, rot, dtype, amplitude=1.0):
    """What a rotation in 32 bits rounded once to dtype may be off by: both products and the sum
    round (2^-24 each), sine and cosine are good to 2^-22 and the reduced angle to 2^-23 of half a
    turn, so 2^-20 of the pair's size is enough; the output rounds once."""
    size = x.double().abs().amax(dim=-1, keepdim=True) * max(1.0, abs(amplitude))
    return 2.0 * size * (2.0 ** -20 + 1.05 * UNIT[dtype]) + TINY[dtype]
