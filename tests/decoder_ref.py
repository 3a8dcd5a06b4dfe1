"""64-bit definitions of the decoder operators, each with a bound on what correct rounding may cost.

The bounds are worst cases counted in half steps: U = 2^-24 for fp32 arithmetic, H = eps / 2 of the stored
type (bf16 2^-8) for every value that is rounded to it. A sum of n products, in any order, is off by at most
n U times the sum of its absolute terms.
"""

from __future__ import annotations

import torch

U = 2.0 ** -24


def half(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def qk_ref(x, w, positions, inv_freq, eps, interleaved, dy=None):
    """(y, bound[, dx, bound, dw, bound]) of one tensor (B, H, S, D), all float64."""
    B, H, S, D = x.shape
    h, x = half(x.dtype), x.double()
    wd = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.double()
    R = 2 * inv_freq.numel()
    pos = positions.double().expand(B, S)
    ang = pos[:, None, :, None] * inv_freq.double()
    cos, sin = ang.cos(), ang.sin()

    def turn(n, c, s):
        a, b = (n[..., 0:R:2], n[..., 1:R:2]) if interleaved else (n[..., : R // 2], n[..., R // 2: R])
        ya, yb = a * c - b * s, a * s + b * c
        y = torch.stack((ya, yb), -1).flatten(-2) if interleaved else torch.cat((ya, yb), -1)
        return torch.cat((y, n[..., R:]), -1)

    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    u = x * r
    y = turn(u * wd, cos, sin)
    one = torch.ones_like(cos)

    def sizes(n):
        """|a cos| + |b sin| (|a sin| + |b cos|) of every pair, and |a| + |b|."""
        n = n.abs()
        both = [torch.maximum(turn(n, c, s).abs(), turn(n, c, -s).abs()) for c, s in ((cos.abs(), sin.abs()), (one, one))]
        return both

    # r: D squares added and halved by the root; u, the weight, two products and a sum. Cosine and sine are off
    # absolutely, not relatively: the turn, at most 1/2, is rounded by 2^-26, so the angle by 2 pi 2^-26 < 1.6 U
    # and cos(t + e) by up to e |sin t|, which |a cos t| says nothing about where cos t is near 0; with the
    # function's own two half steps (values up to 1) and the 64-bit product's error at 10^7 turns, 4 U of |a| + |b|.
    k = (D / 2 + 24) * U
    size, pair = sizes(u * wd)
    err = k * size + 4 * U * pair
    res = [y, h * y.abs() + (1 + h) * err]
    if dy is None:
        return res
    dn = turn(dy.double(), cos, -sin)
    dn_size, dn_pair = sizes(dy.double())
    dn_size = torch.maximum(dn_size, dn_pair)  # the pair's size bounds both kinds of error
    g = dn * wd
    c = (g * u).mean(-1, keepdim=True)
    dx = r * (g - u * c)
    g_size = dn_size * wd.abs()
    c_size = (g_size * u.abs()).mean(-1, keepdim=True)
    k2 = (2 * D + 48) * U
    res += [dx, h * dx.abs() + (k2 + h * k2) * r * (g_size + u.abs() * c_size)]
    rows = B * H * S
    hw = U if w is None else half(w.dtype)
    dw = (dn * u).sum((0, 1, 2))
    dw_size = (dn_size * u.abs()).sum((0, 1, 2))
    # a column's rows are added within a thread, over the groups of a block, and over the blocks
    res += [dw, hw * dw.abs() + (min(rows, 4096) + D / 2 + 64) * U * dw_size]
    return res


def attention_ref(q, k, v, keep, scale, dout=None, low=False):
    """Softmax attention of (B, Hq, Sq, D) over (B, Hkv, Sk, D); ``keep``: bool, broadcast to (B, 1, Sq, Sk).

    Returns out and its bound and, with ``dout``, (dq, bound), (dk, bound), (dv, bound). ``low``: probabilities
    (and dS) are rounded to the operands' 16-bit type before their products, as tensor cores need it."""
    B, Hq, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    G = Hq // Hkv
    h = half(q.dtype)
    hp = h if low else 0.0
    keep = keep.expand(B, 1, Sq, Sk)
    anyone = keep.any(2)[..., None]  # (B, 1, Sk, 1): hidden from every row
    qd = q.double()
    kd = k.double().masked_fill(~anyone, 0.0).repeat_interleave(G, 1)
    vd = v.double().masked_fill(~anyone, 0.0).repeat_interleave(G, 1)
    s = (qd @ kd.transpose(-1, -2) * scale).masked_fill(~keep, float("-inf"))
    live = keep.any(-1, keepdim=True)
    p = torch.softmax(s, -1).masked_fill(~live, 0.0)
    out = p @ vd
    # a score is off by ds; a probability by its own score's and the normaliser's error, the exponentials' few
    # half steps, and the sum over the keys
    ds = ((D + 4) * U * abs(scale) * (qd.abs() @ kd.abs().transpose(-1, -2))).masked_fill(~keep, 0.0)
    size = s.abs().masked_fill(~keep, 0.0)
    worst = (ds + 4 * U * size).amax(-1, keepdim=True) if Sk else torch.zeros_like(live, dtype=torch.float64)
    rho = 2 * worst + (Sk + 32) * U
    mass = p @ vd.abs()
    out_err = (rho + hp + (Sk + 8) * U) * mass
    res = [out, out_err + h * (out.abs() + out_err)]
    if dout is None:
        return res
    do = dout.double()
    delta = (do * out).sum(-1, keepdim=True)
    delta_err = (do.abs() * res[1]).sum(-1, keepdim=True) + (D + 4) * U * (do.abs() * out.abs()).sum(-1, keepdim=True)
    dp = do @ vd.transpose(-1, -2)
    dp_err = (D + 4) * U * (do.abs() @ vd.abs().transpose(-1, -2))
    t = p * (dp - delta)
    t_err = (rho + 4 * U) * t.abs() + (1 + rho) * p * (dp_err + delta_err)
    t_err = t_err + hp * (t.abs() + t_err)
    fin = lambda x, e: (x, e + h * (x.abs() + e))
    sum_g = lambda x: x.view(B, Hkv, G, Sk, D).sum(2)
    dq = scale * (t @ kd)
    dq_err = abs(scale) * ((t_err + (Sk + 8) * U * t.abs()) @ kd.abs())
    n = (G * Sq + 8) * U
    dk = sum_g(scale * (t.transpose(-1, -2) @ qd))
    dk_err = sum_g(abs(scale) * ((t_err + n * t.abs()).transpose(-1, -2) @ qd.abs()))
    p_err = (rho + hp + n) * p
    dv = sum_g(p.transpose(-1, -2) @ do)
    dv_err = sum_g(p_err.transpose(-1, -2) @ do.abs())
    return res + [*fin(dq, dq_err), *fin(dk, dk_err), *fin(dv, dv_err)]


def check(got, ref, bound, what=""):
    got = got.detach().double()
    assert got.shape == ref.shape, f"{what}: shape {tuple(got.shape)}, expected {tuple(ref.shape)}"
    if got.numel() == 0:
        return
    assert torch.isfinite(got).all(), f"{what}: not finite"
    excess = ((got - ref).abs() - bound).max().item()
    assert excess <= 1e-30, f"{what}: {excess:.3e} beyond its bound (largest bound {bound.max().item():.3e})"
