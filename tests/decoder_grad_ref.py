"""Gradients of softmax attention in 64 bits, from the output that a forward pass kept, with two bounds.

The kept output (rounded to the operands' type) is an input of a backward pass: D = rowsum(dout o out). With the same
D in the reference, its rounding costs the comparison nothing, and what is left is

* ``worst``: the largest error of an element, every rounding at its half step and all of one sign (U = 2^-24 for fp32
  arithmetic, H = eps / 2 of the stored type);
* ``spread``: the roundings of P and dS to 16 bits do not conspire. Each is off by at most H, so one element of
  sum_j t_j x_j is off by about sqrt(sum_j (H t_j x_j)^2) and hardly any by more than a few times that; over a
  whole tensor the error's norm cannot pass twice the norm of these, for one standard deviation of a rounding is at
  most H / sqrt(3) (uniform over a half step on either side). What is not a rounding to 16 bits enters at its worst.

A part of the keys or of the rows that was left out, or a missing P D, is several times the second bound and hidden
by the first.
"""

from __future__ import annotations

import torch

from decoder_ref import U, check, half

EXP = 48 * U  # relative error of an exponential taken as a polynomial on the FMA pipe (2.6e-6, 44 U)


def gradients_ref(q, k, v, keep, scale, dout, out, low=False, delta_term=True, key_parts=None, row_parts=None):
    """{"dq", "dk", "dv"}: (gradient, worst, spread, exact part of the spread).

    ``keep``: bool, broadcast to (B, 1, Sq, Sk). The last three arguments plant mistakes: D left out, or only
    some keys (bool, Sk) summed into dq, or only some rows (bool, Sq) into dk and dv."""
    B, Hq, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    G = Hq // Hkv
    h = half(q.dtype)
    hp = h if low else 0.0
    keep = keep.expand(B, 1, Sq, Sk)
    anyone = keep.any(2)[..., None]
    qd, do = q.double(), dout.double()
    kd = k.double().masked_fill(~anyone, 0.0).repeat_interleave(G, 1)
    vd = v.double().masked_fill(~anyone, 0.0).repeat_interleave(G, 1)
    s = (qd @ kd.transpose(-1, -2) * scale).masked_fill(~keep, float("-inf"))
    p = torch.softmax(s, -1).masked_fill(~keep.any(-1, keepdim=True), 0.0)
    # scores: D products and the scale; the exponent 4 U of the score; the kept log-sum-exp the same again, and its sum
    ds = ((D + 4) * U * abs(scale) * (qd.abs() @ kd.abs().transpose(-1, -2))).masked_fill(~keep, 0.0)
    size = s.abs().masked_fill(~keep, 0.0)
    rho = 2 * (ds + 4 * U * size).amax(-1, keepdim=True) + (Sk + 32) * U + (EXP if low else 0.0)
    o = out.double()
    delta = (do * o).sum(-1, keepdim=True) if delta_term else 0.0
    delta_err = (D + 4) * U * (do.abs() * o.abs()).sum(-1, keepdim=True)
    dp = do @ vd.transpose(-1, -2)
    dp_err = (D + 4) * U * (do.abs() @ vd.abs().transpose(-1, -2))
    t = p * (dp - delta)
    t_err = (rho + 4 * U) * t.abs() + (1 + rho) * p * (dp_err + delta_err)

    def group(x):
        return x.view(B, Hkv, G, Sk, D).sum(2)

    def entry(a, a_err, x, n, f, over_rows):
        """f sum a x of n products; a is off by a_err before its rounding to 16 bits."""
        def mm(l, r):
            return group(l.transpose(-1, -2) @ r) if over_rows else l @ r

        def kept(l):
            part = row_parts if over_rows else key_parts
            if part is None:
                return l
            return l * (part[:, None] if over_rows else part)

        g = f * mm(kept(a), x)
        exact = abs(f) * mm(a_err + (n + 8) * U * a.abs(), x.abs())
        worst = exact + hp * abs(f) * mm(a.abs() + a_err, x.abs())
        spread2 = (hp * f) ** 2 * mm((a.abs() + a_err) ** 2, x ** 2) + (h * g) ** 2
        return g, worst + h * (g.abs() + worst), spread2.sqrt(), exact

    n = G * Sq
    return {"dq": entry(t, t_err, kd, Sk, scale, False), "dk": entry(t, t_err, qd, n, scale, True),
            "dv": entry(p, rho * p, do, n, 1.0, True)}


def check_gradients(got: dict, refs: dict, what=""):
    """Every element within its worst case, and every tensor's error within its spread."""
    for name, g in got.items():
        ref, worst, spread, exact = refs[name]
        check(g, ref, worst, f"{what}{name}")
        if g.numel():
            err = (g.detach().double() - ref).norm().item()
            most = 2 * spread.norm().item() + exact.norm().item()
            assert err <= most, f"{what}{name}: error of norm {err:.3e}, at most {most:.3e} (of {ref.norm().item():.3e})"
