"""The gradient bounds accept a backward pass with its roundings and refuse one that lost a part or a term."""

from __future__ import annotations

import pytest
import torch

from decoder_grad_ref import check_gradients, gradients_ref

CASES = [(2, 2, 2, 1, 2000, 64), (1, 4, 1, 300, 100, 64), (2, 2, 1, 40, 300, 32)]


def _case(B, Hq, Hkv, Sq, Sk, D):
    g = torch.Generator().manual_seed(7)
    bf = lambda *s: torch.randn(*s, generator=g).bfloat16()
    q, k, v, dout = bf(B, Hq, Sq, D), bf(B, Hkv, Sk, D), bf(B, Hkv, Sk, D), bf(B, Hq, Sq, D)
    keep = torch.rand(B, 1, 1, Sk, generator=g) < 0.9
    keep[..., 0] = True
    return q, k, v, keep, dout


def _backward(q, k, v, keep, scale, dout):
    """P and dS rounded to bf16 before their products, results rounded once; (out, gradients)."""
    G = q.shape[1] // k.shape[1]
    qd, do = q.double(), dout.double()
    kd, vd = (t.double().repeat_interleave(G, 1) for t in (k, v))
    p = torch.softmax((qd @ kd.transpose(-1, -2) * scale).masked_fill(~keep, float("-inf")), -1)
    low = lambda t: t.bfloat16().double()
    out = (low(p) @ vd).bfloat16()
    t = low(p * (do @ vd.transpose(-1, -2) - (do * out.double()).sum(-1, keepdim=True)))
    group = lambda x: x.view(k.shape[0], k.shape[1], G, *k.shape[2:]).sum(2)
    return out, {"dq": (scale * (t @ kd)).bfloat16(), "dk": group(scale * (t.transpose(-1, -2) @ qd)).bfloat16(),
                 "dv": group(low(p).transpose(-1, -2) @ do).bfloat16()}


@pytest.mark.parametrize("shape", CASES)
def test_roundings_are_within_the_bounds(shape):
    q, k, v, keep, dout = _case(*shape)
    for scale in (shape[-1] ** -0.5, -0.1):
        out, got = _backward(q, k, v, keep, scale, dout)
        check_gradients(got, gradients_ref(q, k, v, keep, scale, dout, out, low=True))


@pytest.mark.parametrize("shape", CASES)
def test_mistakes_are_outside(shape):
    """Planted in the reference: D left out, a tenth of the keys not in dq, an eighth of the rows not in dk and dv."""
    q, k, v, keep, dout = _case(*shape)
    scale = shape[-1] ** -0.5
    out, got = _backward(q, k, v, keep, scale, dout)
    Sq, Sk = shape[3], shape[4]

    def refused(names, **plant):
        refs = gradients_ref(q, k, v, keep, scale, dout, out, low=True, **plant)
        for n in names:
            with pytest.raises(AssertionError, match=n):
                check_gradients({n: got[n]}, refs)

    refused(("dq", "dk"), delta_term=False)
    keys = torch.arange(Sk)
    for part in range(10):
        refused(("dq",), key_parts=keys * 10 // Sk != part)
    if Sq >= 8:
        rows = torch.arange(Sq)
        for part in range(8):
            refused(("dk", "dv"), row_parts=rows * 8 // Sq != part)
