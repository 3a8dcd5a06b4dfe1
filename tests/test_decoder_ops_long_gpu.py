"""Decoder attention over millions of keys walked by one CTA."""

from __future__ import annotations

import pytest
import torch

import trnsparse_b200 as ts
from trnsparse_b200 import _lib
from decoder_ref import check

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _ones(B, Sq, Sk, D, dtype=BF16):
    """Queries, keys and values of ones, the keys of all sequences the same memory. The result is 1: the scores are
    equal, P is 1, and sums of ones are exact in fp32 up to 2^24."""
    q = torch.ones(B, 1, Sq, D, device="cuda", dtype=dtype)
    k = torch.ones(1, 1, Sk, D, device="cuda", dtype=dtype).expand(B, 1, Sk, D)
    out = ts.cross_attention(q, k, k)
    check(out, torch.ones_like(out, dtype=torch.float64), torch.full_like(out, 2.0 ** -8, dtype=torch.float64), "out")
    assert _lib.device_error() == 0


def test_row_sums_pass_2_to_the_24():
    """148 items of 17 rows: a whole one for every CTA."""
    _ones(148, 17, 1 << 25, 8)


@pytest.mark.parametrize("B,Sq,D", [(148, 17, 64), (148, 200, 128), (3, 40, 64)])
def test_long_sums_do_not_shrink(B, Sq, D):
    """2^21 keys, values of mean 1, whole on a CTA or cut. The tensor core cuts a product to the accumulator's last place:
    less than 2^-25 of the sum each, so at most 2^-8 of it over the 2^17 keys of one accumulator. The other roundings
    (P and the result, half a step 2^-8 each) go both ways: their mean over N results stays below 4 2^-8 / sqrt(N)."""
    g = torch.Generator(device="cuda").manual_seed(111)
    n = 1 << 21
    q, k = (torch.randn(1, 1, s, D, generator=g, device="cuda").to(BF16) for s in (Sq, n))
    v = (1 + torch.randn(1, 1, n, D, generator=g, device="cuda")).to(BF16)
    out = ts.cross_attention(*(t.expand(B, *t.shape[1:]) for t in (q, k, v)))
    assert all(torch.equal(out[i], out[0]) for i in range(1, B) if B == 148)
    ref = torch.cat([torch.softmax(r.double() @ k[0, 0].double().T * D ** -0.5, -1) @ v[0, 0].double()
                     for r in q[0, 0].split(20)])
    for o in out[:3, 0].double():
        bias = ((o - ref) * ref.sign()).mean().item() / ref.abs().mean().item()
        assert abs(bias) <= 2.0 ** -8 + 4 * 2.0 ** -8 / ref.numel() ** 0.5
        assert ((o - ref).norm() / ref.norm()).item() <= 2 * 2.0 ** -8


def test_flushed_sums_follow_a_rising_maximum():
    """The scores rise by 40 over the keys, a maximum that moves between and after flushes; the last keys decide."""
    n, D = 1 << 19, 64
    g = torch.Generator(device="cuda").manual_seed(112)
    k = torch.zeros(1, 1, n, D, device="cuda")
    k[..., 0] = torch.linspace(0, 40, n, device="cuda")
    k, v = k.to(BF16), torch.randn(1, 1, n, D, generator=g, device="cuda").to(BF16)
    q = torch.zeros(148, 1, 17, D, device="cuda", dtype=BF16)
    rise = torch.tensor([1.0, 0.0, -1.0, 0.25], device="cuda")
    q[:, 0, :4, 0] = rise.to(BF16)
    out = ts.cross_attention(q, k.expand(148, 1, n, D), v.expand(148, 1, n, D), scale=1.0)
    p = torch.softmax(rise[:, None].double() * k[0, 0, :, 0].double(), -1)
    ref, mass = p @ v[0, 0].double(), p @ v[0, 0].double().abs()
    # P rounded to bf16, the result too, and the chain's cuts (above)
    check(out[0, 0, :4], ref, 3 * 2.0 ** -8 * mass, "out")


def test_an_item_that_takes_more_than_a_second():
    """Sequence 0 has 2^28 keys, 739 others one (1.3 us a tile: 2.8 s). The CTA that has it has five items; the roles
    that are through with their part of the first one (the list of items, the warps of rows 128 to 255) wait for the
    others, longer than a pipeline stage ever takes. The last key of sequence 0 outweighs all others together."""
    B, Sk, D = 740, 1 << 28, 8
    k = torch.zeros(1, 1, Sk, D, device="cuda", dtype=BF16)
    v = torch.ones(1, 1, Sk, D, device="cuda", dtype=BF16)
    k[..., -1, :], v[..., -1, :], v[..., 0, :] = 16, 2, 3
    lengths = torch.ones(B, dtype=torch.int32, device="cuda")
    lengths[0] = Sk
    q = torch.ones(B, 1, 17, D, device="cuda", dtype=BF16)
    out = ts.cross_attention(q, k.expand(B, 1, Sk, D), v.expand(B, 1, Sk, D), lengths, scale=1.0)
    assert _lib.device_error() == 0
    assert (out[0] == 2).all() and (out[1:] == 3).all()  # exp(-128) 2^28 is nothing


def _bias(got, ref):
    """Mean error along the reference, and what the cuts of 2^17 products and the mean of the roundings allow."""
    got, ref = got.double().flatten(), ref.flatten()
    return abs(((got - ref) * ref.sign()).mean().item()) / ref.abs().mean().item(), 2.0 ** -8 * (1 + 4 / ref.numel() ** 0.5)


def test_long_sums_of_dq_do_not_shrink():
    """2^21 keys that are the values too: dq is the keys' covariance times dout, a sum that grows all along."""
    g = torch.Generator(device="cuda").manual_seed(113)
    B, Sq, n, D = 148, 17, 1 << 21, 64
    q, dout = (torch.randn(1, 1, Sq, D, generator=g, device="cuda").to(BF16) for _ in range(2))
    k = torch.randn(1, 1, n, D, generator=g, device="cuda").to(BF16)
    leaf = q.expand(B, 1, Sq, D).contiguous().requires_grad_(True)
    out = ts.cross_attention(leaf, k.expand(B, 1, n, D), k.expand(B, 1, n, D))
    dq, = torch.autograd.grad(out, leaf, dout.expand(B, 1, Sq, D))
    kd, do = k[0, 0].double(), dout[0, 0].double()
    p = torch.softmax(q[0, 0].double() @ kd.T * D ** -0.5, -1)
    delta = (do * out[0, 0].detach().double()).sum(-1, keepdim=True)
    ref = (p * (do @ kd.T - delta)) @ kd * D ** -0.5
    for i in (0, 1, B - 1):
        got, most = _bias(dq[i, 0], ref)
        assert got <= most


def test_long_sums_of_dk_and_dv_do_not_shrink():
    """2^21 query rows: dv is a sum of positive terms, dk of the queries' covariance."""
    g = torch.Generator(device="cuda").manual_seed(114)
    B, Sq, n, D = 75, 1 << 21, 100, 8
    q = torch.randn(1, 1, Sq, D, generator=g, device="cuda").to(BF16)
    k = 0.2 * torch.randn(1, 1, n, D, generator=g, device="cuda")
    k = k.to(BF16).expand(B, 1, n, D).contiguous().requires_grad_(True)
    v = torch.randn(1, 1, n, D, generator=g, device="cuda").to(BF16).expand(B, 1, n, D).contiguous().requires_grad_(True)
    dout = (q + 1).to(BF16)
    out = ts.cross_attention(q.expand(B, 1, Sq, D), k, v)
    dk, dv = torch.autograd.grad(out, (k, v), dout.expand(B, 1, Sq, D))
    qd, do, kd, vd = (t.detach()[0, 0].double() for t in (q, dout, k, v))
    p = torch.softmax(qd @ kd.T * D ** -0.5, -1)
    delta = (do * out[0, 0].detach().double()).sum(-1, keepdim=True)
    refs = (p * (do @ vd.T - delta)).T @ qd * D ** -0.5, p.T @ do
    for i in (0, B - 1):
        for grad, ref in zip((dk, dv), refs):
            got, most = _bias(grad[i, 0], ref)
            assert got <= most


def test_fp32_sums_pass_2_to_the_24():
    """More items of one token than the GPU holds CTAs, so that no range of keys is cut to fill it."""
    _ones(450, 1, 1 << 25, 1, torch.float32)


@pytest.mark.parametrize("B,H,Hkv,prefix", [
    (300, 16, 1, False),
    (300, 16, 1, True),  # 4800 rows of the prefix
    (16, 20, 20, True),  # 16 rows of the prefix, one of each sequence
])
def test_long_sums_of_few_rows_do_not_shrink(B, H, Hkv, prefix):
    """One token over 2^23 keys, in so many items that every CTA has a whole one; with a short prefix before them, too."""
    g = torch.Generator(device="cuda").manual_seed(115)
    n, D = 1 << 23, 64
    q, k = (torch.randn(1, h, s, D, generator=g, device="cuda").to(BF16) for h, s in ((H, 1), (1, n)))
    v = torch.empty(1, 1, n, D, device="cuda", dtype=BF16).normal_(1.0, 1.0, generator=g)
    kd, vd = k[0, 0].double(), v[0, 0].double()
    q, ck, cv = q.expand(B, H, 1, D), k.expand(B, Hkv, n, D), v.expand(B, Hkv, n, D)
    if prefix:
        out = ts.shared_prefix_attention(q, ck[0, :, :7], cv[0, :, :7], ck, cv, torch.full((B,), n, device="cuda"))
        kd, vd = torch.cat((kd[:7], kd)), torch.cat((vd[:7], vd))
    else:
        out = ts.cross_attention(q, ck, cv)
    ref = torch.cat([torch.softmax(r @ kd.T * D ** -0.5, -1) @ vd for r in q[0, :, 0].double().split(4)])
    for i in (0, 1, B - 1):
        got, most = _bias(out[i, :, 0], ref)
        assert got <= most
    assert _lib.device_error() == 0
