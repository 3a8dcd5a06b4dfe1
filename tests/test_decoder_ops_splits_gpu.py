"""The work splits of the bf16 attention kernels that only calls with many items reach, against 64-bit definitions.

The forward gives every CTA whole items (a block of rows against one key head's keys) while there are enough of
them, and cuts the rest into equal runs of key tiles; the backward walks several units a CTA. 148 SMs: an item has
256 rows and 128-key tiles, or up to 16 rows and 64-key tiles on 296 CTAs; a unit of the backward 128 rows or keys.
"""

from __future__ import annotations

import threading

import pytest
import torch

import trnsparse_b200 as ts
from decoder_grad_ref import check_gradients, gradients_ref
from decoder_ref import attention_ref, check

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=BF16):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _hide(g, kind, k, v):
    """(lengths, mask, keep (B, 1, 1, Sk), k, v): a quarter of the sequences without keys, NaN where keys are hidden."""
    B, Sk = k.shape[0], k.shape[2]
    lengths = mask = None
    keep = torch.ones(B, Sk, dtype=torch.bool, device="cuda")
    if kind in ("lengths", "both"):
        lengths = torch.randint(1, Sk + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        lengths[torch.rand(B, generator=g, device="cuda") < 0.25] = 0
        lengths[0], lengths[-1] = 0, Sk
        keep &= torch.arange(Sk, device="cuda") < lengths[:, None]
    if kind in ("mask", "both"):
        mask = torch.rand(B, Sk, generator=g, device="cuda") < 0.6
        mask[:, : Sk // 2] &= torch.rand(B, 1, generator=g, device="cuda") < 0.5
        mask[1] = False
        keep &= mask
    keep = keep[:, None, None]
    if kind != "none":
        hidden = ~keep.transpose(-1, -2)
        k, v = k.masked_fill(hidden, float("nan")), v.masked_fill(hidden, float("nan"))
    return lengths, mask, keep, k, v


FORWARD = [
    # B, Hq, Hkv, Sq, Sk, D, kind                    items: whole ones a CTA, then cut ones
    (40, 8, 8, 33, 300, 128, "lengths"),    # 320: 1, 172
    (40, 16, 8, 100, 300, 64, "lengths"),   # 320 of 200 rows: 1, 172
    (80, 8, 8, 20, 200, 64, "both"),        # 640: 3, 196
    (160, 8, 8, 17, 150, 128, "lengths"),   # 1280: 7, 244 (the ring of segments is used again)
    (10, 15, 15, 20, 260, 128, "none"),     # 150: 1, 2
    (4, 26, 13, 300, 140, 64, "none"),      # 156 of three row tiles: 1, 8
    (4, 13, 13, 513, 200, 80, "mask"),      # 156: 1, 8
    (6, 26, 13, 300, 400, 128, "both"),     # 234, lengths: all cut
    (80, 8, 8, 1, 200, 64, "lengths"),      # few rows, 640: 1, 344
    (80, 16, 8, 1, 200, 128, "both"),       # few rows, 640: 1, 344
    (38, 8, 8, 1, 130, 128, "none"),        # few rows, 304: 1, 8
    (38, 32, 8, 3, 130, 64, "mask"),        # few rows (12), 304: 1, 8
    (200, 8, 8, 1, 70, 96, "lengths"),      # few rows, 1600: 4, 416
    (3, 8, 2, 1, 3000, 128, "mask"),        # few rows, 6: all cut
    (5, 4, 4, 2, 777, 64, "both"),          # few rows, 20: all cut
]


@pytest.mark.parametrize("B,Hq,Hkv,Sq,Sk,D,kind", FORWARD)
@pytest.mark.parametrize("scale", [None, -0.2])
def test_forward_of_many_items(B, Hq, Hkv, Sq, Sk, D, kind, scale):
    g = _gen(101)
    q, k, v = _randn(g, B, Sq, Hq, D).transpose(1, 2), _randn(g, B, Hkv, Sk, D), _randn(g, B, Sk, Hkv, D).transpose(1, 2)
    lengths, mask, keep, k, v = _hide(g, kind, k, v)
    ref, bound = attention_ref(q, k, v, keep, D ** -0.5 if scale is None else scale, low=True)
    first = ts.cross_attention(q, k, v, lengths, mask, scale)
    check(first, ref, bound, "out")
    assert (first[~keep.any(-1)[:, 0, 0]] == 0).all()
    assert torch.equal(first, ts.cross_attention(q, k, v, lengths, mask, scale))


BACKWARD = [
    # B, Hq, Hkv, Sq, Sk, D, kind            units of dQ x steps, units of dK and dV x steps
    (7, 16, 16, 513, 384, 128, "lengths"),  # 560 x 0-3, 336 x 0 or 5
    (20, 8, 4, 200, 500, 64, "both"),       # 320 x 0-4, 320 x 0 or 4
    (26, 6, 2, 100, 700, 80, "mask"),       # 156 x 6, 312 x 3
    (40, 8, 8, 130, 140, 128, "none"),      # 640 x 2, 640 x 2
    (50, 8, 8, 100, 120, 64, "lengths"),    # 400 x 0-1, 400 x 0-1
    (1, 4, 1, 600, 100, 128, "none"),       # columns cut in 5 parts of 4 steps
    (1, 8, 2, 700, 120, 64, "mask"),        # 2 column units, each in 6 parts
    (2, 2, 2, 1, 5000, 64, "none"),         # rows cut in 10 parts
    (2, 4, 2, 60, 3100, 128, "lengths"),    # 8 row units in 6 parts
]


@pytest.mark.parametrize("B,Hq,Hkv,Sq,Sk,D,kind", BACKWARD)
@pytest.mark.parametrize("scale", [None, -0.1])
def test_backward_of_many_units(B, Hq, Hkv, Sq, Sk, D, kind, scale):
    g = _gen(102)
    q, k, v = _randn(g, B, Hq, Sq, D), _randn(g, B, Sk, Hkv, D).transpose(1, 2), _randn(g, B, Hkv, Sk, D)
    if B > 1:
        lengths, mask, keep, k, v = _hide(g, kind, k, v)
    else:
        lengths, mask, keep = None, None, torch.ones(B, 1, 1, Sk, dtype=torch.bool, device="cuda")
        if kind == "mask":
            mask = torch.rand(B, Sk, generator=g, device="cuda") < 0.7
            keep = mask[:, None, None]
    dout = _randn(g, B, Sq, Hq, D).transpose(1, 2)
    s = D ** -0.5 if scale is None else scale
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = ts.cross_attention(*leaves, lengths, mask, scale)
    ref, bound = attention_ref(q.detach(), k.detach(), v.detach(), keep, s, low=True)
    check(out, ref, bound, "out")
    grads = torch.autograd.grad(out, leaves, dout)
    refs = gradients_ref(q.detach(), k.detach(), v.detach(), keep, s, dout, out.detach(), low=True)
    check_gradients(dict(zip(("dq", "dk", "dv"), grads)), refs)
    hidden = ~keep.transpose(-1, -2)
    for t in grads[1:]:
        assert (t.masked_select(hidden) == 0).all()
    assert (grads[0][~keep.any(-1)[:, 0, 0]] == 0).all()


@pytest.mark.parametrize("B,Hq,Hkv,T,D,P,C", [
    (5, 8, 2, 1, 128, 300, 200),    # 20 rows of the prefix, 4 of each sequence: a launch each
    (2, 4, 2, 1, 64, 200, 90),      # 4 rows a key head: both sides in the few-rows form
    (3, 2, 1, 140, 64, 256, 300),   # both in the 256-row form
    (70, 8, 4, 1, 96, 500, 70),     # 140 rows of the prefix, 2 of each sequence: a launch each
])
def test_shared_prefix_with_a_negative_scale(B, Hq, Hkv, T, D, P, C):
    g = _gen(103)
    q, pk, pv = _randn(g, B, Hq, T, D), _randn(g, Hkv, P, D), _randn(g, Hkv, P, D)
    kc, vc = _randn(g, B, Hkv, C, D), _randn(g, B, Hkv, C, D)
    lengths = torch.randint(0, C + 1, (B,), generator=g, device="cuda")
    got = ts.shared_prefix_attention(q, pk, pv, kc, vc, lengths, scale=-0.15)
    seen = lengths[:, None] - T + 1 + torch.arange(T, device="cuda")
    keep = torch.cat((torch.ones(B, 1, T, P, dtype=torch.bool, device="cuda"),
                      (torch.arange(C, device="cuda") < seen[..., None])[:, None]), -1)
    k, v = (torch.cat((a.expand(B, Hkv, P, D), b), 2) for a, b in ((pk, kc), (pv, vc)))
    check(got, *attention_ref(q, k, v, keep, -0.15, low=True), "out")


def test_calls_at_once_from_two_threads():
    """Two host threads, a stream each, the same operators on operands of their own: the bits of a call alone."""
    g = _gen(104)
    cases = []
    for D in (64, 128):
        q, k, v = _randn(g, 3, 8, 150, D), _randn(g, 3, 2, 900, D), _randn(g, 3, 2, 900, D)
        lengths = torch.tensor([900, 0, 333], device="cuda", dtype=torch.int32)
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        dout = _randn(g, 3, 8, 150, D)

        def run(leaves=leaves, lengths=lengths, dout=dout):
            q, k, v = (t.detach().requires_grad_(True) for t in leaves)
            o = ts.cross_attention(q, k, v, lengths)
            s = ts.shared_prefix_attention(q.detach()[:, :, :1], k.detach()[0], v.detach()[0], k.detach(), v.detach(), lengths)
            return (o.detach(), s, *torch.autograd.grad(o, (q, k, v), dout))

        cases.append((run, run()))
    torch.cuda.synchronize()
    bad = []

    def work(run, want):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(20):
                got = run()
                st.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    bad.append(1)

    threads = [threading.Thread(target=work, args=c) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
