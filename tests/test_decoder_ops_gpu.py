"""Decoder operators on the GPU against their 64-bit definitions, within bounds counted in half steps
(tests/decoder_ref.py), at the sizes, layouts and masks where they can go wrong."""

from __future__ import annotations

import pytest
import torch

import trnsparse_b200 as ts
from trnsparse_b200 import workloads as w
from decoder_ref import attention_ref, check, qk_ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _bshd(g, B, H, S, D, dtype):
    """(B, H, S, D) seen through a projection's (B, S, H, D) memory."""
    return _randn(g, B, S, H, D, dtype=dtype).transpose(1, 2)


# ---------------------------------------------------------------------------
# norm and rotation
# ---------------------------------------------------------------------------

QK = [
    # dtype, B, S, Hq, Hkv, D, R, interleaved, weights, positions
    (BF16, 2, 7, 4, 2, 128, 128, False, F32, "far"),
    (BF16, 2, 7, 4, 2, 128, 128, True, BF16, "batch"),
    (BF16, 1, 33, 3, 3, 64, 64, False, None, "row"),
    (BF16, 3, 5, 2, 1, 80, 40, False, F32, "row"),
    (BF16, 3, 5, 2, 1, 80, 40, True, F32, "row"),
    (BF16, 2, 3, 5, 1, 256, 256, False, BF16, "batch"),
    (BF16, 2, 3, 2, 1, 65, 32, False, F32, "row"),
    (BF16, 1, 1, 1, 1, 1, 0, False, F32, "row"),
    (BF16, 1, 1, 20, 7, 96, 96, True, None, "far"),
    (F32, 2, 9, 3, 1, 128, 64, False, F32, "far"),
    (F32, 2, 9, 3, 1, 128, 128, True, F32, "batch"),
    (F32, 1, 4, 2, 2, 250, 30, True, BF16, "row"),
    (F32, 1, 4, 2, 2, 255, 254, False, F32, "row"),
    (F32, 64, 1, 8, 8, 64, 64, False, F32, "far"),
    (F32, 1, 2000, 1, 1, 64, 64, False, F32, "row"),
    (BF16, 1, 5000, 2, 1, 128, 128, False, F32, "row"),
]


@pytest.mark.parametrize("dtype,B,S,Hq,Hkv,D,R,inter,wt,pos", QK)
def test_qk_norm_rope(dtype, B, S, Hq, Hkv, D, R, inter, wt, pos):
    g = _gen(11)
    q, k = _bshd(g, B, Hq, S, D, dtype), _randn(g, B, Hkv, S, D, dtype=dtype)
    qw, kw = ((1 + 0.3 * _randn(g, D)).to(wt) if wt is not None else None for _ in range(2))
    p = torch.arange(S, device="cuda", dtype=torch.int32)
    if pos != "row":
        top = 10_000_000 if pos == "far" else 1000
        p = torch.randint(0, top, (B, S), generator=g, device="cuda")
    freq = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / max(R, 1))
    leaves = [t.requires_grad_(True) for t in (q, k, qw, kw) if t is not None]
    yq, yk = ts.qk_norm_rope(q, k, p, freq, qw, kw, eps=1e-6, interleaved=inter)
    assert yq.is_contiguous() and yk.is_contiguous()
    dq, dk = _randn(g, B, Hq, S, D, dtype=dtype), _bshd(g, B, Hkv, S, D, dtype)
    grads = list(torch.autograd.grad((yq, yk), leaves, (dq, dk)))
    for x, wv, y, dy, i in ((q, qw, yq, dq, 0), (k, kw, yk, dk, 1)):
        ref = qk_ref(x.detach(), None if wv is None else wv.detach(), p, freq, 1e-6, inter, dy)
        check(y, ref[0], ref[1], "y")
        check(grads[i], ref[2], ref[3], "dx")
        if wv is not None:
            check(grads[2 + i], ref[4], ref[5], "dw")
    with torch.no_grad():  # the same bits without a graph
        zq, zk = ts.qk_norm_rope(q, k, p, freq, qw, kw, eps=1e-6, interleaved=inter)
    assert torch.equal(zq, yq) and torch.equal(zk, yk)


def test_qk_norm_rope_layouts_and_values():
    """Odd strides, unaligned bases, expanded inputs, zero rows, huge values, one batch row of positions."""
    g = _gen(12)
    B, S, H, D = 2, 6, 3, 64
    freq = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    pos = torch.arange(S, device="cuda")
    big = _randn(g, B, S, H, D + 3, dtype=BF16)
    views = {
        "unaligned": big[..., 3:].transpose(1, 2),
        "strided": _randn(g, B, H, S, 2 * D, dtype=BF16)[..., ::2],
        "expanded": _randn(g, 1, H, S, D, dtype=BF16).expand(B, H, S, D),
        "zeros": torch.zeros(B, H, S, D, dtype=BF16, device="cuda"),
        "large": _randn(g, B, H, S, D, dtype=BF16) * 1e15,
    }
    for name, q in views.items():
        y, _ = ts.qk_norm_rope(q, q, pos, freq)
        ref = qk_ref(q, None, pos, freq, 1e-6, False)
        check(y, ref[0], ref[1], name)
    base = _randn(g, 1, 1, S, D).requires_grad_(True)  # one head for all: its gradient is the heads' sum
    x = base.expand(B, H, S, D)
    y, z = ts.qk_norm_rope(x, x[:, :1], pos, freq)
    d, e = _randn(g, B, H, S, D), _randn(g, B, 1, S, D)
    got, = torch.autograd.grad((y, z), base, (d, e))
    r1, r2 = qk_ref(x.detach(), None, pos, freq, 1e-6, False, d), qk_ref(x.detach()[:, :1], None, pos, freq, 1e-6, False, e)
    n = B * H + B
    check(got, r1[2].sum((0, 1), True) + r2[2].sum((0, 1), True),
          (r1[3].sum((0, 1), True) + r2[3].sum((0, 1), True)) + n * 2.0 ** -24 * (r1[2].abs().sum((0, 1), True) + r2[2].abs().sum((0, 1), True)))


@pytest.mark.parametrize("B,S,Hq,Hkv", [(0, 3, 2, 1), (2, 0, 2, 1), (2, 3, 0, 1), (2, 3, 2, 0)])
def test_qk_norm_rope_empty(B, S, Hq, Hkv):
    q, k = torch.randn(B, Hq, S, 16, device="cuda"), torch.randn(B, Hkv, S, 16, device="cuda")
    wt = torch.ones(16, device="cuda", requires_grad=True)
    freq = torch.ones(8, dtype=torch.float64, device="cuda")
    q.requires_grad_(True)
    y, z = ts.qk_norm_rope(q, k, torch.arange(S, device="cuda"), freq, wt, wt)
    assert y.shape == q.shape and z.shape == k.shape
    (y.sum() + z.sum()).backward()
    assert q.grad.shape == q.shape and torch.isfinite(wt.grad).all()
    if Hq == 0 and Hkv == 0 or B * S == 0:
        assert (wt.grad == 0).all()


# ---------------------------------------------------------------------------
# cross attention
# ---------------------------------------------------------------------------

CROSS = [
    # dtype, B, Hq, Hkv, Sq, Sk, D, mask
    (BF16, 2, 4, 2, 130, 257, 128, "lengths"),
    (BF16, 2, 4, 4, 300, 128, 64, "none"),
    (BF16, 3, 2, 1, 65, 400, 128, "mask"),
    (BF16, 3, 2, 1, 65, 400, 64, "both"),
    (BF16, 1, 8, 1, 1, 1, 128, "none"),
    (BF16, 4, 8, 2, 1, 1000, 128, "lengths"),
    (BF16, 2, 2, 2, 1, 5000, 64, "none"),
    (BF16, 2, 3, 1, 17, 1, 96, "lengths"),
    (BF16, 2, 6, 3, 200, 129, 80, "lengths"),
    (BF16, 1, 2, 2, 513, 640, 72, "none"),
    (BF16, 2, 2, 1, 40, 70, 50, "lengths"),
    (BF16, 1, 2, 1, 70, 90, 256, "mask"),
    (F32, 2, 4, 2, 70, 131, 64, "both"),
    (F32, 2, 4, 1, 1, 700, 128, "lengths"),
    (F32, 1, 2, 2, 129, 65, 96, "mask"),
    (F32, 1, 3, 1, 33, 50, 33, "none"),
    (F32, 1, 2, 1, 35, 40, 200, "lengths"),
    (F32, 5, 1, 1, 2, 3, 1, "lengths"),
]


def _mask(g, B, Sk, kind, garbage, k, v):
    """(lengths, mask, keep (B, 1, 1, Sk)); hidden keys get NaN and infinities."""
    lengths = mask = None
    keep = torch.ones(B, Sk, dtype=torch.bool, device="cuda")
    if kind in ("lengths", "both"):
        lengths = torch.randint(0, Sk + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        lengths[0] = 0 if B > 1 else max(1, Sk - 3)
        lengths[-1] = Sk + 5 if B > 1 else lengths[-1]  # clamped
        keep &= torch.arange(Sk, device="cuda") < lengths[:, None]
    if kind in ("mask", "both"):
        mask = torch.rand(B, Sk, generator=g, device="cuda") < 0.6
        mask[:, : min(Sk - 1, 140)] &= torch.rand(B, 1, generator=g, device="cuda") < 0.5  # whole tiles hidden
        if B > 1:
            mask[0] = False
        else:
            mask[0, -1] = True
        keep &= mask
    keep = keep[:, None, None, :]
    if garbage:
        hidden = ~keep.transpose(-1, -2)
        k = torch.where(hidden, torch.full_like(k, float("nan")), k)
        v = torch.where(hidden, torch.full_like(v, float("inf")), v)
    return lengths, mask, keep, k, v


def _low(dtype, D):
    return dtype == BF16


@pytest.mark.parametrize("dtype,B,Hq,Hkv,Sq,Sk,D,kind", CROSS)
def test_cross_attention(dtype, B, Hq, Hkv, Sq, Sk, D, kind):
    g = _gen(21)
    q, k, v = (_bshd(g, B, h, s, D, dtype) for h, s in ((Hq, Sq), (Hkv, Sk), (Hkv, Sk)))
    lengths, mask, keep, k, v = _mask(g, B, Sk, kind, True, k, v)
    dout = _randn(g, B, Hq, Sq, D, dtype=dtype)
    scale = D ** -0.5
    ref = attention_ref(q, k, v, keep, scale, dout, low=_low(dtype, D))
    with torch.no_grad():
        out = ts.cross_attention(q, k, v, lengths, mask)
    check(out, ref[0], ref[1], "out")
    dead = ~keep.any(-1)[:, 0, 0]
    assert (out[dead] == 0).all()
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out2 = ts.cross_attention(*leaves, lengths, mask)
    check(out2, ref[0], ref[1], "out with a graph")
    for got, r, b, n in zip(torch.autograd.grad(out2, leaves, dout), ref[2::2], ref[3::2], ("dq", "dk", "dv")):
        check(got, r, b, n)
        if n != "dq":  # hidden keys: exact zeros
            assert (got.masked_select(~keep.transpose(-1, -2)) == 0).all()
        else:
            assert (got[dead] == 0).all()


def test_calls_from_fresh_host_threads():
    """A host thread that has made no CUDA call yet (autograd's worker is one) runs every operator."""
    import threading

    g = _gen(26)
    q, k, v = (_randn(g, 1, 2, s, 64, dtype=BF16) for s in (40, 150, 150))
    want = ts.cross_attention(q, k, v)
    qd = q.detach().requires_grad_(True)
    out = ts.cross_attention(qd, k, v)
    lens = torch.tensor([40], device="cuda")
    shared = ts.shared_prefix_attention(q[:, :, :1], k[0], v[0], k[:, :, :40], v[:, :, :40], lens)
    got = []

    def work():
        got.append(ts.cross_attention(q, k, v))
        got.append(ts.shared_prefix_attention(q[:, :, :1], k[0], v[0], k[:, :, :40], v[:, :, :40], lens))

    def back():
        got.append(torch.autograd.grad(out, qd, torch.ones_like(out), retain_graph=True)[0])

    for f in (work, back):
        t = threading.Thread(target=f)
        t.start()
        t.join()
    assert torch.equal(got[0], want) and torch.equal(got[1], shared)
    assert torch.equal(got[2], torch.autograd.grad(out, qd, torch.ones_like(out))[0])


def test_cross_attention_repeats_bit_for_bit():
    g = _gen(22)
    for dtype, D in ((BF16, 128), (BF16, 64), (F32, 64)):
        q = _randn(g, 2, 8, 300, D, dtype=dtype).requires_grad_(True)
        k, v = (_randn(g, 2, 2, 700, D, dtype=dtype).requires_grad_(True) for _ in range(2))
        lengths = torch.tensor([700, 333], device="cuda")
        runs = []
        for _ in range(3):
            o = ts.cross_attention(q, k, v, lengths)
            runs.append((o.detach(), *torch.autograd.grad(o, (q, k, v), torch.ones_like(o))))
        for r in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_cross_attention_scale_values_and_wanted_gradients(dtype):
    """Negative and zero scale, large scores, and gradients of a part of the operands only."""
    g = _gen(23)
    B, Hq, Hkv, Sq, Sk, D = 1, 2, 1, 50, 150, 64
    q, k, v = (_randn(g, B, h, s, D, dtype=dtype) for h, s in ((Hq, Sq), (Hkv, Sk), (Hkv, Sk)))
    keep = torch.ones(B, 1, 1, Sk, dtype=torch.bool, device="cuda")
    for scale, mul in ((-0.3, 1.0), (0.0, 1.0), (0.125, 30.0)):
        ref = attention_ref(q * mul, k, v, keep, scale, low=dtype == BF16)
        check(ts.cross_attention(q * mul, k, v, scale=scale), ref[0], ref[1], f"scale {scale}")
    dout = _randn(g, B, Hq, Sq, D, dtype=dtype)
    ref = attention_ref(q, k, v, keep, D ** -0.5, dout, low=dtype == BF16)
    for want in ((0,), (1,), (2,), (1, 2)):
        ops = [t.clone().requires_grad_(i in want) for i, t in enumerate((q, k, v))]
        o = ts.cross_attention(*ops)
        for i, got in zip(want, torch.autograd.grad(o, [ops[i] for i in want], dout)):
            check(got, ref[2 + 2 * i], ref[3 + 2 * i], f"gradient {i}")


@pytest.mark.parametrize("B,Hq,Sq,Sk", [(0, 2, 3, 4), (2, 2, 0, 4), (2, 2, 3, 0), (2, 0, 3, 4)])
def test_cross_attention_empty(B, Hq, Sq, Sk):
    for dtype in (F32, BF16):
        q = torch.randn(B, Hq, Sq, 64, device="cuda", dtype=dtype, requires_grad=True)
        k, v = (torch.randn(B, 2, Sk, 64, device="cuda", dtype=dtype, requires_grad=True) for _ in range(2))
        o = ts.cross_attention(q, k, v)
        assert o.shape == q.shape and (o == 0).all()
        gq, gk, gv = torch.autograd.grad(o, (q, k, v), torch.ones_like(o))
        assert gq.shape == q.shape and gk.shape == k.shape and gv.shape == v.shape
        assert (gq == 0).all() and (gk == 0).all() and (gv == 0).all()


def test_cross_attention_layouts():
    """Unaligned bases and strides, expanded keys (their gradient is summed), fused k/v memory, host tensors."""
    g = _gen(24)
    B, H, Sq, Sk, D = 2, 2, 33, 200, 64
    keep = torch.ones(B, 1, 1, Sk, dtype=torch.bool, device="cuda")
    for dtype in (BF16, F32):
        q = _randn(g, B, H, Sq, D + 1, dtype=dtype)[..., 1:]
        kv = _randn(g, B, Sk, 2, H, D, dtype=dtype)
        k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
        ref = attention_ref(q, k, v, keep, D ** -0.5, low=dtype == BF16)
        check(ts.cross_attention(q, k, v), ref[0], ref[1], "fused k/v")
        odd = _randn(g, B, H, Sk, D + 1, dtype=dtype)[..., 1:]
        ref = attention_ref(q, odd, v, keep, D ** -0.5, low=dtype == BF16)
        check(ts.cross_attention(q, odd, v), ref[0], ref[1], "unaligned keys")
        host = ts.cross_attention(q.cpu(), odd.cpu(), v.cpu())
        assert host.device.type == "cpu" and torch.equal(host.cuda(), ts.cross_attention(q, odd, v))
        one = _randn(g, 1, 1, Sk, D, dtype=dtype).requires_grad_(True)
        k1 = one.expand(B, H, Sk, D)
        dout = _randn(g, B, H, Sq, D, dtype=dtype).transpose(-1, -2).contiguous().transpose(-1, -2)
        ref = attention_ref(q, k1.detach(), v, keep, D ** -0.5, dout, low=dtype == BF16)
        got, = torch.autograd.grad(ts.cross_attention(q, k1, v), one, dout)
        s = lambda t: t.sum((0, 1), keepdim=True)
        r, b = s(ref[4]), s(ref[5])
        h = torch.finfo(dtype).eps / 2
        check(got, r, b + (2 * h) * (s(ref[4].abs()) + b), "expanded keys")


def test_cross_attention_long_cache_offsets():
    """Keys that start past 2^31 elements of one buffer."""
    g = _gen(25)
    D, Sk = 64, 300
    buf = torch.empty((1 << 31) + 2 * Sk * D, dtype=BF16, device="cuda")
    far = (1 << 31) + 64
    k = buf.as_strided((2, 1, Sk, D), (far, D, D, 1))
    k.copy_(_randn(g, 2, 1, Sk, D, dtype=BF16))
    v = _randn(g, 2, 1, Sk, D, dtype=BF16)
    q = _randn(g, 2, 1, 5, D, dtype=BF16)
    got, near = ts.cross_attention(q, k, v), ts.cross_attention(q, k.contiguous(), v)
    assert torch.equal(got, near)
    got = ts.shared_prefix_attention(q[:, :, :1], k[0, :, :7], v[0, :, :7], k, v, torch.tensor([Sk, 9], device="cuda"))
    near = ts.shared_prefix_attention(q[:, :, :1], k[0, :, :7].contiguous(), v[0, :, :7], k.contiguous(), v,
                                      torch.tensor([Sk, 9], device="cuda"))
    assert torch.equal(got, near)


# ---------------------------------------------------------------------------
# shared prefix
# ---------------------------------------------------------------------------

PREFIX = [
    # dtype, B, Hq, Hkv, T, D, P, capacity
    (BF16, 5, 8, 2, 1, 128, 300, 200),
    (BF16, 5, 8, 8, 1, 64, 1000, 130),
    (BF16, 70, 8, 1, 1, 128, 500, 40),
    (BF16, 3, 4, 2, 5, 96, 129, 64),
    (BF16, 2, 2, 1, 140, 64, 256, 300),
    (BF16, 1, 1, 1, 1, 64, 1, 1),
    (BF16, 3, 2, 1, 1, 128, 0, 77),
    (BF16, 3, 2, 1, 2, 128, 77, 0),
    (BF16, 2, 2, 1, 1, 50, 90, 60),
    (BF16, 2, 2, 1, 3, 256, 90, 60),
    (F32, 5, 4, 2, 1, 64, 300, 90),
    (F32, 3, 6, 2, 4, 96, 65, 20),
    (F32, 2, 1, 1, 70, 128, 10, 100),
    (F32, 2, 2, 2, 1, 201, 30, 30),
]


@pytest.mark.parametrize("dtype,B,Hq,Hkv,T,D,P,C", PREFIX)
def test_shared_prefix_attention(dtype, B, Hq, Hkv, T, D, P, C):
    g = _gen(31)
    q = _bshd(g, B, Hq, T, D, dtype)
    pk, pv = _randn(g, Hkv, P, D, dtype=dtype), _bshd(g, 1, Hkv, P, D, dtype)[0]
    cache = _randn(g, 2, B, Hkv, C + 3, D, dtype=dtype)
    lengths = torch.randint(0, C + 1, (B,), generator=g, device="cuda")
    lengths[0], lengths[-1] = min(1, C), C + 9  # clamped
    kc, vc = cache[0, :, :, :C], cache[1, :, :, :C]
    n = lengths.clamp(max=C)
    dead = (torch.arange(C, device="cuda") >= n[:, None])[:, None, :, None]
    kc.masked_fill_(dead, float("nan"))
    vc.masked_fill_(dead, float("inf"))
    got = ts.shared_prefix_attention(q, pk, pv, kc, vc, lengths)
    seen = n[:, None] - T + 1 + torch.arange(T, device="cuda")
    keep = torch.cat((torch.ones(B, 1, T, P, dtype=torch.bool, device="cuda"),
                      (torch.arange(C, device="cuda") < seen[..., None])[:, None]), -1)
    k = torch.cat((pk.expand(B, Hkv, P, D), kc), 2)
    v = torch.cat((pv.expand(B, Hkv, P, D), vc), 2)
    ref = attention_ref(q, k, v, keep, D ** -0.5, low=dtype == BF16)
    check(got, ref[0], ref[1], "out")
    # the rows behind a sequence's length stay as they were
    assert torch.isnan(kc.masked_select(dead)).all()


def test_shared_prefix_agrees_with_cross_attention():
    """The same keys as one sequence: the prefix's sharing changes no result beyond its rounding."""
    g = _gen(32)
    B, Hq, Hkv, P, C, D = 6, 8, 2, 700, 90, 128
    q = _randn(g, B, Hq, 1, D, dtype=BF16)
    pk, pv = _randn(g, Hkv, P, D, dtype=BF16), _randn(g, Hkv, P, D, dtype=BF16)
    kc, vc = _randn(g, B, Hkv, C, D, dtype=BF16), _randn(g, B, Hkv, C, D, dtype=BF16)
    lengths = torch.tensor([0, 1, 17, 64, 89, 90], device="cuda", dtype=torch.int32)
    got = ts.shared_prefix_attention(q, pk, pv, kc, vc, lengths)
    k, v = (torch.cat((a.expand(B, Hkv, P, D), b), 2) for a, b in ((pk, kc), (pv, vc)))
    one = ts.cross_attention(q, k, v, key_lengths=lengths + P)
    keep = (torch.arange(P + C, device="cuda") < (lengths + P)[:, None])[:, None, None]
    bound = attention_ref(q, k, v, keep, D ** -0.5, low=True)[1]
    check(got, one.double(), 2 * bound, "shared against joined")


def test_shared_prefix_empty():
    z = lambda *s: torch.zeros(*s, device="cuda", dtype=BF16)
    for B, T in ((0, 1), (2, 0)):
        o = ts.shared_prefix_attention(z(B, 2, T, 64), z(1, 3, 64), z(1, 3, 64), z(B, 1, 4, 64), z(B, 1, 4, 64),
                                       torch.ones(B, dtype=torch.int32, device="cuda"))
        assert o.shape == (B, 2, T, 64)
    o = ts.shared_prefix_attention(z(2, 2, 1, 64) + 1, z(1, 0, 64), z(1, 0, 64), z(2, 1, 4, 64) + 1, z(2, 1, 4, 64) + 1,
                                   torch.tensor([0, 2], device="cuda"))
    assert (o[0] == 0).all() and (o[1] == 1).all()


# ---------------------------------------------------------------------------
# gradients against differences, streams, graphs, and the operators together
# ---------------------------------------------------------------------------


def _difference(f, xs, grads, g, steps=2.0 ** -7):
    """The change of f along a random direction, in fp32, against the gradients' product with it."""
    ds = [_randn(g, *x.shape) for x in xs]
    with torch.no_grad():
        up, down = (f(*[x + s * steps * d for x, d in zip(xs, ds)]) for s in (1, -1))
    want = sum((a.double() * d.double()).sum() for a, d in zip(grads, ds)).item()
    return ((up - down) / (2 * steps)).item(), want, sum(a.double().norm().item() for a in grads)


def test_gradients_against_differences():
    """Central differences with step h = 2^-7 along unit-variance directions: off by h^2 times the third
    derivative (of the order of the gradient's norm for these smooth functions) plus rounding / h."""
    g = _gen(41)
    D = 32
    freq = 100.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    pos = torch.arange(7, device="cuda")
    a, b = _randn(g, 1, 2, 7, D), _randn(g, 1, 1, 7, D)
    xs = [_randn(g, 1, 2, 7, D), _randn(g, 1, 1, 7, D), 1 + 0.1 * _randn(g, D), 1 + 0.1 * _randn(g, D)]

    def f(q, k, qw, kw):
        y, z = ts.qk_norm_rope(q, k, pos, freq, qw, kw)
        return (y.double() * a.double()).sum() + (z.double() * b.double()).sum()

    leaves = [x.clone().requires_grad_(True) for x in xs]
    got, want, size = _difference(f, xs, torch.autograd.grad(f(*leaves), leaves), g)
    assert abs(got - want) <= 1e-3 * size
    c = _randn(g, 2, 2, 9, D)
    xs = [_randn(g, 2, 2, 9, D), _randn(g, 2, 1, 20, D), _randn(g, 2, 1, 20, D)]
    lengths = torch.tensor([20, 7], device="cuda")
    f = lambda q, k, v: (ts.cross_attention(q, k, v, lengths).double() * c.double()).sum()
    leaves = [x.clone().requires_grad_(True) for x in xs]
    got, want, size = _difference(f, xs, torch.autograd.grad(f(*leaves), leaves), g)
    assert abs(got - want) <= 1e-3 * size


def _step(g, B=4, H=4, Hkv=2, D=64, P=300, C=100, Sk=200):
    """A decoder layer's attention part for one token: norm and rotation, own attention over a shared prefix,
    cross attention to encoder states."""
    freq = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    st = dict(x=_randn(g, B, H, 1, D, dtype=BF16), y=_randn(g, B, Hkv, 1, D, dtype=BF16),
              pk=_randn(g, Hkv, P, D, dtype=BF16), pv=_randn(g, Hkv, P, D, dtype=BF16),
              kc=_randn(g, B, Hkv, C, D, dtype=BF16), vc=_randn(g, B, Hkv, C, D, dtype=BF16),
              ek=_randn(g, B, Hkv, Sk, D, dtype=BF16), ev=_randn(g, B, Hkv, Sk, D, dtype=BF16),
              own=torch.tensor([3, 50, 99, 100][:B], device="cuda", dtype=torch.int32),
              enc=torch.tensor([200, 0, 1, 129][:B], device="cuda", dtype=torch.int32))

    def run():
        at = st["own"].long() - 1
        q, k = ts.qk_norm_rope(st["x"], st["y"], (P + at)[:, None], freq)
        st["kc"][torch.arange(B, device="cuda"), :, at] = k[:, :, 0]
        a = ts.shared_prefix_attention(q, st["pk"], st["pv"], st["kc"], st["vc"], st["own"])
        return a, ts.cross_attention(a, st["ek"], st["ev"], st["enc"])

    return st, run


def test_decoder_step_in_a_graph_and_on_streams():
    g = _gen(42)
    st, run = _step(g)
    want = [t.clone() for t in run()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    pool = torch.cuda.graph_pool_handle()
    for _ in range(2):  # two graphs of one memory pool
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, pool=pool):
            out = run()
        graphs.append((gr, out))
    for gr, out in graphs:
        gr.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    st["x"].copy_(_randn(g, *st["x"].shape, dtype=BF16))
    st["own"].copy_(torch.tensor([100, 7, 1, 64], device="cuda"))
    fresh = [t.clone() for t in run()]
    assert not torch.equal(fresh[0], want[0])
    for gr, out in graphs:
        gr.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, fresh))


def test_training_run_together_and_captured():
    """norm + rotation -> block-sparse attention -> cross attention, forward and backward; the same bits when
    captured while an eager graph of the same leaves lives. torch ties a leaf's gradient node to the stream its
    first graph ran on, so that graph has to be made on the stream of the capture."""
    g = _gen(43)
    B, H, S, Sk, D = 1, 2, 256, 300, 64
    freq = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    pos = torch.arange(S, device="cuda")
    mask = w.sliding_window_mask(seq=S, window=1, n_global=1)
    x, y, v = (_bshd(g, B, H, S, D, BF16).requires_grad_(True) for _ in range(3))
    ek, ev = (_bshd(g, B, H, Sk, D, BF16).requires_grad_(True) for _ in range(2))
    wq, wk = (torch.ones(D, device="cuda", requires_grad=True) for _ in range(2))
    leaves = [x, y, v, ek, ev, wq, wk]
    d = _randn(g, B, H, S, D, dtype=BF16)

    def run():
        q, k = ts.qk_norm_rope(x, y, pos, freq, wq, wk)
        a = ts.block_sparse_attention_tiled(q, k, v, mask)
        o = ts.cross_attention(a, ek, ev)
        return o, torch.autograd.grad(o, leaves, d, retain_graph=True)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
        eager, want = run()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.isfinite(t).all() for t in want) and all(t.abs().sum() > 0 for t in want)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=s):
        o, got = run()
    gr.replay()
    assert torch.equal(o, eager)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    again = torch.autograd.grad(eager, leaves, d)  # the eager graph still works
    assert all(torch.equal(a, b) for a, b in zip(again, want))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_lengths_of_64_bits_are_clamped_before_they_are_narrowed(dtype):
    """2^40 and 2^32 have zero low words, -2^40 + 5 a positive one."""
    g = _gen(91)
    B, Hq, Hkv, T, S, D = 4, 4, 2, 3, 70, 64
    wide = torch.tensor([2**40, 2**32, -(2**40) + 5, 33], device="cuda")
    narrow = torch.tensor([S, S, 0, 33], dtype=torch.int32, device="cuda")
    q = _randn(g, B, Hq, T, D, dtype=dtype)
    k, v = (_randn(g, B, Hkv, S, D, dtype=dtype) for _ in range(2))
    pk, pv = (_randn(g, Hkv, 9, D, dtype=dtype) for _ in range(2))
    assert torch.equal(ts.cross_attention(q, k, v, wide), ts.cross_attention(q, k, v, narrow))
    got = ts.shared_prefix_attention(q, pk, pv, k, v, wide)
    assert torch.equal(got, ts.shared_prefix_attention(q, pk, pv, k, v, narrow))
    assert ts.cross_attention(q, k, v, wide)[2].eq(0).all() and ts.cross_attention(q, k, v, wide)[0].ne(0).any()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_walks_without_steps_leave_zero_gradients(D):
    """Sequences without keys, and lengths that end before a range of the walk begins, in fp32."""
    g = _gen(92)
    B, Hq, Hkv, T, S = 16, 4, 2, 130, 1500
    lengths = torch.tensor([0, 1, 0, 40, S, 0, 0, 64] * 2, dtype=torch.int32, device="cuda")
    q, k, v = (_randn(g, B, h, n, D).requires_grad_() for h, n in ((Hq, T), (Hkv, S), (Hkv, S)))
    dout = _randn(g, B, Hq, T, D)
    for _ in range(3):
        dq, dk, dv = torch.autograd.grad(ts.cross_attention(q, k, v, lengths), (q, k, v), dout)
        for b, n in enumerate(lengths.tolist()):
            assert dk[b, :, n:].eq(0).all() and dv[b, :, n:].eq(0).all()
            assert n > 0 or dq[b].eq(0).all()
            assert n == 0 or dv[b, :, :n].ne(0).any()


@pytest.mark.parametrize("dtype,B,Hq,Hkv,Sq,Sk,D,kind", [
    (F32, 3, 8, 2, 100, 700, 64, "both"),      # several ranges of keys and of rows
    (F32, 1, 4, 4, 257, 33, 128, "mask"),      # one row past two tiles, one key past a tile
    (F32, 2, 2, 1, 600, 1300, 48, "lengths"),
    (F32, 1, 2, 2, 300, 500, 256, "both"),
    (F32, 2, 4, 1, 8, 900, 64, "lengths"),     # 32 packed rows: the last of the few-rows form
    (F32, 2, 4, 1, 9, 900, 96, "mask"),        # 36: the first of the other
    (F32, 1, 1, 1, 128, 128, 65, "none"),      # rows that do not start on 16 bytes
    (F32, 1, 1, 1, 64, 6000, 64, "none"),      # long sums
    (BF16, 1, 2, 1, 150, 200, 200, "lengths"),
    (BF16, 2, 2, 1, 70, 300, 36, "both"),
])
def test_cross_attention_at_the_tiles_of_the_split_products(dtype, B, Hq, Hkv, Sq, Sk, D, kind):
    test_cross_attention(dtype, B, Hq, Hkv, Sq, Sk, D, kind)
