"""Workloads of the decoder operators: query/key norm with rotation, cross attention, shared-prefix attention.

``own`` false: the operators in elementary 32-bit torch operations. ``own`` true: the calls a user of
``trnsparse_b200`` makes. Cases are plain dicts; see ``listed`` for what each stands for.
"""

from __future__ import annotations

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one decoding step of a batch: latency of a small call
        {"name": "qk_step_bf16", "op": "qk", "dtype": "bf16", "B": 48, "S": 1, "Hq": 32, "Hkv": 8, "D": 128, "R": 128,
         "inter": False, "train": False, "far": 131072, "wt": "bf16"},
        # a small fp32 training run: odd length, part of the head rotated, adjacent pairs
        {"name": "qk_train_f32", "op": "qk", "dtype": "f32", "B": 3, "S": 1021, "Hq": 12, "Hkv": 4, "D": 80, "R": 40,
         "inter": True, "train": True, "far": 0, "wt": "f32"},
        # what feeds the block-sparse attention benchmark (16 heads, 16384 tokens, 128 wide), in training
        {"name": "qk_train_bf16", "op": "qk", "dtype": "bf16", "B": 1, "S": 16384, "Hq": 16, "Hkv": 16, "D": 128,
         "R": 128, "inter": False, "train": True, "far": 0, "wt": "f32"},
        # one decoding step over encoder states of 30 s of speech
        {"name": "cross_step_bf16", "op": "cross", "dtype": "bf16", "B": 32, "Hq": 16, "Hkv": 16, "Sq": 1, "Sk": 1500,
         "D": 64, "mask": "none", "train": False, "garbage": False},
        # one decoding step over long documents of unequal lengths, shared key heads
        {"name": "cross_step_long", "op": "cross", "dtype": "bf16", "B": 8, "Hq": 32, "Hkv": 8, "Sq": 1, "Sk": 8192,
         "D": 128, "mask": "lengths", "train": False, "garbage": True},
        # a padded batch of prompts: odd sizes, one sequence without any key
        {"name": "cross_prompt_bf16", "op": "cross", "dtype": "bf16", "B": 4, "Hq": 32, "Hkv": 8, "Sq": 777,
         "Sk": 2049, "D": 128, "mask": "lengths", "train": False, "garbage": True},
        # training, full sequences
        {"name": "cross_train_bf16", "op": "cross", "dtype": "bf16", "B": 4, "Hq": 16, "Hkv": 16, "Sq": 2048,
         "Sk": 4096, "D": 128, "mask": "none", "train": True, "garbage": False},
        # a small fp32 training run with holes in the key mask
        {"name": "cross_train_f32", "op": "cross", "dtype": "f32", "B": 2, "Hq": 8, "Hkv": 2, "Sq": 333, "Sk": 517,
         "D": 64, "mask": "mask", "train": True, "garbage": True},
        # a few sequences with a short common prompt: latency
        {"name": "prefix_step_small", "op": "prefix", "dtype": "bf16", "B": 4, "Hq": 8, "Hkv": 2, "T": 1, "D": 64,
         "P": 640, "C": 128, "garbage": True},
        # an ordinary serving step: a system prompt shared by 64 sequences
        {"name": "prefix_step_bf16", "op": "prefix", "dtype": "bf16", "B": 64, "Hq": 32, "Hkv": 8, "T": 1, "D": 128,
         "P": 8192, "C": 1024, "garbage": True},
        # fp32, several tokens at once (drafted tokens to be checked), odd sizes
        {"name": "prefix_chunk_f32", "op": "prefix", "dtype": "f32", "B": 7, "Hq": 12, "Hkv": 4, "T": 5, "D": 96,
         "P": 1001, "C": 333, "garbage": True},
        # the largest: a long document shared by 96 sequences
        {"name": "prefix_step_long", "op": "prefix", "dtype": "bf16", "B": 96, "Hq": 32, "Hkv": 8, "T": 1, "D": 128,
         "P": 32768, "C": 2048, "garbage": True},
    ]


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    hkv = rng.choice([1, 2, 3, 4, 8, 16])
    return hkv * rng.choice([g for g in (1, 2, 3, 4, 8) if g * hkv <= 32]), hkv


def _draw(rng):
    op = rng.choice(["qk", "cross", "prefix"])
    hq, hkv = _heads(rng)
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if op == "qk":
        d = rng.choice([64, 80, 96, 128, 192, 256])
        r = rng.choice([d, d, d // 2])
        s = rng.choice([1, _spread(rng, 2, 16384)])
        return {"op": op, "dtype": dtype, "B": _spread(rng, 1, 64), "S": s, "Hq": hq, "Hkv": hkv, "D": d,
                "R": r, "inter": rng.random() < 0.3, "train": s > 1 and rng.random() < 0.6,
                "far": rng.choice([0, 4096, 131072, 1000000]), "wt": rng.choice(["f32", "bf16", "none"])}
    d = rng.choice([64, 64, 80, 96, 128, 128, 128])
    if op == "cross":
        sq = rng.choice([1, _spread(rng, 2, 4096)])
        mask = rng.choice(["none", "lengths", "lengths", "mask"])
        train = sq > 1 and rng.random() < 0.5
        sk = _spread(rng, 16 if train else 1, 8192)  # over one key, dQ and dK are zero but for rounding
        return {"op": op, "dtype": dtype, "B": _spread(rng, 1, 32), "Hq": hq, "Hkv": hkv, "Sq": sq, "Sk": sk, "D": d,
                "mask": mask, "train": train, "garbage": mask != "none"}
    return {"op": op, "dtype": dtype, "B": _spread(rng, 1, 96), "Hq": hq, "Hkv": hkv,
            "T": rng.choice([1, 1, 1, rng.randint(2, 8)]), "D": d, "P": _spread(rng, 1, 32768),
            "C": _spread(rng, 8, 2048), "garbage": True}


def _cost(case):
    w = work(case)
    # the plain forms compute in 32 bits: about 50 TFLOP/s and 6 TB/s
    return w["flops"] / 50e12 + w["bytes"] / 6e12


def draw(rng):
    caps = {}
    for c in listed():
        key = (c["op"], c["dtype"] == "f32" and c["op"] == "cross")
        caps[key] = max(caps.get(key, 0.0), _cost(c))
    caps[("cross", True)] *= 16  # fp32 training is real up to here; still far below the largest listed case
    while True:
        c = _draw(rng)
        key = (c["op"], c["dtype"] == "f32" and c["op"] == "cross")
        if _cost(c) <= caps[key]:
            return c


def _kept(case):
    """Keys of each sequence, a fixed multiset (its order comes from the seed)."""
    B, Sk = case["B"], case["Sk"]
    if case["mask"] == "none":
        return [Sk] * B
    if B == 1:
        return [max(1, (3 * Sk) // 4)]
    return [round(Sk * i / (B - 1)) for i in range(B)] if B > 2 else [0, Sk]


def _suffix(case):
    """Own keys of each sequence, the new tokens included."""
    B, C, T = case["B"], case["C"], case["T"]
    lo = min(T, C)
    if B == 1:
        return [(lo + C) // 2]
    return [lo + round((C - lo) * i / (B - 1)) for i in range(B)]


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    D = case["D"]
    if case["op"] == "qk":
        n = case["B"] * case["S"] * (case["Hq"] + case["Hkv"]) * D
        passes = 2 + (3 if case["train"] else 0)  # x in, y out; x, dy in, dx out
        return {"bytes": n * es * passes + case["B"] * case["S"] * 8, "flops": n * (10 + (20 if case["train"] else 0))}
    if case["op"] == "cross":
        keys = sum(_kept(case))
        rows = case["B"] * case["Hq"] * case["Sq"]
        q, kv = rows * D * es, keys * case["Hkv"] * D * es
        pairs = keys * case["Hq"] * case["Sq"]
        if not case["train"]:
            return {"bytes": 2 * q + 2 * kv, "flops": 4 * D * pairs}
        full = case["B"] * case["Hkv"] * case["Sk"] * D * es  # dK, dV are whole
        return {"bytes": (2 * q + 2 * kv) + (4 * q + 2 * kv + 2 * full), "flops": 14 * D * pairs}
    T, rows = case["T"], case["B"] * case["Hq"] * case["T"]
    suf = _suffix(case)
    kv = (case["P"] + sum(suf)) * case["Hkv"] * D * es
    own_pairs = sum(max(0, n - T + 1 + t) for n in suf for t in range(T))
    pairs = rows * case["P"] + case["Hq"] * own_pairs
    return {"bytes": 2 * rows * D * es + 2 * kv, "flops": 4 * D * pairs}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _DT[case["dtype"]]
    D = case["D"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev).to(dt)

    def order(values):
        t = torch.tensor(values, device=dev)
        return t[torch.randperm(len(values), generator=g, device=dev)]

    st = {"case": case}
    if case["op"] == "qk":
        B, S, Hq, Hkv, R = case["B"], case["S"], case["Hq"], case["Hkv"], case["R"]
        # the projections' outputs, (batch, token, head, D), seen as (batch, head, token, D)
        st["q"] = normal(B, S, Hq, D).transpose(1, 2)
        st["k"] = normal(B, S, Hkv, D).transpose(1, 2)
        if case["far"]:
            start = torch.randint(0, case["far"], (B, 1), generator=g, device=dev)
            st["pos"] = start + torch.arange(S, device=dev)
        else:
            st["pos"] = torch.arange(S, device=dev)
        st["freq"] = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device=dev) / R)
        st["qw"] = st["kw"] = None
        if case["wt"] != "none":
            st["qw"], st["kw"] = ((1 + 0.2 * torch.randn(D, generator=g, device=dev)).to(_DT[case["wt"]])
                                  for _ in range(2))
        if case["train"]:
            st["dq"], st["dk"] = normal(B, Hq, S, D), normal(B, Hkv, S, D)
            st["leaves"] = [t.requires_grad_(True) for t in (st["q"], st["k"], st["qw"], st["kw"]) if t is not None]
        return st
    if case["op"] == "cross":
        B, Hq, Hkv, Sq, Sk = case["B"], case["Hq"], case["Hkv"], case["Sq"], case["Sk"]
        st["q"] = normal(B, Sq, Hq, D).transpose(1, 2)
        st["k"] = normal(B, Sk, Hkv, D).transpose(1, 2)
        st["v"] = normal(B, Sk, Hkv, D).transpose(1, 2)
        st["lengths"] = st["mask"] = None
        keep = None
        if case["mask"] == "lengths":
            st["lengths"] = order(_kept(case)).to(torch.int32)
            keep = torch.arange(Sk, device=dev)[None, :] < st["lengths"][:, None]
        elif case["mask"] == "mask":
            n = order(_kept(case))
            rank = torch.rand(B, Sk, generator=g, device=dev).argsort(1).argsort(1)
            st["mask"] = keep = rank < n[:, None]
        if case["garbage"] and keep is not None:  # padding is whatever the buffer held
            bad = ~keep[:, None, :, None]
            st["k"] = st["k"].masked_fill(bad, float("nan"))
            st["v"] = st["v"].masked_fill(bad, float("nan"))
        if case["train"]:
            st["do"] = normal(B, Hq, Sq, D)
            for n in ("q", "k", "v"):
                st[n].requires_grad_(True)
        return st
    B, Hq, Hkv, T, P, C = case["B"], case["Hq"], case["Hkv"], case["T"], case["P"], case["C"]
    st["q"] = normal(B, Hq, T, D)
    st["pk"], st["pv"] = normal(Hkv, P, D), normal(Hkv, P, D)
    st["kc"], st["vc"] = normal(B, Hkv, C, D), normal(B, Hkv, C, D)
    st["lengths"] = order(_suffix(case)).to(torch.int32)
    if case["garbage"]:
        bad = (torch.arange(C, device=dev)[None, :] >= st["lengths"][:, None])[:, None, :, None]
        st["kc"] = st["kc"].masked_fill(bad, float("nan"))
        st["vc"] = st["vc"].masked_fill(bad, float("nan"))
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(state):
    case = state["case"]
    return (_own if own else _plain)[case["op"]](state)


def _own_qk(st):
    import trnsparse_b200 as ts

    yq, yk = ts.qk_norm_rope(st["q"], st["k"], st["pos"], st["freq"], st["qw"], st["kw"], eps=1e-6,
                             interleaved=st["case"]["inter"])
    if not st["case"]["train"]:
        return yq, yk
    grads = torch.autograd.grad((yq, yk), st["leaves"], (st["dq"], st["dk"]))
    return (yq.detach(), yk.detach(), *grads)


def _own_cross(st):
    import trnsparse_b200 as ts

    o = ts.cross_attention(st["q"], st["k"], st["v"], key_lengths=st["lengths"], key_mask=st["mask"])
    if not st["case"]["train"]:
        return o
    return (o.detach(), *torch.autograd.grad(o, (st["q"], st["k"], st["v"]), st["do"]))


def _own_prefix(st):
    import trnsparse_b200 as ts

    return ts.shared_prefix_attention(st["q"], st["pk"], st["pv"], st["kc"], st["vc"], st["lengths"])


_own = {"qk": _own_qk, "cross": _own_cross, "prefix": _own_prefix}


def _rotate(x, cos, sin, R, inter, back=False):
    """The pairs of the first R elements turned by their angles (the other way for ``back``)."""
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if inter else (x[..., : R // 2], x[..., R // 2: R])
    s = -sin if back else sin
    ya, yb = a * cos - b * s, b * cos + a * s
    y = torch.stack((ya, yb), -1).flatten(-2) if inter else torch.cat((ya, yb), -1)
    return torch.cat((y, x[..., R:]), -1)


@torch.no_grad()
def _plain_qk(st):
    case = st["case"]
    R, inter, dt = case["R"], case["inter"], _DT[case["dtype"]]
    ang = st["pos"].double()[..., None] * st["freq"]
    ang = ang if ang.dim() == 2 else ang[:, None]
    cos, sin = torch.cos(ang).float(), torch.sin(ang).float()
    outs, dxs, dws = [], [], []
    for x0, w0, dy in ((st["q"], st["qw"], st.get("dq")), (st["k"], st["kw"], st.get("dk"))):
        x = x0.float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        xh = x * r
        n = xh if w0 is None else xh * w0.float()
        outs.append(_rotate(n, cos, sin, R, inter).to(dt).contiguous())
        if dy is None:
            continue
        dn = _rotate(dy.float(), cos, sin, R, inter, back=True)
        if w0 is not None:
            dws.append((dn * xh).sum((0, 1, 2)).to(w0.dtype))
            dn = dn * w0.float()
        dxs.append((r * (dn - xh * (dn * xh).mean(-1, keepdim=True))).to(dt))
    return tuple(outs + dxs + dws)


@torch.no_grad()
def _plain_cross(st):
    case = st["case"]
    dt, train = _DT[case["dtype"]], case["train"]
    B, Hq, Hkv, Sq, Sk, D = (case[n] for n in ("B", "Hq", "Hkv", "Sq", "Sk", "D"))
    G, scale = Hq // Hkv, D ** -0.5
    out = torch.empty(B, Hq, Sq, D, dtype=dt, device=st["q"].device)
    dq, dk, dv = torch.empty_like(out), *(torch.empty(B, Hkv, Sk, D, dtype=dt, device=out.device) for _ in range(2))
    keep = st["mask"]
    if st["lengths"] is not None:
        keep = torch.arange(Sk, device=out.device)[None, :] < st["lengths"][:, None]
    # as many sequences at a time as keep the scores within 4 GB
    step = max(1, min(B, (1 << 30) // max(1, Hq * Sq * Sk)))
    for b in range(0, B, step):
        e = min(B, b + step)
        q = st["q"][b:e].float().reshape(e - b, Hkv, G * Sq, D)
        k, v = st["k"][b:e].float(), st["v"][b:e].float()
        s = None
        if keep is not None:
            m = keep[b:e, None, :, None]
            k, v = k.masked_fill(~m, 0.0), v.masked_fill(~m, 0.0)
            row = keep[b:e, None, None, :]
            s = (q @ k.transpose(-1, -2) * scale).masked_fill(~row, float("-inf"))
        else:
            s = q @ k.transpose(-1, -2) * scale
        mx = s.amax(-1, keepdim=True)
        p = torch.exp(s - mx.masked_fill(mx == float("-inf"), 0.0))
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
        o = p @ v
        out[b:e] = o.view(e - b, Hq, Sq, D).to(dt)
        if train:
            do = st["do"][b:e].float().reshape(e - b, Hkv, G * Sq, D)
            dv[b:e] = (p.transpose(-1, -2) @ do).to(dt)
            ds = p * (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True)) * scale
            dq[b:e] = (ds @ k).view(e - b, Hq, Sq, D).to(dt)
            dk[b:e] = (ds.transpose(-1, -2) @ q).to(dt)
    return (out, dq, dk, dv) if train else out


@torch.no_grad()
def _plain_prefix(st):
    case = st["case"]
    B, Hq, Hkv, T, P, C, D = (case[n] for n in ("B", "Hq", "Hkv", "T", "P", "C", "D"))
    G, scale = Hq // Hkv, D ** -0.5
    dev = st["q"].device
    q = st["q"].float().view(B, Hkv, G * T, D)
    seen = st["lengths"][:, None] - T + 1 + torch.arange(T, device=dev)  # (B, T)
    live = (torch.arange(C, device=dev) < st["lengths"][:, None])[:, None, :, None]
    kc, vc = st["kc"].float().masked_fill(~live, 0.0), st["vc"].float().masked_fill(~live, 0.0)
    # the prefix once for the whole batch
    qp = q.transpose(0, 1).reshape(Hkv, B * G * T, D)
    sp = (qp @ st["pk"].float().transpose(-1, -2) * scale).reshape(Hkv, B, G * T, P).transpose(0, 1)
    so = q @ kc.transpose(-1, -2) * scale
    ok = (torch.arange(C, device=dev) < seen[..., None])[:, None, None].expand(B, Hkv, G, T, C).reshape(so.shape)
    so = so.masked_fill(~ok, float("-inf"))
    m = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    pp, po = torch.exp(sp - m), torch.exp(so - m)
    den = pp.sum(-1, keepdim=True) + po.sum(-1, keepdim=True)
    op = (pp.transpose(0, 1).reshape(Hkv, B * G * T, P) @ st["pv"].float()).reshape(Hkv, B, G * T, D).transpose(0, 1)
    return ((op + po @ vc) / den).reshape(B, Hq, T, D).to(_DT[case["dtype"]])


_plain = {"qk": _plain_qk, "cross": _plain_cross, "prefix": _plain_prefix}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


@torch.no_grad()
def exact(case, seed):
    st = prepare(case, seed)
    return {"qk": _exact_qk, "cross": _exact_cross, "prefix": _exact_prefix}[case["op"]](case, st)


def _exact_qk(case, st):
    D, R = case["D"], case["R"]
    dev = st["q"].device
    lo = torch.arange(R // 2, device=dev)
    a, b = (2 * lo, 2 * lo + 1) if case["inter"] else (lo, lo + R // 2)
    pos = st["pos"].double()
    pos = pos.expand(case["B"], case["S"]) if pos.dim() == 1 else pos
    res = {"y": [], "dx": [], "dw": []}
    for name in ("q", "k"):
        x, w, dy = st[name].detach(), st[name + "w"], st.get("d" + name)
        w64 = torch.ones(D, dtype=torch.float64, device=dev) if w is None else w.detach().double()
        y = torch.empty(x.shape, dtype=torch.float64, device=dev)
        dx = torch.empty_like(y)
        dw = torch.zeros(D, dtype=torch.float64, device=dev)
        for h in range(x.shape[1]):
            xs = x[:, h].double()
            inv = 1.0 / torch.sqrt(xs.square().mean(-1, keepdim=True) + 1e-6)
            n = xs * inv * w64
            z = torch.complex(n[..., a], n[..., b])
            turn = torch.polar(torch.ones_like(z.real), pos[..., None] * st["freq"])
            z2 = z * turn
            out = n.clone()
            out[..., a], out[..., b] = z2.real, z2.imag
            y[:, h] = out
            if dy is not None:
                d = dy[:, h].double()
                gz = torch.complex(d[..., a], d[..., b]) * turn.conj()
                d[..., a], d[..., b] = gz.real, gz.imag
                u = xs * inv
                dw += (d * u).flatten(0, 1).sum(0)
                d = d * w64
                dx[:, h] = inv * (d - u * (d * u).mean(-1, keepdim=True))
        res["y"].append(y)
        if dy is not None:
            res["dx"].append(dx)
            if w is not None:
                res["dw"].append(dw)
    return tuple(res["y"] + res["dx"] + res["dw"])


def _exact_cross(case, st):
    B, Hq, Hkv, Sq, Sk, D = (case[n] for n in ("B", "Hq", "Hkv", "Sq", "Sk", "D"))
    if 14.0 * D * B * Hq * Sq * Sk > 4e13:
        return None
    dev, G = st["q"].device, Hq // Hkv
    z = lambda h, s: torch.zeros(B, h, s, D, dtype=torch.float64, device=dev)
    o, dq, dk, dv = z(Hq, Sq), z(Hq, Sq), z(Hkv, Sk), z(Hkv, Sk)
    for b in range(B):
        idx = torch.arange(Sk, device=dev)
        if st["lengths"] is not None:
            idx = idx[: int(st["lengths"][b])]
        if st["mask"] is not None:
            idx = st["mask"][b].nonzero()[:, 0]
        if idx.numel() == 0:
            continue
        for h in range(Hq):
            q = st["q"][b, h].detach().double()
            k = st["k"][b, h // G].detach()[idx].double()
            v = st["v"][b, h // G].detach()[idx].double()
            p = torch.softmax(torch.einsum("sd,td->st", q, k) / math.sqrt(D), -1)
            o[b, h] = torch.einsum("st,td->sd", p, v)
            if case["train"]:
                do = st["do"][b, h].double()
                dv[b, h // G].index_add_(0, idx, torch.einsum("st,sd->td", p, do))
                dp = torch.einsum("sd,td->st", do, v)
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(D)
                dq[b, h] = torch.einsum("st,td->sd", ds, k)
                dk[b, h // G].index_add_(0, idx, torch.einsum("st,sd->td", ds, q))
    return (o, dq, dk, dv) if case["train"] else o


def _exact_prefix(case, st):
    B, Hq, Hkv, T, P, D = (case[n] for n in ("B", "Hq", "Hkv", "T", "P", "D"))
    G = Hq // Hkv
    out = torch.zeros(B, Hq, T, D, dtype=torch.float64, device=st["q"].device)
    for h in range(Hkv):
        pk, pv = st["pk"][h].double(), st["pv"][h].double()
        for b in range(B):
            n = int(st["lengths"][b])
            k = torch.cat((pk, st["kc"][b, h, :n].double()))
            v = torch.cat((pv, st["vc"][b, h, :n].double()))
            for t in range(T):
                m = P + max(0, n - T + 1 + t)
                s = st["q"][b, h * G:(h + 1) * G, t].double() @ k[:m].T / math.sqrt(D)
                out[b, h * G:(h + 1) * G, t] = torch.softmax(s, -1) @ v[:m]
    return out
