"""Decoder operators that stand beside ``block_sparse_attention_tiled``.

``qk_norm_rope`` makes its queries and keys (norm of every head and position
rotation in one pass), ``cross_attention`` attends another sequence, and
``shared_prefix_attention`` decodes a batch over a prompt it shares. The
reference has no counterpart of them. As with the other operators, tensors
may live on the host or on the GPU (host inputs are copied to the current
CUDA device and the result is copied back), work is queued on the current
stream of the operands' device without a synchronisation, and workspaces
come from torch's allocator. There is no CPU compute path.
"""

from __future__ import annotations

import ctypes as C

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _back, _dev_of

_DTYPES = (torch.float32, torch.bfloat16)


def _on_device(dev: torch.device, run) -> None:
    """``run(stream handle)`` with ``dev`` as the current device."""
    if dev.index == torch.cuda.current_device():
        run(torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            run(torch._C._cuda_getCurrentRawStream(dev.index))


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with unit stride along its last dimension (as it is, if it has it)."""
    return t if t.stride(-1) == 1 else t.contiguous()


def _tiles(t: torch.Tensor) -> torch.Tensor:
    """``t`` as the attention kernels load it fastest: unit last stride, and where head_dim allows it rows that
    start on 16 bytes (an operand that does not have them is copied once, which costs less than narrow loads)."""
    *outer, last = t.stride()
    n = 16 // t.element_size()
    if last == 1:
        if t.shape[-1] % n:
            return t
        bits = 0
        for size, stride in zip(t.shape, outer):
            if size > 1:
                bits |= stride
        if bits % n == 0 and bits >= 0 and (outer[-1] or t.shape[-2] <= 1):
            return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)
    return t.contiguous()


def _to(t: torch.Tensor | None, dev: torch.device, dtype: torch.dtype | None = None) -> torch.Tensor | None:
    if t is None or (t.device == dev and (dtype is None or t.dtype == dtype)):
        return t
    return t.to(device=dev, dtype=dtype)


def _grad_wanted(*ts: torch.Tensor | None) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _refuse_dropped(name: str, operands: tuple, constants: dict) -> None:
    """Refuses derivatives that the kernels would drop: tangents of forward mode on any operand (``requires_grad`` does
    not show them), and gradients of ``constants``, which the operator is not differentiable in."""
    if forward_ad._current_level >= 0:
        for t in (*operands, *constants.values()):
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{name} has no forward-mode derivative: an operand has a tangent")
    for what, t in constants.items():
        if isinstance(t, torch.Tensor) and _grad_wanted(t):
            raise RuntimeError(f"{name} is not differentiable in {what}: detach it")


def _result(out: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    if like.is_cuda:
        return out
    return out.to(like.device) if out.requires_grad else _back(out, like)


def _check_dtype(name: str, *ts: torch.Tensor) -> None:
    if ts[0].dtype not in _DTYPES:
        raise TypeError(f"{name}: dtype {ts[0].dtype} not supported (float32, bfloat16)")
    for t in ts[1:]:
        if t.dtype != ts[0].dtype:
            raise TypeError(f"{name}: operands of different dtypes ({ts[0].dtype}, {t.dtype})")


# ---------------------------------------------------------------------------
# norm and rotation of queries and keys
# ---------------------------------------------------------------------------


def _qk_args(xs, outs, dys, weights, dws, positions, inv_freq, eps, interleaved):
    a = _lib.QkNormRopeArgs()
    q = xs[0]
    a.batch, a.seq, a.head_dim, a.rotary_dim = q.shape[0], q.shape[2], q.shape[3], 2 * inv_freq.shape[0]
    wdt = None
    for i, x in enumerate(xs):
        a.heads[i] = x.shape[1]
        a.x[i], a.out[i] = x.data_ptr(), outs[i].data_ptr()
        a.x_strides[i][:] = x.stride()[:3]
        a.out_strides[i][:] = outs[i].stride()[:3]
        if dys is not None:
            a.dy[i] = dys[i].data_ptr()
            a.dy_strides[i][:] = dys[i].stride()[:3]
        if weights[i] is not None:
            a.weight[i], wdt = weights[i].data_ptr(), weights[i].dtype
        if dws is not None and dws[i] is not None:
            a.dw[i] = dws[i].data_ptr()
    a.positions, a.position_type = positions.data_ptr(), _lib.index_code(positions.dtype)
    a.position_batch_stride = positions.shape[1] if positions.dim() == 2 else 0
    a.inv_freq = inv_freq.data_ptr()
    a.eps, a.interleaved = eps, int(interleaved)
    a.dtype, a.weight_dtype = _lib.dtype_code(q.dtype), _lib.dtype_code(wdt or torch.float32)
    return a


def _qk_forward(q, k, positions, inv_freq, qw, kw, eps, interleaved):
    outs = [torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k)]
    a = _qk_args((q, k), outs, None, (qw, kw), None, positions, inv_freq, eps, interleaved)
    _on_device(q.device, lambda stream: _lib.call("trnsparse_qk_norm_rope", C.byref(a), stream))
    return outs


class _QkNormRopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, qw, kw, positions, inv_freq, eps, interleaved):
        ctx.save_for_backward(q, k, qw, kw, positions, inv_freq)
        ctx.eps, ctx.interleaved = eps, interleaved
        return tuple(_qk_forward(q, k, positions, inv_freq, qw, kw, eps, interleaved))

    @staticmethod
    @once_differentiable
    def backward(ctx, dyq, dyk):
        q, k, qw, kw, positions, inv_freq = ctx.saved_tensors
        dys = [_rows(t) for t in (dyq, dyk)]
        dxs = [torch.empty_like(t) for t in (q, k)]  # in the inputs' layout where that is dense
        dxs = [t if t.stride(-1) == 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in dxs]
        need = ctx.needs_input_grad
        dws = [torch.empty_like(w) if w is not None and need[2 + i] else None for i, w in enumerate((qw, kw))]
        a = _qk_args((q, k), dxs, dys, (qw, kw), dws, positions, inv_freq, ctx.eps, ctx.interleaved)

        def run(stream):
            n = _lib.raw("trnsparse_qk_norm_rope_workspace_size")(C.byref(a))
            ws = torch.empty(max(n, 16), dtype=torch.uint8, device=q.device)
            _lib.call("trnsparse_qk_norm_rope_backward", C.byref(a), ws.data_ptr(), ws.numel(), stream)

        _on_device(q.device, run)
        return dxs[0], dxs[1], dws[0], dws[1], None, None, None, None


def qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every query and key head and its position rotation, in one pass.

    ``q``: ``(batch, q_heads, seq, head_dim)``, ``k``: ``(batch, k_heads, seq,
    head_dim)``, float32 or bfloat16, head_dim up to 256; any strides, so the
    ``transpose(1, 2)`` of a projection's ``(batch, seq, heads, head_dim)``
    output needs no copy. Returns both as contiguous ``(batch, heads, seq,
    head_dim)``, the layout the attention operators read fastest.

    Each head vector becomes ``x / sqrt(mean(x**2) + eps) * weight`` (weights
    of shape ``(head_dim,)``, float32 or bfloat16, ``None`` for ones), then the
    pairs of its first ``2 * len(inv_freq)`` elements are turned by
    ``position * inv_freq[j]``: pair j is elements ``(j, j + len(inv_freq))``,
    or ``(2j, 2j + 1)`` when ``interleaved``. ``positions``: integers, ``(seq,)``
    or ``(batch, seq)``. ``inv_freq``: the table a program keeps, usually
    ``base ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)``; keep it in
    float64 on the device (other types are converted at every call). Angles
    are formed in 64 bits, everything else in 32, rounded once.
    Differentiable in ``q``, ``k`` and the weights; gradients of the weights
    are summed in a fixed order. An ``inv_freq`` or ``eps`` that requires a
    gradient, and forward-mode tangents, are refused.
    """
    assert q.dim() == 4 and k.dim() == 4, f"qk_norm_rope: q and k must be 4-D, got {tuple(q.shape)}, {tuple(k.shape)}"
    B, _, S, D = q.shape
    assert k.shape[0] == B and k.shape[2] == S and k.shape[3] == D, (
        f"qk_norm_rope: k {tuple(k.shape)} does not match q {tuple(q.shape)}")
    assert 1 <= D <= 256, f"qk_norm_rope: head_dim must be in [1, 256], got {D}"
    _check_dtype("qk_norm_rope", q, k)
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"qk_norm_rope: positions must be int32 or int64, got {positions.dtype}")
    assert tuple(positions.shape) in ((S,), (B, S)), (
        f"qk_norm_rope: positions must be ({S},) or ({B}, {S}), got {tuple(positions.shape)}")
    assert inv_freq.dim() == 1 and 2 * inv_freq.shape[0] <= D, (
        f"qk_norm_rope: inv_freq {tuple(inv_freq.shape)} has more pairs than head_dim {D}")
    if not inv_freq.dtype.is_floating_point:
        raise TypeError(f"qk_norm_rope: inv_freq must be floating point, got {inv_freq.dtype}")
    wdt = None
    for w in (q_weight, k_weight):
        if w is None:
            continue
        assert tuple(w.shape) == (D,), f"qk_norm_rope: weights must be ({D},), got {tuple(w.shape)}"
        if w.dtype not in _DTYPES or (wdt is not None and w.dtype != wdt):
            raise TypeError("qk_norm_rope: weights must be float32 or bfloat16, both alike")
        wdt = w.dtype
    _refuse_dropped("qk_norm_rope", (q, k, q_weight, k_weight), {"inv_freq": inv_freq, "eps": eps})
    dev = _dev_of(q, k)
    qd, kd = _rows(_to(q, dev)), _rows(_to(k, dev))
    qw, kw = (None if w is None else _to(w, dev).contiguous() for w in (q_weight, k_weight))
    pos = _to(positions, dev).contiguous()
    freq = _to(inv_freq, dev, torch.float64).contiguous()
    if _grad_wanted(qd, kd, qw, kw):
        yq, yk = _QkNormRopeFn.apply(qd, kd, qw, kw, pos, freq, float(eps), bool(interleaved))
    else:
        yq, yk = _qk_forward(qd, kd, pos, freq, qw, kw, float(eps), bool(interleaved))
    return _result(yq, q), _result(yk, k)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------


def _attention_args(q, k, v, out, lse, lengths, mask, scale):
    a = _lib.AttentionArgs()
    a.batch, a.q_heads, a.q_len, a.head_dim = q.shape
    a.kv_heads, a.k_len = k.shape[1], k.shape[2]
    a.q, a.k, a.v, a.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    a.q_strides[:], a.k_strides[:] = q.stride()[:3], k.stride()[:3]
    a.v_strides[:], a.out_strides[:] = v.stride()[:3], out.stride()[:3]
    if lse is not None:
        a.lse = lse.data_ptr()
    if lengths is not None:
        a.key_lengths = lengths.data_ptr()
    if mask is not None:
        a.key_mask, a.key_mask_stride = mask.data_ptr(), mask.stride(0)
    a.scale, a.dtype = scale, _lib.dtype_code(q.dtype)
    return a


def _like(t: torch.Tensor) -> torch.Tensor:
    """An empty tensor in ``t``'s layout where that is dense with unit last stride, else contiguous."""
    out = torch.empty_like(t)
    return out if out.stride(-1) == 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _run_attention(name, a, dev):
    def run(stream):
        n = _lib.raw(name + "_workspace_size")(C.byref(a))
        ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
        _lib.call(name, C.byref(a), _lib.ptr(ws), n, stream)

    _on_device(dev, run)


def _cross_forward(q, k, v, lengths, mask, scale, want_lse):
    out = _like(q)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device) if want_lse else None
    if out.numel():
        _run_attention("trnsparse_cross_attention", _attention_args(q, k, v, out, lse, lengths, mask, scale), q.device)
    return out, lse


class _CrossAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, mask, scale):
        out, lse = _cross_forward(q, k, v, lengths, mask, scale, True)
        ctx.save_for_backward(q, k, v, out, lse, lengths, mask)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, lengths, mask = ctx.saved_tensors
        want_q, want_kv = ctx.needs_input_grad[0], ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dq = _like(q) if want_q else None
        dk, dv = (_like(k), _like(v)) if want_kv else (None, None)
        if q.numel() == 0:
            return dq, None if dk is None else dk.zero_(), None if dv is None else dv.zero_(), None, None, None
        dout = _tiles(dout)
        a = _attention_args(q, k, v, out, lse, lengths, mask, ctx.scale)
        a.dout, a.dout_strides[:] = dout.data_ptr(), dout.stride()[:3]
        for t, ptr, strides in ((dq, "dq", a.dq_strides), (dk, "dk", a.dk_strides), (dv, "dv", a.dv_strides)):
            if t is not None:
                setattr(a, ptr, t.data_ptr())
                strides[:] = t.stride()[:3]
        _run_attention("trnsparse_cross_attention_backward", a, q.device)
        return dq, dk, dv, None, None, None


def _check_attention(name, q, k, v):
    assert q.dim() == 4 and k.dim() == 4, f"{name}: q, k, v must be 4-D, got {tuple(q.shape)}, {tuple(k.shape)}"
    assert k.shape == v.shape, f"{name}: k {tuple(k.shape)} and v {tuple(v.shape)} differ"
    assert k.shape[0] == q.shape[0] and k.shape[3] == q.shape[3], (
        f"{name}: k {tuple(k.shape)} does not match q {tuple(q.shape)}")
    assert 1 <= q.shape[3] <= 256, f"{name}: head_dim must be in [1, 256], got {q.shape[3]}"
    assert k.shape[1] > 0 and q.shape[1] % k.shape[1] == 0, (
        f"{name}: {q.shape[1]} query heads are not a multiple of {k.shape[1]} key heads")
    _check_dtype(name, q, k, v)


def _check_scale(name, scale, D):
    scale = float(D ** -0.5 if scale is None else scale)
    assert abs(scale) <= 1e38, f"{name}: scale must be finite in float32, got {scale}"  # a NaN fails too
    return scale


def _check_lengths(name, lengths, B):
    if lengths.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name}: lengths must be int32 or int64, got {lengths.dtype}")
    assert tuple(lengths.shape) == (B,), f"{name}: lengths must be ({B},), got {tuple(lengths.shape)}"


def _lengths32(lengths, dev, most):
    """``lengths`` as the kernels read them; 64-bit values are clamped before they are narrowed (two small launches)."""
    if lengths.dtype == torch.int64:
        lengths = lengths.clamp(0, most).to(torch.int32)
    return _to(lengths, dev).contiguous()


def cross_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    key_lengths: torch.Tensor | None = None,
    key_mask: torch.Tensor | None = None,
    scale: float | None = None,
) -> torch.Tensor:
    """Softmax attention of ``q`` over another sequence's keys (encoder states).

    ``q``: ``(batch, q_heads, q_len, head_dim)``; ``k``, ``v``: ``(batch,
    kv_heads, k_len, head_dim)``, any lengths, ``q_heads`` a multiple of
    ``kv_heads`` (query head i reads key head ``i // (q_heads // kv_heads)``),
    head_dim up to 256, float32 or bfloat16, any strides. One token per
    sequence (decoding) splits the keys over the GPU. ``key_lengths``:
    ``(batch,)`` integers, the leading keys of each sequence that count
    (clamped to ``[0, k_len]``). ``key_mask``: ``(batch, k_len)`` bool, True
    where a key counts; given both, a key must pass both. What hidden keys
    hold (NaN included) does not matter, the others are finite; a row without
    keys is zero, and so are its gradients. ``scale``, any finite number,
    defaults to ``head_dim ** -0.5``. The result has ``q``'s layout.

    Softmax and sums are float32. bfloat16 calls whose head_dim is a multiple
    of 8 up to 128 round the probabilities to bfloat16 before they weigh the
    values, and in the backward pass them and the scores' gradients before
    their products: results are off by 2.3e-3 of their size, gradients by
    2.4e-3, where the rounding of the result alone makes 1.7e-3.

    Differentiable in ``q``, ``k``, ``v``; gradients are summed in a fixed
    order. A ``scale`` that requires a gradient, and forward-mode tangents,
    are refused. ``k_len`` and ``batch * q_heads * q_len`` are below ``2**30``.
    """
    name = "cross_attention"
    _check_attention(name, q, k, v)
    B, Sk = k.shape[0], k.shape[2]
    if key_lengths is not None:
        _check_lengths(name, key_lengths, B)
    if key_mask is not None:
        if key_mask.dtype != torch.bool:
            raise TypeError(f"{name}: key_mask must be bool, got {key_mask.dtype}")
        assert tuple(key_mask.shape) == (B, Sk), f"{name}: key_mask must be ({B}, {Sk}), got {tuple(key_mask.shape)}"
    _refuse_dropped(name, (q, k, v), {"scale": scale})
    scale = _check_scale(name, scale, q.shape[3])
    dev = _dev_of(q, k, v)
    qd, kd, vd = (_tiles(_to(t, dev)) for t in (q, k, v))
    lengths = None if key_lengths is None else _lengths32(key_lengths, dev, Sk)
    mask = None if key_mask is None else _rows(_to(key_mask, dev))
    if _grad_wanted(qd, kd, vd):
        out = _CrossAttentionFn.apply(qd, kd, vd, lengths, mask, scale)
    else:
        out, _ = _cross_forward(qd, kd, vd, lengths, mask, scale, False)
    return _result(out, q)


def shared_prefix_attention(
    q: torch.Tensor,
    prefix_k: torch.Tensor,
    prefix_v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    lengths: torch.Tensor,
    scale: float | None = None,
) -> torch.Tensor:
    """Decoding attention of a batch that shares a prefix, read once for all of it.

    ``q``: ``(batch, q_heads, tokens, head_dim)``, the new tokens of each
    sequence (usually one). ``prefix_k``, ``prefix_v``: ``(kv_heads,
    prefix_len, head_dim)``. ``k_cache``, ``v_cache``: ``(batch, kv_heads,
    capacity, head_dim)``, each sequence's own keys; ``lengths``: ``(batch,)``
    integers, how many of them are filled (clamped to ``[0, capacity]``), the
    new tokens included: token t of T attends the whole prefix and the first
    ``lengths - T + 1 + t`` own keys. Rows behind a length are never read into
    a result; what is read is finite. float32 or bfloat16, head_dim up to 256, any strides (a slice of
    a larger cache needs no copy). A row without any key is zero. Probabilities
    of bfloat16 calls are rounded as in ``cross_attention``. For serving:
    operands that require gradients or have forward-mode tangents are refused.
    """
    name = "shared_prefix_attention"
    _check_attention(name, q, k_cache, v_cache)
    Hkv, D = k_cache.shape[1], q.shape[3]
    assert prefix_k.dim() == 3 and prefix_k.shape == prefix_v.shape, (
        f"{name}: prefix_k {tuple(prefix_k.shape)} and prefix_v {tuple(prefix_v.shape)} must be 3-D and alike")
    assert prefix_k.shape[0] == Hkv and prefix_k.shape[2] == D, (
        f"{name}: prefix {tuple(prefix_k.shape)} does not match the cache {tuple(k_cache.shape)}")
    _check_dtype(name, q, prefix_k, prefix_v)
    _check_lengths(name, lengths, q.shape[0])
    if _grad_wanted(q, prefix_k, prefix_v, k_cache, v_cache):
        raise RuntimeError(f"{name} has no backward pass: call it under torch.no_grad() or detach its operands")
    _refuse_dropped(name, (q, prefix_k, prefix_v, k_cache, v_cache), {"scale": scale})
    scale = _check_scale(name, scale, D)
    dev = _dev_of(q, prefix_k, k_cache)
    qd, pk, pv, kc, vc = (_tiles(_to(t, dev)) for t in (q, prefix_k, prefix_v, k_cache, v_cache))
    lens = _lengths32(lengths, dev, kc.shape[2])
    out = _like(qd)
    if out.numel():
        a = _attention_args(qd, kc, vc, out, None, lens, None, scale)
        a.prefix_k, a.prefix_v, a.prefix_len = pk.data_ptr(), pv.data_ptr(), pk.shape[1]
        a.prefix_k_strides[:], a.prefix_v_strides[:] = pk.stride()[:2], pv.stride()[:2]
        _run_attention("trnsparse_shared_prefix_attention", a, dev)
    return _result(out, q)
