"""Argument values that the decoder operators' entry points refuse, on the host."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

import trnsparse_b200 as ts
from trnsparse_b200 import _lib

INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("scale", [NAN, INF, -INF, 1e39])
def test_attention_scale_is_finite(scale):
    t = lambda *s: torch.zeros(*s)
    with pytest.raises(AssertionError, match="cross_attention: scale"):
        ts.cross_attention(t(2, 4, 3, 8), t(2, 2, 5, 8), t(2, 2, 5, 8), scale=scale)
    with pytest.raises(AssertionError, match="shared_prefix_attention: scale"):
        ts.shared_prefix_attention(t(2, 4, 1, 8), t(2, 9, 8), t(2, 9, 8), t(2, 2, 5, 8), t(2, 2, 5, 8),
                                   torch.ones(2, dtype=torch.int32), scale=scale)
    lib = _lib.load()
    for dtype in (_lib.F32, _lib.BF16):
        a = _lib.AttentionArgs()
        a.batch, a.q_heads, a.kv_heads, a.q_len, a.k_len, a.head_dim = 1, 2, 1, 1, 8, 64
        a.scale, a.dtype = scale, dtype
        for name in ("trnsparse_cross_attention", "trnsparse_shared_prefix_attention",
                     "trnsparse_cross_attention_backward"):
            assert getattr(lib, name)(C.byref(a), None, 0, None) == _lib.ERR_ARG
            assert b"scale" in lib.trnsparse_last_error()


@pytest.mark.parametrize("field,value,code", [
    ("position_type", 2, _lib.ERR_DTYPE), ("position_type", -1, _lib.ERR_DTYPE),
    ("batch", 1 << 33, _lib.ERR_ARG),  # batch * seq would pass 64 bits
])
def test_qk_norm_rope_positions_and_sizes(field, value, code):
    """Refused by all three entry points, also where there is no head to work on."""
    lib = _lib.load()
    a = _lib.QkNormRopeArgs()
    a.batch, a.seq, a.head_dim, a.rotary_dim, a.dtype, a.weight_dtype = 1, (1 << 31) - 1, 64, 64, _lib.F32, _lib.F32
    setattr(a, field, value)
    assert lib.trnsparse_qk_norm_rope(C.byref(a), None) == code
    assert lib.trnsparse_qk_norm_rope_backward(C.byref(a), None, 0, None) == code
    assert lib.trnsparse_qk_norm_rope_workspace_size(C.byref(a)) == 0
