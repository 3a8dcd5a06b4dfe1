"""Refusals of the decoder operators: made by the argument checks, before any CUDA call."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

import trnsparse_b200 as ts
from trnsparse_b200 import _lib


def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def _qk(**kw):
    a = dict(q=_t(2, 4, 3, 8), k=_t(2, 2, 3, 8), positions=torch.arange(3), inv_freq=torch.ones(4, dtype=torch.float64))
    a.update(kw)
    return ts.qk_norm_rope(**a)


@pytest.mark.parametrize("kw,err", [
    (dict(q=_t(4, 3, 8)), AssertionError),
    (dict(k=_t(2, 2, 5, 8)), AssertionError),
    (dict(k=_t(1, 2, 3, 8)), AssertionError),
    (dict(k=_t(2, 2, 3, 16)), AssertionError),
    (dict(q=_t(2, 4, 3, 258), k=_t(2, 2, 3, 258)), AssertionError),
    (dict(q=_t(2, 4, 3, 8, dtype=torch.float16), k=_t(2, 2, 3, 8, dtype=torch.float16)), TypeError),
    (dict(k=_t(2, 2, 3, 8, dtype=torch.bfloat16)), TypeError),
    (dict(positions=torch.arange(3).float()), TypeError),
    (dict(positions=torch.arange(4)), AssertionError),
    (dict(positions=torch.zeros(3, 3, dtype=torch.int32)), AssertionError),
    (dict(inv_freq=torch.ones(5)), AssertionError),
    (dict(inv_freq=torch.ones(2, 2)), AssertionError),
    (dict(inv_freq=torch.ones(4, dtype=torch.int64)), TypeError),
    (dict(q_weight=_t(4)), AssertionError),
    (dict(q_weight=_t(8, dtype=torch.float16)), TypeError),
    (dict(q_weight=_t(8), k_weight=_t(8, dtype=torch.bfloat16)), TypeError),
])
def test_qk_norm_rope_refuses(kw, err):
    with pytest.raises(err, match="qk_norm_rope"):
        _qk(**kw)


def _cross(**kw):
    a = dict(q=_t(2, 4, 3, 8), k=_t(2, 2, 5, 8), v=_t(2, 2, 5, 8))
    a.update(kw)
    return ts.cross_attention(**a)


@pytest.mark.parametrize("kw,err", [
    (dict(q=_t(4, 3, 8)), AssertionError),
    (dict(v=_t(2, 2, 6, 8)), AssertionError),
    (dict(q=_t(3, 4, 3, 8)), AssertionError),
    (dict(q=_t(2, 4, 3, 16)), AssertionError),
    (dict(q=_t(2, 3, 3, 8)), AssertionError),
    (dict(q=_t(2, 4, 3, 257), k=_t(2, 2, 5, 257), v=_t(2, 2, 5, 257)), AssertionError),
    (dict(k=_t(2, 0, 5, 8), v=_t(2, 0, 5, 8)), AssertionError),
    (dict(q=_t(2, 4, 3, 8, dtype=torch.float64)), TypeError),
    (dict(v=_t(2, 2, 5, 8, dtype=torch.bfloat16)), TypeError),
    (dict(key_lengths=torch.zeros(2)), TypeError),
    (dict(key_lengths=torch.zeros(3, dtype=torch.int32)), AssertionError),
    (dict(key_mask=torch.zeros(2, 5)), TypeError),
    (dict(key_mask=torch.zeros(2, 4, dtype=torch.bool)), AssertionError),
])
def test_cross_attention_refuses(kw, err):
    with pytest.raises(err, match="cross_attention"):
        _cross(**kw)


def _prefix(**kw):
    a = dict(q=_t(2, 4, 1, 8), prefix_k=_t(2, 9, 8), prefix_v=_t(2, 9, 8), k_cache=_t(2, 2, 5, 8),
             v_cache=_t(2, 2, 5, 8), lengths=torch.ones(2, dtype=torch.int32))
    a.update(kw)
    return ts.shared_prefix_attention(**a)


@pytest.mark.parametrize("kw,err", [
    (dict(prefix_k=_t(2, 8, 8)), AssertionError),
    (dict(prefix_k=_t(1, 2, 9, 8), prefix_v=_t(1, 2, 9, 8)), AssertionError),
    (dict(prefix_k=_t(4, 9, 8), prefix_v=_t(4, 9, 8)), AssertionError),
    (dict(v_cache=_t(2, 2, 6, 8)), AssertionError),
    (dict(lengths=torch.ones(2)), TypeError),
    (dict(lengths=torch.ones(1, dtype=torch.int64)), AssertionError),
    (dict(prefix_k=_t(2, 9, 8, dtype=torch.bfloat16)), TypeError),
    (dict(q=_t(2, 4, 1, 8).requires_grad_(True)), RuntimeError),
])
def test_shared_prefix_attention_refuses(kw, err):
    with pytest.raises(err, match="shared_prefix_attention"):
        _prefix(**kw)


def _args():
    a = _lib.AttentionArgs()
    a.batch, a.q_heads, a.kv_heads, a.q_len, a.k_len, a.head_dim = 1, 2, 1, 1, 8, 64
    a.dtype = _lib.BF16
    return a


@pytest.mark.parametrize("field,value,code", [
    ("batch", -1, _lib.ERR_ARG), ("head_dim", 0, _lib.ERR_ARG), ("head_dim", 300, _lib.ERR_ARG),
    ("kv_heads", 0, _lib.ERR_ARG), ("kv_heads", 3, _lib.ERR_ARG), ("q_len", 1 << 40, _lib.ERR_ARG),
    ("dtype", _lib.F16, _lib.ERR_DTYPE), ("q", None, _lib.ERR_ARG),
])
def test_attention_entry_points_refuse(field, value, code):
    lib = _lib.load()
    for name in ("trnsparse_cross_attention", "trnsparse_shared_prefix_attention",
                 "trnsparse_cross_attention_backward"):
        a = _args()
        setattr(a, field, value)
        assert getattr(lib, name)(C.byref(a), None, 0, None) == code
        assert b"attention" in lib.trnsparse_last_error()
        assert getattr(lib, name)(None, None, 0, None) == _lib.ERR_ARG


def test_qk_norm_rope_entry_point_refuses():
    lib = _lib.load()
    for field, value, code in (("batch", -1, _lib.ERR_ARG), ("head_dim", 257, _lib.ERR_ARG),
                               ("rotary_dim", 3, _lib.ERR_ARG), ("rotary_dim", 66, _lib.ERR_ARG),
                               ("dtype", _lib.F64, _lib.ERR_DTYPE), ("weight_dtype", _lib.F16, _lib.ERR_DTYPE),
                               ("positions", None, _lib.ERR_ARG)):
        a = _lib.QkNormRopeArgs()
        a.batch, a.seq, a.head_dim, a.rotary_dim, a.dtype, a.weight_dtype = 1, 1, 64, 64, _lib.F32, _lib.F32
        a.heads[:] = [1, 1]
        setattr(a, field, value)
        assert lib.trnsparse_qk_norm_rope(C.byref(a), None) == code


def test_argument_structs_match_the_header():
    """The ctypes mirrors list the header's struct fields in its order."""
    import re
    from pathlib import Path

    text = (Path(_lib.__file__).resolve().parent.parent / "include" / "trnsparse_b200.h").read_text()
    for name, cls in (("trnsparse_qk_norm_rope_args", _lib.QkNormRopeArgs),
                      ("trnsparse_attention_args", _lib.AttentionArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = []
        for decl in body.split(";"):
            decl = decl.strip()
            if not decl:
                continue
            m = re.match(r"(?:const\s+)?(?:unsigned\s+)?\w+\s*(.*)", decl, re.S)
            fields += [re.sub(r"[\s\*]|\[.*", "", f) for f in m.group(1).split(",")]
        assert fields == [f[0] for f in cls._fields_]
