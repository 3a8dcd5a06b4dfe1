"""Derivatives the decoder operators do not have are refused, before any CUDA call, never dropped."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import trnsparse_b200 as ts


def _t(*shape):
    return torch.zeros(*shape)


def _qk(**kw):
    return ts.qk_norm_rope(**{**dict(q=_t(2, 4, 3, 8), k=_t(2, 2, 3, 8), positions=torch.arange(3),
                                     inv_freq=torch.ones(4, dtype=torch.float64), q_weight=_t(8), k_weight=_t(8)), **kw})


def _cross(**kw):
    return ts.cross_attention(**{**dict(q=_t(2, 4, 3, 8), k=_t(2, 2, 5, 8), v=_t(2, 2, 5, 8)), **kw})


def _prefix(**kw):
    return ts.shared_prefix_attention(**{**dict(
        q=_t(2, 4, 1, 8), prefix_k=_t(2, 9, 8), prefix_v=_t(2, 9, 8), k_cache=_t(2, 2, 5, 8), v_cache=_t(2, 2, 5, 8),
        lengths=torch.ones(2, dtype=torch.int32)), **kw})


@pytest.mark.parametrize("op,arg,shape", [
    (_qk, "q", (2, 4, 3, 8)), (_qk, "k", (2, 2, 3, 8)), (_qk, "q_weight", (8,)), (_qk, "k_weight", (8,)),
    (_qk, "inv_freq", (4,)), (_cross, "q", (2, 4, 3, 8)), (_cross, "k", (2, 2, 5, 8)), (_cross, "v", (2, 2, 5, 8)),
    (_cross, "scale", ()), (_prefix, "q", (2, 4, 1, 8)), (_prefix, "prefix_k", (2, 9, 8)),
    (_prefix, "prefix_v", (2, 9, 8)), (_prefix, "k_cache", (2, 2, 5, 8)), (_prefix, "v_cache", (2, 2, 5, 8)),
])
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(op, arg, shape, grad):
    """Also without a graph: torch.no_grad() leaves forward mode on."""
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        dual = forward_ad.make_dual(torch.zeros(shape), torch.ones(shape))
        with pytest.raises(RuntimeError, match="has no forward-mode derivative"):
            op(**{arg: dual})


@pytest.mark.parametrize("op,arg,value", [
    (_qk, "inv_freq", torch.ones(4, dtype=torch.float64)), (_qk, "eps", torch.tensor(1e-6)),
    (_cross, "scale", torch.tensor(0.3)), (_prefix, "scale", torch.tensor(0.3)),
])
def test_gradients_of_constants_are_refused(op, arg, value):
    with pytest.raises(RuntimeError, match=f"not differentiable in {arg}"):
        op(**{arg: value.clone().requires_grad_(True)})
