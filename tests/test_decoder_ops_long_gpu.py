"""Decoder attention over millions of keys walked by one CTA."""

from __future__ import annotations

import pytest
import torch

import trnsparse_b200 as ts
from trnsparse_b200 import _lib
from decoder_ref import check

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _ones(B, Sq, Sk, D, lengths=None):
    """Queries, keys and values of ones, the keys of all sequences the same memory. The result is 1: the scores are
    equal, P is 1, and 16 ones (a product's step) added to a multiple of 16 below 2^28 are exact in fp32."""
    q = torch.ones(B, 1, Sq, D, device="cuda", dtype=BF16)
    k = torch.ones(1, 1, Sk, D, device="cuda", dtype=BF16).expand(B, 1, Sk, D)
    out = ts.cross_attention(q, k, k, lengths)
    check(out, torch.ones_like(out, dtype=torch.float64), torch.full_like(out, 2.0 ** -8, dtype=torch.float64), "out")
    assert _lib.device_error() == 0


def test_row_sums_pass_2_to_the_24():
    """148 items of 17 rows: a whole one for every CTA."""
    _ones(148, 17, 1 << 25, 8)
