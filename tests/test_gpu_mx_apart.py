"""Attention over a microscaled cache where a key far too low to weigh anything has a V
far larger than the others': it adds nothing."""
from __future__ import annotations

import math

import pytest
import torch

from mx_shared import FORMS, TYPES, Shared

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bf16,hd,bits", TYPES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("small,large", [(2.0 ** -80, 2.0 ** 50), (2.0 ** -100, 2.0 ** 20), (1.0, 2.0 ** 54)])
def test_large_values_without_weight(small, large, form, bf16, hd, bits):
    """Every third key scores some 300 below the others (a weight of 2^-433) and has V of
    `large`; the others' V is of `small`."""
    g = torch.Generator().manual_seed(20)
    nkv, news = FORMS[form]
    k, v = torch.randn(2048, hd, generator=g).double(), torch.randn(2048, hd, generator=g).double()
    q = torch.randn(sum(news), nkv, hd, generator=g)
    q[:, :, 0] = math.sqrt(hd)
    k[:, 0] = 0.0
    k[1::3, 0] = -300.0
    v = (1.0 + v.abs().clamp(max=3.0)) * small
    v[1::3] *= large / small
    b = Shared(k, v, q, news, nkv, bits, bf16, times=8)
    b.check(*b.run(), few=2.0 ** -126)
