"""Attention over a microscaled cache whose first scores are past fp32's range: keys that
overflow to -infinity weigh nothing, whatever the others' scores are."""
from __future__ import annotations

import math

import pytest
import torch

from mx_shared import FORMS, TYPES, Shared

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bf16,hd,bits", TYPES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("low", [-50.0, -212.0, -3000.0])
def test_scores_that_overflow_first(low, form, bf16, hd, bits):
    """The first 512 keys (the first stage of each of a work-group's eight waves) score -2^130;
    the others near `low`, whose weights relative to 0 are all 0 from -104 down."""
    nkv, news = FORMS[form]
    if form == "one":
        nkv = 256  # one work-group to a head
    g = torch.Generator().manual_seed(19)
    k, v = torch.randn(1536, hd, generator=g).double(), torch.randn(1536, hd, generator=g).double()
    q = torch.randn(sum(news), nkv, hd, generator=g)
    q[:, :, 0], q[:, :, 32] = -2.0 ** 60, -1.0
    k[:, 0], k[:, 32] = 0.0, -low * math.sqrt(hd)
    k[:512, 0] = 2.0 ** 70
    b = Shared(k, v, q, news, nkv, bits, bf16)
    b.check(*b.run())
