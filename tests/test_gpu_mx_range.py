"""Attention over a microscaled cache where the numbers lie far apart: V near the least
that the cache holds, behind weights of every size."""
from __future__ import annotations

import math

import pytest
import torch

from mx_shared import FORMS, TYPES, Shared

pytestmark = pytest.mark.gpu

# a result below 2^-126 may be 0
LEAST = 2.0 ** -126


def inputs(form, hd, seed, n=2048):
    g = torch.Generator().manual_seed(seed)
    nkv, news = FORMS[form]
    k, v = torch.randn(n, hd, generator=g), torch.randn(n, hd, generator=g)
    # (of one sign, so that weights that are left out show)
    return k.bfloat16().double(), 1.0 + v.double().abs().clamp(max=3.0), torch.randn(sum(news), nkv, hd, generator=g), news, nkv


@pytest.mark.parametrize("bf16,hd,bits", TYPES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("size,wide", [(1e-34, 2.0), (1e-34, 3.0), (1e-32, 3.0), (1e-20, 3.0)])
def test_small_values_behind_small_weights(size, wide, form, bf16, hd, bits):
    """Scores of deviation `wide` over 16384 keys: most of the sum is of weights far below
    the largest."""
    k, v, q, news, nkv = inputs(form, hd, 17)
    b = Shared(k, v * size, q * wide, news, nkv, bits, bf16, times=8)
    b.check(*b.run(), few=LEAST)


@pytest.mark.parametrize("bf16,hd,bits", TYPES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("size,lead,own", [(1e-34, 10.0, 1.0), (1e-32, 10.0, 1.0), (2.0 ** -112, 8.0, 0.0)])
def test_small_values_behind_one_key(size, lead, own, form, bf16, hd, bits):
    """A key whose score is `lead` above the others', its V of their size or 0: theirs are a
    good part of the result."""
    k, v, q, news, nkv = inputs(form, hd, 18)
    q[:, :, 0] = math.sqrt(hd)
    k[:, 0] = 0.0
    k[700, 0] = lead
    v[700] *= own
    b = Shared(k, v * size, q, news, nkv, bits, bf16, times=8)
    b.check(*b.run(), few=LEAST)
