"""Rotary positions and the cache append at the ends of what they take: rows that do
not begin on 16 bytes, and lengths at the ends of 32 bits."""
from __future__ import annotations

import pytest
import torch

import mx230_amd as mx
from mx230_amd.autograd import rotary_embedding

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("python", [False, True])
def test_embedding_of_rows_off_16_bytes(dt, python, monkeypatch):
    """Contiguous Q and K that begin between 16-byte boundaries, and gradients that
    do: as of tensors on them."""
    if python:
        monkeypatch.setattr(mx.autograd, "_calls", lambda: mx._NoBinding)
    f, _ = mx.rotary_frequencies(64)
    g = torch.Generator().manual_seed(6)
    q, k = (torch.randn(2, h, 9, 64, generator=g).to(dt).cuda() for h in (4, 2))
    wq, wk = (torch.randn(x.shape, generator=g).to(dt).cuda() for x in (q, k))

    def off(x):
        y = torch.empty(x.numel() + 1, dtype=dt, device="cuda")[1:].view(x.shape)
        y.copy_(x)
        assert y.is_contiguous() and y.data_ptr() % 16
        return y
    want = rotary_embedding(q.requires_grad_(), k.requires_grad_(), f)
    torch.autograd.backward(want, (wq, wk))
    a, b = off(q.detach()).requires_grad_(), off(k.detach()).requires_grad_()
    got = rotary_embedding(a, b, f)
    torch.autograd.backward(got, (off(wq), off(wk)))
    for x, y in zip((*want, q.grad, k.grad), (*got, a.grad, b.grad)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("length", [-2 ** 31, -2 ** 31 + 1, -1, 0])
def test_append_at_negative_positions(length):
    """A token at a position below 0, however far, is left out."""
    bs = 1 << 24
    table = torch.full((1, 128), 0, dtype=torch.int32, device="cuda")
    k, v = (torch.full((bs, 8), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    qkv = torch.ones(2, 24, dtype=torch.bfloat16, device="cuda")
    out = torch.full((2, 8), 7.0, dtype=torch.bfloat16, device="cuda")
    cu, lens = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 2], [length]))
    mx.run_cache_append(qkv, out, k, v, table, bs, cu, lens, 1, 1, 8, mx.rotary_frequencies(8)[0])
    assert bool((out == 7.0).all()) and bool((k == 7.0).all()) and bool((v == 7.0).all())
