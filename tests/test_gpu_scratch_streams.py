"""Scratch memory that a call on a given stream allocates for itself is of that
stream: once its tensor is gone, the current stream does not get it while the call
still runs."""
from __future__ import annotations

import pytest
import torch

import mx230_amd as mx

pytestmark = pytest.mark.gpu


def apart(a, b):
    return a[0] + a[1] <= b[0] or b[0] + b[1] <= a[0]


def span(t):
    return t.data_ptr(), t.numel() * t.element_size()


@pytest.mark.parametrize("paged", [False, True])
def test_split_prefill(paged):
    g = torch.Generator(device="cuda").manual_seed(1)
    nh, nkv, hd, pos0, n = 4, 2, 64, 4000, 8
    q = torch.randn(n, nh * hd, device="cuda", generator=g).bfloat16()
    k, v = (torch.randn(pos0 + 96, nkv * hd, device="cuda", generator=g).bfloat16() for _ in range(2))
    table = torch.arange(256, dtype=torch.int32, device="cuda")
    out = [torch.zeros_like(q) for _ in range(3)]
    s = torch.cuda.Stream()
    torch.cuda.synchronize()

    def call(o, stream):
        if paged:
            return mx.run_prefill_paged(q, k, v, o, table, 16, pos0, nh, nkv, hd, stream=stream, split=True)
        return mx.run_prefill_split(q, k, v, o, pos0, nh, nkv, hd, stream=stream)
    spans = []
    for o, stream in zip(out, (None, s, None)):
        ws = call(o, stream)
        spans.append(span(ws))
        del ws
    assert spans[0][1] > 16 and apart(spans[0], spans[1]) and apart(spans[1], spans[2])
    torch.cuda.synchronize()
    assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2]) and bool(out[0].any())


def test_backward(monkeypatch):
    """Delta, and the partial dK and dV of grouped heads."""
    g = torch.Generator(device="cuda").manual_seed(2)
    q, do = (torch.randn(1, 8, 2048, 64, device="cuda", generator=g).bfloat16() for _ in range(2))
    k, v = (torch.randn(1, 2, 2048, 64, device="cuda", generator=g).bfloat16() for _ in range(2))
    o, lse = mx.attention_fwd(q, k, v, True)
    want = mx.attention_bwd(q, k, v, o, lse, do, True)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    spans, run = [], mx.run_bwd_ws

    def seen(*a):
        spans.append(span(a[6]))
        if a[10] is not None:
            spans.append(span(a[10]))
        return run(*a)
    monkeypatch.setattr(mx, "run_bwd_ws", seen)
    got = mx.attention_bwd(q, k, v, o, lse, do, True, stream=s)
    here = [torch.empty(n, dtype=torch.uint8, device="cuda") for _, n in spans for _ in range(2)]
    assert spans and all(apart(span(x), y) for x in here for y in spans)
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_streams_of_other_kinds():
    """Whatever has a cuda_stream is a stream."""
    class Other:
        def __init__(self, s):
            self.cuda_stream = s.cuda_stream
    g = torch.Generator(device="cuda").manual_seed(3)
    q, do = (torch.randn(1, 4, 300, 64, device="cuda", generator=g).bfloat16() for _ in range(2))
    k, v = (torch.randn(1, 2, 300, 64, device="cuda", generator=g).bfloat16() for _ in range(2))
    o, lse = mx.attention_fwd(q, k, v, True)
    want = mx.attention_bwd(q, k, v, o, lse, do, True)
    rows = torch.randn(8, 4 * 64, device="cuda", generator=g).bfloat16()
    cache = torch.randn(4096, 2 * 64, device="cuda", generator=g).bfloat16()
    out, two = torch.empty_like(rows), torch.empty_like(rows)
    mx.run_prefill_split(rows, cache, cache, out, 4000, 4, 2, 64)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = mx.attention_bwd(q, k, v, o, lse, do, True, stream=Other(s))
    mx.run_prefill_split(rows, cache, cache, two, 4000, 4, 2, 64, stream=Other(s))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(out, two)
