"""Rotary positions (mxfa_run_rotary): both pairings, parts of a head, far positions,
strided and in-place tensors, the gradient, and the attention block that uses it,
against the rotation in 64 bits."""
from __future__ import annotations

import pytest
import torch

import mx230_amd as mx
from cache_helpers import turned, turned_tolerance

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _check(got, x, positions, f, interleaved=False, factor=1.0, sign=1.0):
    x = x.cpu()
    want = turned(x, positions, f.cpu(), interleaved, factor, sign)
    off = (got.cpu().double() - want).abs()
    tol = turned_tolerance(x, want, f.numel(), interleaved, factor)
    assert got.dtype == x.dtype and bool((off <= tol).all()), float((off - tol).max())


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,Hq,Hkv,N,d,dim", [
    (1, 1, 1, 1, 64, 64), (2, 4, 2, 33, 64, 64), (1, 14, 2, 100, 64, 32), (3, 5, 5, 7, 128, 128), (1, 3, 1, 50, 128, 24),
    (1, 2, 1, 9, 64, 2), (2, 1, 1, 65, 96, 50), (1, 9, 3, 130, 8, 8), (1, 40, 8, 257, 256, 256), (1, 6, 2, 70, 64, 44)])
def test_rotary(B, Hq, Hkv, N, d, dim, interleaved, dt):
    g = torch.Generator().manual_seed(B + N + dim)
    q, k = (torch.randn(B, h, N, d, generator=g).to(dt).cuda() for h in (Hq, Hkv))
    f, _ = mx.rotary_frequencies(dim)
    qo, ko = (torch.full_like(x, float("nan")) for x in (q, k))
    mx.run_rotary(q, k, qo, ko, f, pos0=5, interleaved=interleaved, factor=1.25)
    at = torch.arange(5, 5 + N)
    for got, x in ((qo, q), (ko, k)):
        _check(got, x, at, f, interleaved, 1.25)
    # Q alone, its positions given, the other direction
    at = torch.randint(-3000, 200000, (B, N), generator=g, dtype=torch.int32)
    mx.run_rotary(q, None, qo, None, f, positions=at.cuda(), interleaved=interleaved, inverse=True)
    _check(qo, q, at[:, None], f, interleaved, sign=-1.0)


@pytest.mark.parametrize("pos", [0, 1, -1, 4095, 2 ** 20, 2 ** 30 + 12345, 2 ** 31 - 2, -2 ** 31])
def test_far_positions(pos):
    """The angle of a far position keeps its accuracy (2^31 times the fastest
    frequency, off by a rounding of 64 bits, is 5e-7 of a radian)."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(1, 2, 1, 64, generator=g).cuda()
    f, _ = mx.rotary_frequencies(64)
    at = torch.tensor([pos], dtype=torch.int32)
    y = torch.empty_like(x)
    mx.run_rotary(x, None, y, None, f, positions=at.cuda())
    want = turned(x.cpu(), at, f.cpu())
    tol = turned_tolerance(x.cpu(), want, 32)
    size = (x.cpu().double()[..., :32].abs() + x.cpu().double()[..., 32:].abs()).repeat(1, 1, 1, 2)
    # position times frequency is rounded three times here, twice in the reference
    tol = tol + size * abs(pos) * 5 * 2.0 ** -53
    assert bool(((y.cpu().double() - want).abs() <= tol).all())


def test_special_values_stay_in_their_pair():
    x = torch.ones(1, 1, 4, 64, device="cuda")
    x[0, 0, 1, 3], x[0, 0, 2, 40], x[0, 0, 3, 63] = float("nan"), float("inf"), -0.0
    y = torch.empty_like(x)
    f, _ = mx.rotary_frequencies(64)
    mx.run_rotary(x, None, y, None, f)
    bad = ~torch.isfinite(y[0, 0]).cpu()
    want = torch.zeros(4, 64, dtype=torch.bool)
    want[1, [3, 35]] = want[2, [8, 40]] = True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_strided_and_in_place(dt, interleaved):
    """Q and K as columns of a fused buffer of token rows, with and without a batch;
    in place there; the V columns stay as they are."""
    B, N, Hq, Hkv, d = 2, 37, 6, 2, 64
    g = torch.Generator().manual_seed(4)
    f, _ = mx.rotary_frequencies(48)
    qkv = torch.randn(B, N, Hq + 2 * Hkv, d, generator=g).to(dt).cuda()
    q, k = qkv[:, :, :Hq].transpose(1, 2), qkv[:, :, Hq:Hq + Hkv].transpose(1, 2)
    plain = [torch.empty(x.shape, dtype=dt, device="cuda") for x in (q, k)]
    mx.run_rotary(q, k, *plain, f, interleaved=interleaved)
    for got, x in zip(plain, (q, k)):
        _check(got, x, torch.arange(N), f, interleaved)
    rows = qkv[0, :, :Hq]  # [N, H, d]
    out = torch.empty(N, Hq, d, dtype=dt, device="cuda")
    mx.run_rotary(rows, None, out, None, f, interleaved=interleaved)
    assert torch.equal(out, plain[0][0].transpose(0, 1))
    before = qkv.clone()
    mx.run_rotary(q, k, q, k, f, interleaved=interleaved)
    assert torch.equal(q, plain[0]) and torch.equal(k, plain[1])
    assert torch.equal(qkv[:, :, Hq + Hkv:], before[:, :, Hq + Hkv:])
    # repeated rows as an input: a head broadcast over three
    one = before[:, :, :1].transpose(1, 2)
    out = torch.empty(B, 3, N, d, dtype=dt, device="cuda")
    mx.run_rotary(one.expand(B, 3, N, d), None, out, None, f, interleaved=interleaved)
    assert torch.equal(out[:, 0], out[:, 2]) and torch.equal(out[:, 0], plain[0][:, 0])


def test_python_path_gives_the_same():
    g = torch.Generator().manual_seed(5)
    q = torch.randn(2, 3, 20, 64, generator=g).cuda()
    f, _ = mx.rotary_frequencies(64)
    a, b = torch.empty_like(q), torch.empty_like(q)
    mx.run_rotary(q, None, a, None, f, pos0=3)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    mx.run_rotary(q, None, b, None, f, pos0=3, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(a, b)
    for bad in (dict(positions=torch.zeros(19, dtype=torch.int32, device="cuda")),
                dict(positions=torch.zeros(20, device="cuda"))):
        with pytest.raises(ValueError):
            mx.run_rotary(q, None, a, None, f, **bad)
    with pytest.raises(ValueError):
        mx.run_rotary(q, None, a, None, f.float())
    with pytest.raises(ValueError):
        mx.run_rotary(q, None, a[:1], None, f)
    with pytest.raises(ValueError):
        mx.run_rotary(q, q, a, None, f)
    with pytest.raises(ValueError):
        mx.run_rotary(q.half(), None, a.half(), None, f)
    with pytest.raises(mx.MxfaError):  # the output a token further on over the input
        mx.run_rotary(q[:, :, :10], None, q[:, :, 1:11], None, f)


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient(interleaved):
    """Against the transpose in 64 bits, and against differences of the forward."""
    from mx230_amd.autograd import rotary_embedding
    B, N, Hq, Hkv, d = 2, 11, 4, 2, 64
    g = torch.Generator().manual_seed(6)
    f, _ = mx.rotary_frequencies(40)
    qkv = torch.randn(B, N, Hq + 2 * Hkv, d, generator=g).cuda()
    q = qkv[:, :, :Hq].transpose(1, 2).requires_grad_(True)
    k = qkv[:, :, Hq:Hq + Hkv].transpose(1, 2).requires_grad_(True)
    at = torch.randint(0, 5000, (N,), generator=g, dtype=torch.int32)
    dy = [torch.randn(B, h, N, d, generator=g).cuda() for h in (Hq, Hkv)]
    y = rotary_embedding(q, k, f, positions=at.cuda(), interleaved=interleaved, factor=1.5)
    dx = torch.autograd.grad(y, (q, k), dy)
    for got, up in zip(dx, dy):
        _check(got, up, at, f, interleaved, 1.5, -1.0)
    # <dy, R (x + e t) - R x> / e = <R^T dy, t>, exact for a linear map but for rounding
    t = torch.randn(q.shape, generator=g).cuda()
    with torch.no_grad():
        moved = rotary_embedding(q + t, k, f, positions=at.cuda(), interleaved=interleaved, factor=1.5)[0]
    lhs = ((moved - y[0]).double() * dy[0].double()).sum()
    rhs = (dx[0].double() * t.double()).sum()
    # B Hq N d products of values up to about 10, each off by a few 2^-24 of that, at random
    assert abs(float(lhs - rhs)) <= q.numel() ** 0.5 * 10 * 12 * 2.0 ** -24 * 4
    # a gradient broadcast by sum(), and one output unused
    y = rotary_embedding(q, k, f, interleaved=interleaved)
    dq, dk = torch.autograd.grad(y[0].sum(), (q, k), allow_unused=True)
    _check(dq, torch.ones_like(dq), torch.arange(N), f, interleaved, sign=-1.0)
    assert dk is None or not dk.any()


def test_second_gradient_and_the_python_node(monkeypatch):
    """The rotation is linear, so the gradient of its gradient is the rotation again;
    the Python node gives the C++ one's bits, gradients included."""
    from mx230_amd import autograd
    g = torch.Generator().manual_seed(16)
    f, _ = mx.rotary_frequencies(64)
    q, k = (torch.randn(1, h, 9, 64, generator=g).cuda().requires_grad_(True) for h in (3, 1))
    dy = [torch.randn(x.shape, generator=g).cuda().requires_grad_(True) for x in (q, k)]
    t = [torch.randn(x.shape, generator=g).cuda() for x in (q, k)]

    def go():
        y = autograd.rotary_embedding(q, k, f, pos0=7, factor=1.5)
        dx = torch.autograd.grad(y, (q, k), dy, create_graph=True)
        return (*y, *dx, *torch.autograd.grad(dx, dy, t))
    native = go()
    _check(native[4].detach(), t[0], torch.arange(7, 16), f, factor=1.5)
    monkeypatch.setattr(autograd, "_calls", lambda: mx._NoBinding)
    for a, b in zip(native, go()):
        assert torch.equal(a, b)
    # what the C++ node leaves: the error is the package's
    monkeypatch.undo()
    z = torch.zeros(1, 1, 2, 68, device="cuda")
    with pytest.raises(mx.MxfaError):
        autograd.rotary_embedding(z, z, f)
    with pytest.raises(ValueError):
        autograd.rotary_embedding(q, k, f, positions=torch.zeros(4, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        autograd.rotary_embedding(q, k[:, :, :5], f)
    # rows that are not on 16 bytes are copied
    odd = torch.randn(1, 3, 9, 65, generator=g).cuda()[..., 1:]
    y = autograd.rotary_embedding(odd, k, f)[0]
    _check(y, odd, torch.arange(9), f)


@pytest.mark.parametrize("bf16", [False, True])
def test_attention_block(bf16):
    """CausalSelfAttention with rotary positions against the same block made of
    plain operations in 64 bits, output and gradients."""
    from mx230_amd.autograd import CausalSelfAttention
    torch.manual_seed(7)
    dim, nh, nkv, hd, B, N = 128, 4, 2, 64, 2, 70
    f, a = mx.rotary_frequencies(hd, scaling="yarn", factor=4.0, original_length=32)
    m = CausalSelfAttention(dim, nh, nkv, hd, rotary=(f, a)).cuda()
    x = torch.randn(B, N, dim, device="cuda")
    dy = torch.randn(B, N, dim, device="cuda")
    if bf16:
        m, x, dy = m.bfloat16(), x.bfloat16(), dy.bfloat16()
    x.requires_grad_(True)
    y = m(x)
    got = [y, *torch.autograd.grad(y, (x, m.qkv.weight, m.out.weight), dy)]
    x64 = x.detach().cpu().double().requires_grad_(True)
    wq, wo = (w.detach().cpu().double().requires_grad_(True) for w in (m.qkv.weight, m.out.weight))
    q, k, v = (t.view(B, N, -1, hd).transpose(1, 2) for t in (x64 @ wq.T).split([nh * hd, nkv * hd, nkv * hd], -1))
    ang = torch.arange(N).double()[:, None] * f.cpu()
    c, s = a * ang.cos(), a * ang.sin()

    def turn(z):
        u, w = z[..., :hd // 2], z[..., hd // 2:]
        return torch.cat([u * c - w * s, w * c + u * s], -1)
    q, k = turn(q), turn(k).repeat_interleave(nh // nkv, 1)
    p = (q @ k.transpose(-1, -2) / hd ** 0.5).masked_fill(torch.ones(N, N).triu(1).bool(), float("-inf")).softmax(-1)
    y64 = (p @ v.repeat_interleave(nh // nkv, 1)).transpose(1, 2).reshape(B, N, nh * hd) @ wo.T
    want = [y64, *torch.autograd.grad(y64, (x64, wq, wo), dy.cpu().double())]
    for g, w in zip(got, want):
        off = (g.detach().cpu().double() - w.detach()).norm() / w.detach().norm()
        # norms over thousands of values: bf16 rounds at six places along the way
        # (2^-8 of each at most), fp32 sums of 128 at as many
        assert float(off) <= (6 * 2.0 ** -8 if bf16 else 6 * 128 * 2.0 ** -24), float(off)


def test_graph():
    """Captured, with its gradient, and replayed on new inputs with eager work between."""
    from mx230_amd.autograd import rotary_embedding
    torch.manual_seed(8)
    f, _ = mx.rotary_frequencies(64)
    q = torch.randn(1, 4, 50, 64, device="cuda").requires_grad_(True)
    k = torch.randn(1, 2, 50, 64, device="cuda").requires_grad_(True)
    dy = torch.randn_like(q), torch.randn_like(k)
    at = torch.arange(50, dtype=torch.int32, device="cuda")

    def step():
        y = rotary_embedding(q, k, f, positions=at)
        return (*y, *torch.autograd.grad(y, (q, k), dy))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for i in range(3):
        with torch.no_grad():
            for x in (q, k, *dy):
                x.copy_(torch.randn_like(x))
            at.add_(1000 * i)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
