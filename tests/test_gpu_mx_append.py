"""The append into a microscaled cache and the read out of it, against the format on the
CPU in 64 bits: codes and powers byte by byte, Q by the ordinary append's tolerance,
what is left as it was, borders between codes, and values that are not finite."""
from __future__ import annotations

import math

import pytest
import torch

import mx230_amd as mx
from cache_helpers import turned, turned_tolerance
from mx_helpers import MxBatch, block_bytes, levels, packed, parts, quantised, stands_for

pytestmark = pytest.mark.gpu

BITS = [8, 4]


def positions(b):
    """Each new token's position and sequence."""
    at, seq = [], []
    for s, (n, ln) in enumerate(b.pairs):
        at += list(range(ln - n, ln))
        seq += [s] * n
    return torch.tensor(at, dtype=torch.long), seq


def append(b, freq=None, interleaved=False, factor=1.0, inplace=False, seed=0, **kw):
    """q_out, kp, vp after the append over pools of noise, and the pools before it."""
    g = torch.Generator().manual_seed(seed)
    k0, v0 = (torch.randint(0, 256, b.kp.shape, generator=g, dtype=torch.uint8) for _ in range(2))
    kp, vp = k0.cuda(), v0.cuda()
    qkv, table, cu, lens = b.cuda("qkv", "table", "cu_q", "lens")
    out = qkv[:, :b.nh * b.hd] if inplace else torch.full((b.n_tok, b.nh * b.hd), 7.0, dtype=b.dt, device="cuda")
    print(f"\n[append mx] {b.pairs[:5]}.. heads {b.nh}/{b.nkv} d {b.hd} block {b.bs} bits {b.bits} {b.dt}", flush=True)
    mx.run_cache_append_mx(qkv, out, kp, vp, b.bits, table, b.bs, cu, lens, b.nh, b.nkv, b.hd,
                           frequencies=None if freq is None else freq.cuda(), interleaved=interleaved, factor=factor, **kw)
    torch.cuda.synchronize()
    return out.cpu(), kp.cpu(), vp.cpu(), k0, v0


def expected(b, k0, v0, freq=None, interleaved=False, factor=1.0):
    """Q in 64 bits and the pools."""
    at, seq = positions(b)
    n, nh, nkv, hd, bs = b.n_new, b.nh, b.nkv, b.hd, b.bs
    x = b.qkv[:n].view(n, nh + 2 * nkv, hd)
    y = x.double()
    if freq is not None:
        y = y.clone()
        y[:, :nh + nkv] = turned(x[:, :nh + nkv], at[:, None].expand(n, nh + nkv), freq, interleaved, factor)
    kp, vp = k0.clone(), v0.clone()
    for pool, part in ((kp, y[:, nh:nh + nkv]), (vp, y[:, nh + nkv:])):
        codes, E = parts(pool, nkv, bs, hd, b.bits)
        c, e = quantised(part, b.bits)
        for i in range(n):
            j = int(at[i]) // bs
            if at[i] < 0 or j >= b.table.shape[1] or not 0 <= int(b.table[seq[i], j]) < b.n_blocks:
                continue
            blk = int(b.table[seq[i], j])
            codes[blk, :, int(at[i]) % bs], E[blk, :, int(at[i]) % bs] = packed(c[i], b.bits), e[i].to(torch.uint8)
    return y[:, :nh], kp, vp


def check(b, got, freq=None, interleaved=False, factor=1.0):
    out, kp, vp, k0, v0 = got
    q, wk, wv = expected(b, k0, v0, freq, interleaved, factor)
    at, _ = positions(b)
    n, x = b.n_new, b.qkv[:b.n_new, :b.nh * b.hd].view(b.n_new, b.nh, b.hd)
    tol = torch.zeros_like(q) if freq is None else turned_tolerance(x, q, freq.numel(), interleaved, abs(factor))
    off = (out[:n].view(n, b.nh, b.hd).double() - q).abs()
    seen = at >= 0
    assert bool((off <= tol)[seen].all()), float((off - tol)[seen].max())
    for g, w in ((kp, wk), (vp, wv)):
        assert torch.equal(g, w), int((g != w).sum())
    return out


def freqs(dim, base=10000.0):
    return base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("hd", [64, 128, 32, 96, 224, 256])
def test_append(hd, bf16, bits):
    b = MxBatch([(1, 40), (5, 5), (0, 9), (70, 100), (1, 1)], 6, 2, hd, 16, bits, bf16, seed=hd, extra_rows=3)
    f = freqs(hd)
    out = check(b, append(b, f), f)
    assert bool((out[b.n_new:] == 7.0).all())
    check(b, append(b))


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("dim,interleaved", [(64, True), (32, False), (32, True), (24, False), (24, True), (2, False), (10, True), (62, False)])
def test_rotated_parts(dim, interleaved, bf16, bits):
    b = MxBatch([(3, 1000), (66, 400), (2, 2)], 4, 4, 64, 32, bits, bf16, seed=dim)
    f = freqs(dim, 500.0)
    check(b, append(b, f, interleaved, 1.25), f, interleaved, 1.25)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("bs", [1, 2, 8, 128])
def test_blocks(bs, bits):
    """Blocks of any power of two, whose bytes are no multiple of 16, in wider rows."""
    for nkv in (1, 3):
        b = MxBatch([(9, 20), (1, 130), (130, 131)], 3, nkv, 64, bs, bits, True, seed=bs, gap=32)
        f = freqs(64)
        check(b, append(b, f), f)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("hd", [64, 96, 224])
@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place(interleaved, hd, bits):
    """q_out may be qkv: rows of U threads that straddle no wave."""
    b = MxBatch([(90, 200), (1, 50), (77, 77)], 9, 3, hd, 16, bits, True, seed=hd)
    f = freqs(hd)
    check(b, append(b, f, interleaved, inplace=True), f, interleaved)


@pytest.mark.parametrize("bits", BITS)
def test_far_positions(bits):
    """Keys far on, whose angles 32 bits would lose; and a factor of 64 bits."""
    b = MxBatch([(40, 60)], 2, 2, 64, 16, bits, False, seed=1)
    far = 131072
    b.pairs = [(40, far)]
    b.lens = torch.tensor([far], dtype=torch.int32)
    b.table = torch.full((1, far // 16), -1, dtype=torch.int32)
    b.table[0, -4:] = torch.arange(4, dtype=torch.int32)
    f, factor = freqs(64), 0.1 * math.log(8.0) + 1.0
    check(b, append(b, f, factor=factor), f, factor=factor)


def rows_of(values, nkv, hd, bits, bf16):
    """A batch of one sequence whose V rows are `values` [n, hd]."""
    n = values.shape[0]
    b = MxBatch([(n, n)], nkv, nkv, hd, 16, bits, bf16, seed=0)
    b.qkv = torch.zeros(n, 3 * nkv * hd, dtype=b.dt)
    b.qkv[:, nkv * hd:2 * nkv * hd] = values.repeat(1, nkv).to(b.dt)
    b.qkv[:, 2 * nkv * hd:] = values.flip(1).repeat(1, nkv).to(b.dt)
    return b


@pytest.mark.parametrize("bits", BITS)
def test_borders(bits):
    """Values on the borders between codes, a step of 32 bits to either side of them, on
    the codes, at both signs and several powers; largest elements around the one that
    moves the power."""
    lv = levels(bits)
    mid = (lv[1:] + lv[:-1]) / 2
    v = torch.cat([lv, mid]).float()
    v = torch.cat([v, torch.nextafter(v, torch.full_like(v, 1e9)), torch.nextafter(v, torch.full_like(v, -1e9))])
    v = torch.cat([v, -v])
    top = 448.0 if bits == 8 else 7.0
    v = v[v.abs() <= top]
    v = torch.cat([v, torch.zeros(-v.numel() % 31)]).view(-1, 31)
    rows = [torch.cat([v, torch.full((v.shape[0], 1), top)], 1) * 2.0 ** k for k in (0, -3, 20, -100, 110)]
    for x in (top, top / 2, 6.0, 4.0, 448.0, 464.0, 1.75, 1.0):
        for y in (x, math.nextafter(x, 1e9), x * (1 + 2.0 ** -23), x * (1 - 2.0 ** -24)):
            r = torch.linspace(-y, y, 32, dtype=torch.float64).float()[None]
            rows += [r, r * 2.0 ** -50]
    x = torch.cat(rows)
    x = torch.cat([x, x.flip(0)], 1)
    b = rows_of(x, 1, 64, bits, False)
    check(b, append(b))


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("bf16", [True, False])
def test_sizes_and_what_is_not_finite(bf16, bits):
    """Zeros, the smallest and largest values of the type, and groups that hold an
    infinity or NaN: those alone read back as NaN."""
    g = torch.Generator().manual_seed(bits)
    x = torch.randn(48, 64, generator=g)
    x[0] = 0.0
    x[1, :32] = 0.0
    x[2] *= 1e-38
    x[3] *= 1e-44
    x[4] *= 1e37
    x[5] = torch.finfo(torch.bfloat16).max
    x[6, 0] = torch.finfo(torch.bfloat16).max
    x[7] = -0.0
    x[8, 3], x[9, 40], x[10, 63] = math.inf, -math.inf, math.nan
    x[11, 0], x[12, 31], x[13, 32] = math.nan, math.inf, math.nan
    x[14] *= 2.0 ** -110
    b = rows_of(x, 2, 64, bits, bf16)
    out, kp, vp, k0, v0 = append(b)
    _, wk, wv = expected(b, k0, v0)
    assert torch.equal(kp, wk) and torch.equal(vp, wv)
    table, cu, lens = b.cuda("table", "cu_q", "lens")
    ko, vo = (torch.zeros(48, 128, dtype=b.dt, device="cuda") for _ in range(2))
    mx.run_cache_read_mx(kp.cuda(), vp.cuda(), bits, ko, vo, table, 16, cu, lens, 2, 64)
    for got, want in ((ko, b.qkv[:, 128:256]), (vo, b.qkv[:, 256:])):
        c, e = quantised(want.unflatten(1, (2, 64)), bits)
        w = stands_for(c, e, bits).flatten(1)
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(w)) and int(torch.isnan(w).sum()) == 6 * 32 * 2
        assert torch.equal(got.cpu().double().nan_to_num(), w.nan_to_num())
        # off by half a step at most: of the code's, or of the smallest code (from what
        # is above 1.75 2^127 counts as)
        fine = torch.isfinite(w)
        x64 = want.double().clamp(-1.75 * 2.0 ** 127, 1.75 * 2.0 ** 127)
        power = torch.exp2(e.double() - 127).repeat_interleave(32, -1).flatten(1)
        step = 2.0 ** -4 * x64.abs() if bits == 8 else torch.zeros_like(x64)
        step = torch.maximum(step, power * (2.0 ** -10 if bits == 8 else 0.25))
        if bits == 4:
            step = torch.maximum(step, torch.where(x64.abs() > 4 * power, power, torch.where(x64.abs() > 2 * power, power / 2, step)))
        assert bool(((w - x64).abs() <= step)[fine].all())


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("hd,bs", [(64, 16), (128, 16), (32, 1), (96, 8), (256, 128)])
def test_read(hd, bs, bf16, bits):
    """Whole sequences and their last rows; rows of no position stay."""
    pairs = [(1, 40), (5, 5), (0, 9), (70, 300), (3, 1)]
    b = MxBatch(pairs, 3, 3, hd, bs, bits, bf16, seed=hd, gap=16)
    kp, vp, table, lens = b.cuda("kp", "vp", "table", "lens")
    for counts in ([n for n, _ in pairs], [max(ln, 0) for _, ln in pairs]):
        cu = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
        n = int(cu[-1])
        wide = torch.full((n + 2, 2 * 3 * hd + 32), 7.0, dtype=b.dt, device="cuda")
        ko, vo = wide[:, :3 * hd], wide[:, 3 * hd + 16:6 * hd + 16]  # columns of the same rows
        print(f"\n[read mx] d {hd} block {bs} bits {bits} {b.dt} rows {n}", flush=True)
        mx.run_cache_read_mx(kp, vp, bits, ko, vo, table, bs, cu.cuda(), lens, 3, hd)
        got = wide.cpu()
        r = 0
        for s, c in enumerate(counts):
            for i in range(c):
                at = pairs[s][1] - c + i
                row = got[r]
                if at < 0:
                    assert bool((row == 7.0).all())
                else:
                    src = int(b.rows[s][at])
                    assert torch.equal(row[:3 * hd], b.k[src]) and torch.equal(row[3 * hd + 16:6 * hd + 16], b.v[src])
                    assert bool((row[3 * hd:3 * hd + 16] == 7.0).all()) and bool((row[6 * hd + 16:] == 7.0).all())
                r += 1
        assert bool((got[n:] == 7.0).all())


@pytest.mark.parametrize("bits", BITS)
def test_positions_and_blocks_that_are_not_there(bits):
    """Tokens at negative positions, past the table, in blocks outside the pool: left
    out, the append's Q but for the first written; nothing else is touched."""
    b = MxBatch([(4, 2), (40, 100), (3, 60)], 2, 2, 64, 16, bits, True, seed=4)
    b.table[1, 4], b.table[2, 3] = -1, b.n_blocks
    b.table = b.table[:, :6].contiguous()  # positions 96 .. 99 of the second are past it
    f = freqs(64)
    out = check(b, append(b, f), f)
    assert bool((out[:2] == 7.0).all()) and not bool((out[2:b.n_new] == 7.0).all(1).any())
    kp, vp, table, cu, lens = b.cuda("kp", "vp", "table", "cu_q", "lens")
    ko, vo = (torch.full((b.n_tok, 128), 7.0, dtype=b.dt, device="cuda") for _ in range(2))
    mx.run_cache_read_mx(kp, vp, bits, ko, vo, table, 16, cu, lens, 2, 64)
    at, seq = positions(b)
    for i in range(b.n_new):
        j = int(at[i]) // 16
        there = at[i] >= 0 and j < 6 and 0 <= int(b.table[seq[i], j]) < b.n_blocks
        assert bool((ko[i] == 7.0).all()) != bool(there)


def test_offsets_past_32_bits():
    """A block more than 4 GiB into the pools."""
    bs, nkv, hd, bits = 16, 8, 128, 8
    wide = block_bytes(bs, nkv, hd, bits)
    n_blocks = (1 << 32) // wide + 3
    pools = [torch.zeros(n_blocks, wide, dtype=torch.uint8, device="cuda") for _ in range(2)]
    b = MxBatch([(20, 20)], 8, nkv, hd, bs, bits, True, seed=2)
    table = torch.tensor([[n_blocks - 1, n_blocks - 2]], dtype=torch.int32, device="cuda")
    qkv, cu, lens = b.cuda("qkv", "cu_q", "lens")
    out = torch.empty(20, nkv * hd, dtype=b.dt, device="cuda")
    print("\n[append mx] past 4 GiB", flush=True)
    mx.run_cache_append_mx(qkv, out, *pools, bits, table, bs, cu, lens, 8, nkv, hd)
    ko, vo = torch.empty_like(out), torch.empty_like(out)
    mx.run_cache_read_mx(*pools, bits, ko, vo, table, bs, cu, lens, nkv, hd)
    for got, x in ((ko, qkv[:, nkv * hd:2 * nkv * hd]), (vo, qkv[:, 2 * nkv * hd:])):
        c, e = quantised(x.cpu().unflatten(1, (nkv, hd)), bits)
        assert torch.equal(got.cpu().double(), stands_for(c, e, bits).flatten(1))
    assert not any(bool(p[:n_blocks - 2].any()) for p in pools)
