"""Attention over a microscaled cache against 64-bit attention over the values that its
codes stand for: lengths around the stages and units, single tokens and chunks side by
side, split sequences, grouped heads, rows that see nothing, and what stands in
positions that a row does not see."""
from __future__ import annotations

import math

import pytest
import torch

import mx230_amd as mx
from mx_helpers import MxBatch, parts

pytestmark = pytest.mark.gpu

TYPES = [(True, 64, 8), (True, 64, 4), (True, 128, 8), (True, 128, 4), (False, 64, 8), (False, 64, 4)]


def run(b, lse=True, max_q=None, fill=7.0, **kw):
    k, v, table, cu, lens, qkv = b.cuda("kp", "vp", "table", "cu_q", "lens", "qkv")
    out = torch.full((b.n_tok, b.nh * b.hd), fill, dtype=b.dt, device="cuda")
    e = torch.full((b.n_tok, b.nh), fill, device="cuda") if lse else None
    print(f"\n[prefill batch mx] {b.pairs[:6]}.. heads {b.nh}/{b.nkv} d {b.hd} block {b.bs} bits {b.bits} {b.dt}", flush=True)
    mx.run_prefill_batch_mx(qkv[:, :b.nh * b.hd], k, v, b.bits, out, table, b.bs, cu, lens, max_q or b.max_q, b.nh, b.nkv,
                            b.hd, lse=e, **kw)
    torch.cuda.synchronize()
    return out.cpu(), None if e is None else e.cpu()


def check(b, out, lse, scale=None):
    want, mag, wlse, reach = b.attention(scale)
    mine = slice(0, b.n_new)
    off = (out[mine].double() - want[mine]).abs()
    tol = b.tolerance(want, mag, reach)[mine]
    assert bool((off <= tol).all()), (float((off - tol).max()), float(off.max()))
    if lse is not None:
        fin = torch.isfinite(wlse[mine])
        assert torch.equal(lse[mine][~fin].double(), wlse[mine][~fin])
        off = (lse[mine].double() - wlse[mine])[fin].abs()
        assert float(off.max() if off.numel() else 0.0) <= b.lse_tolerance(reach)
    assert bool((out[b.n_new:] == 7.0).all()) and (lse is None or bool((lse[b.n_new:] == 7.0).all()))


@pytest.mark.parametrize("bf16,hd,bits", TYPES)
@pytest.mark.parametrize("bs", [1, 16, 128])
@pytest.mark.parametrize("pairs", [
    [(1, 1)], [(1, 63), (1, 64), (1, 65)], [(1, 700), (1, 1), (1, 513), (1, 128)], [(2, 2), (3, 700), (1, 90)],
    [(64, 64)], [(65, 65), (1, 200), (63, 127), (5, 5)], [(17, 300), (16, 81), (1, 1025)], [(130, 1000)]])
def test_lengths(pairs, bs, bf16, hd, bits):
    b = MxBatch(pairs, 4, 2, hd, bs, bits, bf16, seed=len(pairs) + bs)
    check(b, *run(b))


@pytest.mark.parametrize("bf16,hd,bits", TYPES)
@pytest.mark.parametrize("nh,nkv", [(1, 1), (7, 1), (14, 2), (16, 1), (17, 1), (40, 1), (6, 6), (9, 3)])
def test_heads(nh, nkv, bf16, hd, bits):
    b = MxBatch([(1, 150), (3, 70), (30, 95), (1, 64)], nh, nkv, hd, 16, bits, bf16, seed=nh, gap=48)
    check(b, *run(b))


@pytest.mark.parametrize("bf16,hd,bits", TYPES)
@pytest.mark.parametrize("pairs", [
    [(1, 9000)], [(1, 5000), (1, 3), (1, 2500), (0, 0), (1, 4097)], [(70, 6000)], [(40, 5000), (1, 4500), (2, 30), (33, 33)]])
def test_split_over_keys(pairs, bf16, hd, bits):
    b = MxBatch(pairs, 2, 1, hd, 16, bits, bf16, seed=len(pairs))
    out, lse = run(b)
    check(b, out, lse)
    again, lse2 = run(b)
    assert torch.equal(out, again) and torch.equal(lse, lse2)  # equal calls, equal bits


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("pairs,nh,nkv,hd", [
    ([(400, 1500)], 14, 2, 64), ([(350, 900), (64, 2000)], 14, 2, 64),    # units of 64 rows
    ([(900, 1100)] * 4 + [(1, 40)], 14, 2, 64),                          # of 128
    ([(1100, 1200)], 4, 1, 128), ([(600, 700)] * 2, 32, 4, 128),
    ([(129, 1400), (1, 3000), (1, 200), (1, 64)], 14, 2, 64)])           # beside few rows
def test_unit_sizes(pairs, nh, nkv, hd, bits):
    b = MxBatch(pairs, nh, nkv, hd, 16, bits, True, seed=hd)
    check(b, *run(b))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n_seq", [63, 130])
def test_many_sequences(n_seq, bits):
    g = torch.Generator().manual_seed(n_seq)
    pairs = [(int(n), int(n) + int(x)) for n, x in zip(torch.randint(0, 4, (n_seq,), generator=g),
                                                       torch.randint(0, 150, (n_seq,), generator=g))]
    pairs[n_seq - 1] = (20, 333)
    pairs[n_seq // 2] = (1, 3000)
    b = MxBatch(pairs, 4, 2, 64, 16, bits, True, seed=n_seq)
    check(b, *run(b))


@pytest.mark.parametrize("bf16,hd,bits", TYPES)
@pytest.mark.parametrize("bs", [4, 64])
def test_short_sequences_in_one_run(bs, bf16, hd, bits):
    """Some ten sequences to a work-group, of fewer stages than it has waves and of more,
    of none, and of one whose K is NaN: the others' bits stay."""
    g = torch.Generator().manual_seed(bs)
    lens = torch.randint(0, 9, (300,), generator=g) ** 3 + torch.randint(0, 90, (300,), generator=g)
    pairs = [(1 + i % 2, max(int(n), 1 + i % 2)) if i % 7 else (1, 0) for i, n in enumerate(lens)]
    b = MxBatch(pairs, 16, 8, hd, bs, bits, bf16, seed=bs)
    out, lse = run(b)
    check(b, out, lse)
    # (the 150th, KV head 3, its first token)
    ke = parts(b.kp, 8, bs, hd, bits)[1]
    at = int(b.rows[150][0])
    ke[at // bs, 3, at % bs] = 255
    got, lse2 = run(b)
    t0 = sum(n for n, _ in pairs[:150])
    hit = torch.zeros(out.shape, dtype=torch.bool)
    hit[t0:t0 + pairs[150][0], 6 * hd:8 * hd] = True
    assert bool(torch.isnan(got[hit]).all()) and torch.equal(got[~hit], out[~hit])


@pytest.mark.parametrize("bf16,hd,bits", TYPES)
def test_rows_that_see_nothing(bf16, hd, bits):
    b = MxBatch([(0, 50), (3, 0), (5, 2), (0, 0), (40, 10), (2, 90)], 4, 2, hd, 16, bits, bf16, seed=3, extra_rows=6, wide=3)
    out, lse = run(b)
    check(b, out, lse)
    assert not out[0:3].any() and not out[3:6].any() and bool(out[6:8].any())


@pytest.mark.parametrize("bf16,hd,bits", TYPES)
def test_values_a_row_does_not_see(bf16, hd, bits):
    """A group of a later token that is NaN by its power, or by a code of 8 bits, reaches
    no earlier row; those it does reach are NaN."""
    for pairs in ([(4, 40), (80, 100)], [(40, 3000), (3, 2900)]):
        for by_code in ((False, True) if bits == 8 else (False,)):
            b = MxBatch(pairs, 4, 2, hd, 16, bits, bf16, seed=11)
            clean, lse0 = run(b)
            kc, ke = parts(b.kp, 2, 16, hd, bits)
            vc, ve = parts(b.vp, 2, 16, hd, bits)
            for s, (n, ln) in enumerate(pairs):
                last, one = int(b.rows[s][ln - 1]), int(b.rows[s][ln - 2])
                if by_code:
                    vc[one // 16, 0, one % 16], kc[last // 16, 1, last % 16] = 0x7f, 0xff
                else:  # the last token but one, first KV head; the last, second
                    ve[one // 16, 0, one % 16], ke[last // 16, 1, last % 16] = 255, 255
            out, lse = run(b)
            t0 = 0
            for n, ln in pairs:
                for h in range(4):
                    c = slice(h * hd, (h + 1) * hd)
                    fine = n - 2 if h < 2 else n - 1
                    got, had = out[t0:t0 + fine, c].double(), clean[t0:t0 + fine, c].double()
                    assert bool(torch.isfinite(got).all())
                    assert float((got - had).abs().max()) <= 2.0 ** -6 * float(had.abs().max())
                    assert float((lse[t0:t0 + fine, h] - lse0[t0:t0 + fine, h]).abs().max()) <= 1e-3
                    assert bool(torch.isnan(out[t0 + fine:t0 + n, c]).all())
                t0 += n


@pytest.mark.parametrize("bf16,hd,bits", TYPES)
def test_large_scores(bf16, hd, bits):
    """Scores of some hundreds, rising along the keys."""
    pairs = [(1, 900), (40, 700), (2, 300)]
    b = MxBatch(pairs, 4, 2, hd, 16, bits, bf16, seed=5)
    for s, (_, ln) in enumerate(pairs):
        rise = torch.linspace(0.2, 6.0, ln, dtype=torch.float64)[:, None]
        b.k[b.rows[s]] = (b.k[b.rows[s]].double() * rise).to(b.dt)
    b.again()
    b.qkv[:, :4 * hd] *= 4
    check(b, *run(b))


@pytest.mark.parametrize("bf16,hd,bits", TYPES)
@pytest.mark.parametrize("size", [1e-34, 1e-20, 1e20])
def test_sizes_of_v(size, bf16, hd, bits):
    """Values far from one: the result is as exact relative to them."""
    b = MxBatch([(1, 700), (33, 200)], 4, 2, hd, 16, bits, bf16, seed=6)
    b.v = (b.v.double() * size).to(b.dt)
    b.vp, b.v = b.pool(b.v)
    out, _ = run(b)
    want, mag, _, reach = b.attention()
    tol = b.tolerance(want, mag, reach) - 1e-30 + 1e-42
    assert bool(((out.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("bf16,hd,bits", TYPES)
def test_scale_max_q_and_strides(bf16, hd, bits):
    """A scale of its own; rows past max_q stay; out in other columns of q's rows."""
    b = MxBatch([(5, 200), (20, 64), (1, 64)], 4, 2, hd, 16, bits, bf16, seed=7)
    check(b, *run(b, scale=0.3), scale=0.3)
    out, lse = run(b, max_q=3)
    full, _ = run(b)
    assert bool((out[3:5] == 7.0).all()) and bool((out[8:25] == 7.0).all()) and bool((lse[8:25] == 7.0).all())
    kp, vp, table, cu, lens, qkv = b.cuda("kp", "vp", "table", "cu_q", "lens", "qkv")
    w = 4 * hd
    wide = torch.full((b.n_tok, 2 * w + 16), 7.0, dtype=b.dt, device="cuda")
    wide[:, :w] = qkv[:, :w]
    mx.run_prefill_batch_mx(wide[:, :w], kp, vp, bits, wide[:, w:2 * w], table, 16, cu, lens, 20, 4, 2, hd)
    assert torch.equal(wide[:, w:2 * w].cpu(), full) and bool((wide[:, 2 * w:] == 7.0).all())
    mx.run_prefill_batch_mx(wide[:, :w], kp, vp, bits, wide[:, :w], table, 16, cu, lens, 20, 4, 2, hd)
    assert torch.equal(wide[:, :w].cpu(), full)
