"""Attention of a batch of sequences over a paged cache (mxfa_run_prefill_batch) against
64-bit attention of each sequence by itself: lengths around the kernels' 64-key
stages and 16- and 64-row units, single tokens and chunks side by side, long
sequences whose keys are split, grouped heads, empty sequences and rows that see
nothing, and what stands in blocks, rows and positions that are not a
sequence's."""
from __future__ import annotations

import math
import random

import pytest
import torch

import mx230_amd as mx
from cache_helpers import Batch

pytestmark = pytest.mark.gpu


def run(b, lse=True, max_q=None, q=None, fill=7.0, **kw):
    k, v, table, cu, lens, qkv = b.cuda("k", "v", "table", "cu_q", "lens", "qkv")
    q = qkv[:, :b.nh * b.hd] if q is None else q
    out = torch.full((b.n_tok, b.nh * b.hd), fill, dtype=b.dt, device="cuda")
    e = torch.full((b.n_tok, b.nh), fill, device="cuda") if lse else None
    print(f"\n[prefill batch] {b.pairs[:6]}.. heads {b.nh}/{b.nkv} d {b.hd} block {b.bs} {b.dt}", flush=True)
    mx.run_prefill_batch(q, k, v, out, table, b.bs, cu, lens, max_q or b.max_q, b.nh, b.nkv, b.hd, lse=e, **kw)
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
    # rows of no sequence stay as they were
    assert bool((out[b.n_new:] == 7.0).all()) and (lse is None or bool((lse[b.n_new:] == 7.0).all()))


TYPES = [(True, 64), (True, 128), (False, 64)]


@pytest.mark.parametrize("bf16,hd", TYPES)
@pytest.mark.parametrize("bs", [1, 16, 128])
@pytest.mark.parametrize("pairs", [
    [(1, 1)], [(1, 63), (1, 64), (1, 65)], [(1, 700), (1, 1), (1, 513), (1, 128)], [(2, 2), (3, 700), (1, 90)],
    [(64, 64)], [(65, 65), (1, 200), (63, 127), (5, 5)], [(17, 300), (16, 81), (1, 1025)], [(130, 1000)]])
def test_lengths(pairs, bs, bf16, hd):
    b = Batch(pairs, 4, 2, hd, bs, bf16, seed=len(pairs) + bs)
    check(b, *run(b))


@pytest.mark.parametrize("bf16,hd", TYPES)
@pytest.mark.parametrize("nh,nkv", [(1, 1), (7, 1), (14, 2), (16, 1), (17, 1), (40, 1), (6, 6), (9, 3)])
def test_heads(nh, nkv, bf16, hd):
    """Groups that fill a 16-row tile, pass it, and do not divide it; a token's heads
    may span units."""
    b = Batch([(1, 150), (3, 70), (30, 95), (1, 64)], nh, nkv, hd, 16, bf16, seed=nh)
    check(b, *run(b))


@pytest.mark.parametrize("bf16,hd", TYPES)
@pytest.mark.parametrize("pairs", [
    [(1, 9000)], [(1, 5000), (1, 3), (1, 2500), (0, 0), (1, 4097)], [(70, 6000)], [(40, 5000), (1, 4500), (2, 30), (33, 33)]])
def test_split_over_keys(pairs, bf16, hd):
    """Lengths whose keys are split and joined."""
    b = Batch(pairs, 2, 1, hd, 16, bf16, seed=len(pairs))
    out, lse = run(b)
    check(b, out, lse)
    again, lse2 = run(b)
    assert torch.equal(out, again) and torch.equal(lse, lse2)  # equal calls, equal bits


@pytest.mark.parametrize("pairs", [[(1000, 1000)] * 4, [(600, 900), (777, 1000)] * 2, [(900, 1010)] * 5])
def test_more_units_than_cus_that_stay_whole(pairs):
    """Tables too short for any split: a launch of more work-groups than CUs, in the
    order that balances those a CU holds, has them all."""
    b = Batch(pairs, 14, 2, 64, 16, True, seed=len(pairs))
    check(b, *run(b))


@pytest.mark.parametrize("pairs,nh,nkv,hd", [
    ([(400, 1500)], 14, 2, 64), ([(350, 900), (64, 2000)], 14, 2, 64),    # units of 64 rows
    ([(900, 1100)] * 4 + [(1, 40)], 14, 2, 64),                          # of 128
    ([(1100, 1200)], 4, 1, 128), ([(600, 700)] * 2, 32, 4, 128),
    ([(129, 1400), (1, 3000), (1, 200), (1, 64)], 14, 2, 64)])           # beside few rows
def test_unit_sizes(pairs, nh, nkv, hd):
    b = Batch(pairs, nh, nkv, hd, 16, True, seed=hd)
    check(b, *run(b))


@pytest.mark.parametrize("n_seq", [63, 64, 65, 130])
def test_many_sequences(n_seq):
    """More sequences than a wave's lanes, some without new tokens."""
    g = torch.Generator().manual_seed(n_seq)
    pairs = [(int(n), int(n) + int(x)) for n, x in zip(torch.randint(0, 4, (n_seq,), generator=g),
                                                       torch.randint(0, 150, (n_seq,), generator=g))]
    pairs[n_seq - 1] = (20, 333)
    pairs[n_seq // 2] = (1, 3000)
    b = Batch(pairs, 4, 2, 64, 16, True, seed=n_seq)
    check(b, *run(b))


@pytest.mark.parametrize("bf16,hd", TYPES)
def test_rows_that_see_nothing(bf16, hd):
    """Sequences without new tokens or without positions, tokens at negative
    positions (zeros, lse -inf), rows behind the last sequence."""
    b = Batch([(0, 50), (3, 0), (5, 2), (0, 0), (40, 10), (2, 90)], 4, 2, hd, 16, bf16, seed=3, extra_rows=6, wide=3)
    out, lse = run(b)
    check(b, out, lse)
    assert not out[0:3].any() and not out[3:6].any() and bool(out[6:8].any())


@pytest.mark.parametrize("bf16,hd", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_a_row_does_not_see(bad, bf16, hd):
    """An infinity or NaN in a later token's K or V reaches no earlier row, single
    tokens' and chunks', split over keys or not; those it does reach are not
    finite."""
    for pairs in ([(4, 40), (80, 100)], [(40, 3000), (3, 2900)]):
        b = Batch(pairs, 4, 2, hd, 16, bf16, seed=11)
        clean, lse0 = run(b)
        for s, (n, ln) in enumerate(pairs):
            b.v[b.rows[s][ln - 2], :hd] = bad           # the last token but one, first KV head
            b.k[b.rows[s][ln - 1], hd:] = math.nan      # the last, second KV head
        out, lse = run(b)
        t0 = 0
        for n, ln in pairs:
            for h in range(4):
                c = slice(h * hd, (h + 1) * hd)
                fine = n - 2 if h < 2 else n - 1
                got, had = out[t0:t0 + fine, c].double(), clean[t0:t0 + fine, c].double()
                # the plain arithmetic's rounding instead of the matrix products'
                assert bool(torch.isfinite(got).all()) and float((got - had).abs().max()) <= 2.0 ** -6 * float(had.abs().max())
                assert float((lse[t0:t0 + fine, h] - lse0[t0:t0 + fine, h]).abs().max()) <= 1e-3
                assert not bool(torch.isfinite(out[t0 + fine:t0 + n, c]).any())
            t0 += n


@pytest.mark.parametrize("bf16,hd", TYPES)
def test_large_scores(bf16, hd):
    """Scores of some hundreds, rising along the keys: one weight takes a row, and
    the running maximum moves at every stage."""
    b = Batch([(1, 700), (50, 400)], 2, 1, hd, 16, bf16, seed=12)
    for s, (n, ln) in enumerate(b.pairs):
        ramp = torch.linspace(0.1, 40.0, ln)[:, None]
        b.k[b.rows[s]] = (b.k[b.rows[s]].float() * ramp).to(b.dt)
    check(b, *run(b))
    b = Batch([(1, 700), (50, 400)], 2, 1, hd, 16, bf16, seed=13)
    check(b, *run(b, scale=1e-6), scale=1e-6)


def test_strides_and_shared_rows():
    """Wider cache, query, output and table rows than needed; one table row for two
    sequences (a shared prefix); a table wider than the longest sequence."""
    nh, nkv, hd, bs = 4, 2, 64, 16
    b = Batch([(3, 100), (2, 77)], nh, nkv, hd, bs, True, seed=14, wide=2)
    b.lens[1], b.pairs = 99, [(3, 100), (2, 99)]
    b.table[1], b.rows[1] = b.table[0], b.rows[0][:99]
    wide = torch.full((b.k.shape[0], 2 * nkv * hd + 8), math.nan, dtype=b.dt)
    wide[:, :nkv * hd], wide[:, nkv * hd:2 * nkv * hd] = b.k, b.v
    w = wide.cuda()
    out = torch.full((b.n_tok, nh * hd + 24), 7.0, dtype=b.dt, device="cuda")
    table = torch.full((2, b.table.shape[1] + 5), 10 ** 6, dtype=torch.int32)
    table[:, :b.table.shape[1]] = b.table
    tab = table.cuda()[:, :b.table.shape[1]]
    qkv, cu, lens = b.cuda("qkv", "cu_q", "lens")
    ws = torch.empty(mx.prefill_batch_workspace_bytes(b.n_tok, 2, 3, nh, nkv, hd), dtype=torch.uint8, device="cuda")
    got = mx.run_prefill_batch(qkv[:, :nh * hd], w[:, :nkv * hd], w[:, nkv * hd:2 * nkv * hd], out, tab, bs, cu, lens, 3,
                               nh, nkv, hd, workspace=ws)
    assert got is ws
    torch.cuda.synchronize()
    check(b, out[:, :nh * hd].cpu(), None)
    assert bool((out[:, nh * hd:] == 7.0).all())
    far = torch.zeros(2, 1000, dtype=torch.int32, device="cuda")  # a table whose sequences may be split
    with pytest.raises(mx.MxfaError):
        mx.run_prefill_batch(qkv[:, :nh * hd], w[:, :nkv * hd], w[:, nkv * hd:2 * nkv * hd], out, far, bs, cu, lens, 3,
                             nh, nkv, hd, workspace=ws[:256])
    with pytest.raises(ValueError):
        mx.run_prefill_batch(qkv[:, :nh * hd], w[:, :nkv * hd], w[:, nkv * hd:2 * nkv * hd], out, tab[:1], bs, cu, lens,
                             3, nh, nkv, hd)


@pytest.mark.parametrize("pairs", [[(1, 900), (3, 5000), (1, 1)], [(150, 4000), (1, 3000), (200, 200)], [(90, 90)]])
def test_output_over_the_queries(pairs):
    b = Batch(pairs, 14, 2, 64, 16, True, seed=len(pairs))
    k, v, table, cu, lens, qkv = b.cuda("k", "v", "table", "cu_q", "lens", "qkv")
    q = qkv[:, :b.nh * b.hd].clone()
    out, _ = run(b, lse=False)
    mx.run_prefill_batch(q, k, v, q, table, b.bs, cu, lens, b.max_q, b.nh, b.nkv, b.hd)
    torch.cuda.synchronize()
    assert torch.equal(q[:b.n_new].cpu(), out[:b.n_new])


def test_numbers_past_32_bits():
    b = Batch([(1, 9)], 4, 2, 64, 16, True, seed=1)
    k, v, table, cu, lens, qkv = b.cuda("k", "v", "table", "cu_q", "lens", "qkv")
    out = torch.empty(b.n_tok, b.nh * b.hd, dtype=b.dt, device="cuda")
    for kw in (dict(max_q=2 ** 32 + 1), dict(block_size=2 ** 32 + 16), dict(n_head=2 ** 32 + 4)):
        a = dict(block_table=table, block_size=b.bs, cu_q=cu, lens=lens, max_q=1, n_head=b.nh, n_kv_head=b.nkv, head_dim=b.hd)
        with pytest.raises(ValueError, match="past 32 bits"):
            mx.run_prefill_batch(qkv[:, :b.nh * b.hd], k, v, out, **(a | kw))
    f, _ = mx.rotary_frequencies(64)
    x = torch.zeros(1, 2, 3, 64, device="cuda")
    with pytest.raises(ValueError, match="past 32 bits"):
        mx.run_rotary(x, None, x, None, f, pos0=2 ** 32)


@pytest.mark.parametrize("fill", [0, 1, 0x7f, 0xff])
@pytest.mark.parametrize("pairs", [[(1, 5000), (1, 70), (2, 2500)], [(200, 4000), (1, 3000), (1, 9), (1, 6000)], [(300, 5000)],
                                   [(1, 3000)] * 3 + [(0, 0)]])
def test_what_the_workspace_holds_before(pairs, fill):
    """Whatever it is, notes of another call among it: outputs are those of a fresh one."""
    b = Batch(pairs, 14, 2, 64, 16, True, seed=len(pairs))
    other = Batch([(120, 6000), (1, 5000), (1, 40)], 14, 2, 64, 16, True, seed=5)
    n = max(mx.prefill_batch_workspace_bytes(x.n_tok, len(x.pairs), 300, 14, 2, 64) for x in (b, other))
    ws = torch.full((n,), fill, dtype=torch.uint8, device="cuda")
    got, glse = run(b, max_q=300, workspace=ws)
    want, wlse = run(b, max_q=300)
    check(b, got, glse)
    assert torch.equal(got, want) and torch.equal(glse, wlse)
    run(other, max_q=300, workspace=ws)
    again, _ = run(b, max_q=300, workspace=ws)
    assert torch.equal(again, want)


def test_hundreds_of_sequences():
    r = random.Random(4)
    pairs = [(n, r.randint(max(n, 1), 700)) for n in (r.choice([0, 1, 1, 1, 1, 2, 40]) for _ in range(700))]
    b = Batch(pairs, 4, 2, 64, 16, True, seed=3)
    check(b, *run(b))


def test_max_q_bounds_the_rows():
    """Rows of a sequence past max_q are left as they were."""
    b = Batch([(6, 100), (2, 30)], 4, 2, 64, 16, True, seed=15)
    out, lse = run(b, max_q=4)
    whole, _ = run(b)
    assert torch.equal(out[:4], whole[:4]) and torch.equal(out[6:], whole[6:]) and bool((out[4:6] == 7.0).all())


def test_tables_and_lengths_that_are_wrong():
    """Blocks outside the pool, lengths past the table and rows past q: nothing
    outside the buffers is touched, and the other sequences are as ever."""
    b = Batch([(2, 100), (3, 60), (2, 90)], 4, 2, 64, 16, True, seed=16, wide=1, extra_rows=2)
    want, _ = run(b)
    b.table[1, :2] = torch.tensor([-5, 2 ** 31 - 1], dtype=torch.int32)
    b.lens[1] = 2 ** 31 - 1
    out, _ = run(b)
    assert torch.equal(out[:2], want[:2]) and torch.equal(out[5:], want[5:])
    b.lens[1] = -7
    out, _ = run(b)
    assert torch.equal(out[:2], want[:2]) and not out[2:5].any()
    b.cu_q[3] = 2 ** 30  # a last sequence that says it has more rows than q
    run(b, max_q=2 ** 30)
    b.cu_q[1:3] = torch.tensor([-9, 4])
    run(b)


def test_python_path_stream_and_two_streams():
    """The Python path on a stream of its own gives the same bits, and so do two calls
    at once on two streams with a workspace each."""
    b = Batch([(1, 4000), (1, 300), (40, 2500)], 4, 2, 64, 16, True, seed=17)
    want, wl = run(b)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    k, v, table, cu, lens, qkv = b.cuda("k", "v", "table", "cu_q", "lens", "qkv")
    outs = [torch.zeros(b.n_tok, b.nh * b.hd, dtype=b.dt, device="cuda") for _ in range(6)]
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        mx.run_prefill_batch(qkv[:, :b.nh * b.hd], k, v, o, table, b.bs, cu, lens, 40, b.nh, b.nkv, b.hd,
                             stream=(s1, s2)[i % 2])
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o.cpu(), want)


def test_graph_follows_the_lengths():
    """A captured call replayed while lengths, tables and tokens change, with eager
    work between; two graphs on one workspace, replayed in turn."""
    b = Batch([(1, 2000), (2, 150), (30, 900)], 4, 2, 64, 16, True, seed=18, wide=4)
    k, v, table, cu, lens, qkv = b.cuda("k", "v", "table", "cu_q", "lens", "qkv")
    ws = torch.empty(mx.prefill_batch_workspace_bytes(b.n_tok, 3, 30, 4, 2, 64), dtype=torch.uint8, device="cuda")
    outs = [torch.zeros(b.n_tok, 256, dtype=b.dt, device="cuda") for _ in range(3)]

    def call(o, w):
        mx.run_prefill_batch(qkv[:, :256], k, v, o, table, 16, cu, lens, 30, 4, 2, 64, workspace=w)
    call(outs[0], ws)
    torch.cuda.synchronize()
    graphs = []
    for o in outs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(o, ws)
        graphs.append(g)
    for step in range(3):
        lens.sub_(37 * step)
        qkv.mul_(-0.5)
        for o in outs:
            o.zero_()
        for g in graphs:
            g.replay()
        call(outs[2], None)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[2]) and bool(outs[2].any())


def test_same_as_the_single_sequence_prefill():
    """One sequence: what run_prefill_paged gives, to rounding."""
    b = Batch([(100, 500)], 14, 2, 64, 16, True, seed=19)
    out, _ = run(b)
    k, v, table, qkv = b.cuda("k", "v", "table", "qkv")
    one = torch.empty(100, 14 * 64, dtype=b.dt, device="cuda")
    mx.run_prefill_paged(qkv[:, :14 * 64], k, v, one, table[0], 16, 400, 14, 2, 64)
    want, mag, _, reach = b.attention()
    assert bool(((one.cpu().double() - out.double()).abs() <= 2 * b.tolerance(want, mag, reach)).all())


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes (and 2^31 elements) whose far end is used."""
    nkv, hd, bs, n_blocks = 8, 128, 128, 17000
    rows = n_blocks * bs
    assert rows * nkv * hd > 2 ** 31
    k = torch.zeros(rows, nkv * hd, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(rows, nkv * hd, dtype=torch.bfloat16, device="cuda")
    b = Batch([(1, 300), (20, 200)], 8, nkv, hd, bs, True, seed=20, spare=0)
    far = torch.tensor([n_blocks - 1 - i for i in range(b.n_blocks)])
    for x, y in ((k, b.k), (v, b.v)):
        for i in range(b.n_blocks):
            x[int(far[i]) * bs:int(far[i] + 1) * bs] = y[i * bs:(i + 1) * bs].cuda()
    qkv, cu, lens = b.cuda("qkv", "cu_q", "lens")
    table = torch.where(b.table >= 0, far[b.table.clamp(min=0).long()].int(), b.table).cuda()
    out = torch.full((b.n_tok, 8 * hd), 7.0, dtype=b.dt, device="cuda")
    mx.run_prefill_batch(qkv[:, :8 * hd], k, v, out, table, bs, cu, lens, 20, 8, nkv, hd)
    torch.cuda.synchronize()
    check(b, out.cpu(), None)
