"""Attention of a batch over a paged cache where it is easily wrong: rows of a cache
gigabytes apart, scores that are all -infinity, infinities in the V of keys that are
split, and workspaces on the stream of their call."""
from __future__ import annotations

import math

import pytest
import torch

import mx230_amd as mx
from cache_helpers import Batch
from test_gpu_prefill_batch import TYPES, check, run

pytestmark = pytest.mark.gpu


def reach_of(b, heads, skip=0):
    """Batch.attention's `reach` over some query heads, and keys from position `skip` on."""
    group, hd, t0, reach = b.nh // b.nkv, b.hd, 0, 0.0
    for s, (n, _) in enumerate(b.pairs):
        for h in heads:
            q = b.qkv[t0:t0 + n, h * hd:(h + 1) * hd].double().abs()
            k = b.k[b.rows[s][skip:], h // group * hd:(h // group + 1) * hd].double().abs()
            reach = max(reach, float((q @ k.T).max()) / math.sqrt(hd))
        t0 += n
    return reach


@pytest.mark.parametrize("bf16,stride,nh,n", [
    (False, 2 ** 30, 2, 1), (False, 2 ** 30 + 16, 2, 1), (False, 2 ** 30 + 16, 32, 1), (False, 2 ** 30, 2, 2),
    (True, 2 ** 31 - 8, 2, 1), (True, 2 ** 31 - 8, 32, 1)])
def test_rows_past_32_bits_apart(bf16, stride, nh, n):
    """Cache rows (and rows of q and out) whose distance in bytes passes 32 bits: few
    rows and many, read and appended."""
    nkv, hd = 1, 64
    b = Batch([(n, 2)], nh, nkv, hd, 1, bf16, seed=nh, spare=0)
    w = nkv * hd
    cols = 2 * w + 2 * (nh + 2) * hd
    big = torch.empty(stride + cols, dtype=b.dt, device="cuda")

    def at(c, wide, rows=2):
        return big.as_strided((rows, wide), (stride, 1), c)
    k, v, q, out = at(0, w), at(w, w), at(2 * w, (nh + 2) * hd), at(2 * w + (nh + 2) * hd, nh * hd)
    table, cu, lens, qkv = b.cuda("table", "cu_q", "lens", "qkv")
    k.copy_(b.k.cuda())
    v.copy_(b.v.cuda())
    q[:n].copy_(qkv)
    print(f"\n[rows apart] {stride} {b.dt} heads {nh} new {n}", flush=True)
    mx.run_prefill_batch(q[:n, :nh * hd], k, v, out[:n], table, 1, cu, lens, n, nh, nkv, hd)
    check(b, out[:n].cpu(), None)
    # the append's rows, both new: K and V as they came
    cu2 = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    two = torch.randn(2, (nh + 2) * hd, generator=torch.Generator().manual_seed(1)).to(b.dt).cuda()
    q.copy_(two)
    mx.run_cache_append(q, out, k, v, table, 1, cu2, lens, nh, nkv, hd)
    order = table[0].long()
    assert torch.equal(k[order], two[:, nh * hd:(nh + 1) * hd]) and torch.equal(v[order], two[:, (nh + 1) * hd:])
    assert torch.equal(out, two[:, :nh * hd])


@pytest.mark.parametrize("bf16,hd", TYPES)
@pytest.mark.parametrize("how", ["infinite", "overflow"])
@pytest.mark.parametrize("pairs", [
    [(1, 40), (1, 1), (2, 130)], [(80, 100), (70, 200)], [(1, 3000), (3, 2900)], [(70, 6000)], [(40, 5000), (1, 4500), (5, 3)]])
def test_scores_all_minus_infinity(pairs, how, bf16, hd):
    """Every score that a row of the first KV head sees is -infinity, by K or by
    products past the type's range: no softmax exists, so NaN, its lse -infinity (not
    the zeros of a row that sees no position). The other head is as ever."""
    b = Batch(pairs, 4, 2, hd, 16, bf16, seed=21)
    rows = torch.cat(b.rows)
    for h in range(2):
        b.qkv[:, h * hd] = 3e38 if how == "overflow" else b.qkv[:, h * hd].abs() + 0.5
    b.k[rows, 0] = -3e38 if how == "overflow" else -math.inf
    out, lse = run(b)
    t0 = 0
    for n, ln in pairs:
        for i in range(t0, t0 + n):
            got = out[i, :2 * hd]
            assert not got.any() if ln - n + i - t0 < 0 else bool(torch.isnan(got).all()), (n, ln, i - t0)
        t0 += n
    assert bool((lse[:, :2] == -math.inf).all())
    want, mag, wlse, _ = b.attention()
    reach, other = reach_of(b, (2, 3)), slice(2 * hd, None)
    assert bool(((out.double() - want).abs() <= b.tolerance(want, mag, reach))[:, other].all())
    fine = torch.isfinite(wlse[:, 2:])
    assert torch.equal(lse[:, 2:][~fine].double(), wlse[:, 2:][~fine])
    assert float((lse.double() - wlse)[:, 2:][fine].abs().max()) <= b.lse_tolerance(reach)


@pytest.mark.parametrize("bf16,hd", TYPES)
@pytest.mark.parametrize("pairs", [[(1, 200), (3, 190)], [(80, 200)], [(1, 5000), (3, 4900)], [(70, 6000)]])
def test_scores_minus_infinity_at_first(pairs, bf16, hd):
    """Keys whose score is -infinity weigh nothing beside others: the first 100
    positions, whole stages and shares among them."""
    b = Batch(pairs, 2, 1, hd, 16, bf16, seed=22)
    b.qkv[:, 0], b.qkv[:, hd] = (b.qkv[:, c].abs() + 0.5 for c in (0, hd))
    for s in range(len(pairs)):
        b.k[b.rows[s][:100], 0] = -math.inf
    out, lse = run(b)
    want, mag, wlse, _ = b.attention()
    assert bool(torch.isfinite(want).all())
    reach = reach_of(b, (0, 1), skip=100)
    off = (out.double() - want).abs()
    assert bool((off <= b.tolerance(want, mag, reach)).all()), float(off.max())
    assert float((lse.double() - wlse).abs().max()) <= b.lse_tolerance(reach)


@pytest.mark.parametrize("bf16,hd", TYPES)
@pytest.mark.parametrize("pairs", [[(1, 200), (3, 190)], [(80, 200)], [(1, 5000), (3, 4900)], [(70, 6000)],
                                   [(1, 9000)], [(1, 30), (40, 3000)]])
@pytest.mark.parametrize("signs", ["+", "-", "+-"])
def test_infinite_values(pairs, signs, bf16, hd):
    """An infinite V that a row sees, in the last position: the sum is that infinity,
    and NaN where both are seen, whether the keys are split or not."""
    b = Batch(pairs, 4, 2, hd, 16, bf16, seed=23)
    for s, (n, ln) in enumerate(pairs):
        last = b.rows[s][ln - n:]
        b.v[last, :hd] = -math.inf if signs == "-" else math.inf
        if signs == "+-":
            b.v[b.rows[s][0], :hd] = -math.inf
    out, lse = run(b)
    want, _, wlse, reach = b.attention()
    c = slice(0, 2 * hd)
    assert torch.equal(torch.isnan(out[:, c]), torch.isnan(want[:, c]))
    fine = ~torch.isnan(want[:, c])
    assert torch.equal(out[:, c][fine].double(), want[:, c][fine])
    assert bool(torch.isfinite(out[:, 2 * hd:]).all())
    assert float((lse.double() - wlse).abs().max()) <= b.lse_tolerance(reach)


def test_workspace_belongs_to_the_stream():
    """The workspace that a call on a given stream allocates comes from that stream's
    memory: not what a call on the current stream still uses, whose tensor is gone."""
    b = Batch([(1, 4000), (1, 300), (40, 2500)], 4, 2, 64, 16, True, seed=24)
    want, _ = run(b)
    k, v, table, cu, lens, qkv = b.cuda("k", "v", "table", "cu_q", "lens", "qkv")
    out = [torch.zeros(b.n_tok, b.nh * b.hd, dtype=b.dt, device="cuda") for _ in range(3)]
    s = torch.cuda.Stream()
    torch.cuda.synchronize()

    def call(o, stream):
        return mx.run_prefill_batch(qkv[:, :b.nh * b.hd], k, v, o, table, b.bs, cu, lens, 40, b.nh, b.nkv, b.hd, stream=stream)
    ws = call(out[0], None)
    mine, size = ws.data_ptr(), ws.numel()
    del ws
    ws = call(out[1], s)
    assert ws.data_ptr() + ws.numel() <= mine or mine + size <= ws.data_ptr()
    theirs = ws.data_ptr()
    del ws
    # and the other way about: the next call here does not get the stream's
    ws = call(out[2], None)
    assert ws.data_ptr() + ws.numel() <= theirs or theirs + size <= ws.data_ptr()
    torch.cuda.synchronize()
    for o in out:
        assert torch.equal(o.cpu(), want)


@pytest.mark.parametrize("pairs", [[(1, 900), (3, 700), (1, 1)], [(150, 400), (1, 300)], [(1, 1)]])
def test_neighbours_in_memory(pairs):
    """The output in the free columns of q's rows, and every tensor right behind the
    one before it in one allocation, are not over each other."""
    nh, nkv, hd = 2, 1, 64
    b = Batch(pairs, nh, nkv, hd, 16, True, seed=25)
    k, v, table, cu, lens, qkv = b.cuda("k", "v", "table", "cu_q", "lens", "qkv")
    mx.run_prefill_batch(qkv[:, :nh * hd], k, v, qkv[:, nh * hd:], table, 16, cu, lens, b.max_q, nh, nkv, hd)
    check(b, qkv[:, nh * hd:].cpu(), None)
    assert torch.equal(qkv[:, :nh * hd].cpu(), b.qkv[:, :nh * hd])
    need = mx.prefill_batch_workspace_bytes(b.n_tok, len(pairs), b.max_q, nh, nkv, hd)
    rows = -(-need // (2 * hd))
    arena = torch.full((2 * k.shape[0] + 2 * nh * b.n_tok + rows + -(-2 * nh * b.n_tok // hd), hd), 7.0, dtype=b.dt,
                       device="cuda")
    parts = arena.split([k.shape[0], nh * b.n_tok, k.shape[0], nh * b.n_tok, rows, -(-2 * nh * b.n_tok // hd)])
    ak, aq, av, ao, ws, lse = parts
    aq, ao = aq.view(b.n_tok, nh * hd), ao.view(b.n_tok, nh * hd)
    lse = lse.view(torch.float32).flatten()[:b.n_tok * nh].view(b.n_tok, nh)
    for x, y in ((ak, k), (av, v), (aq, b.qkv[:, :nh * hd])):
        x.copy_(y)
    mx.run_prefill_batch(aq, ak, av, ao, table, 16, cu, lens, b.max_q, nh, nkv, hd, lse=lse, workspace=ws)
    check(b, ao.cpu(), lse.cpu())
