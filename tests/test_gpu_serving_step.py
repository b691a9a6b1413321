"""The cache append (mxfa_run_cache_append), and the paged-cache operators together as an
engine has them: prompts enter in chunks, tokens are generated, beams fork, sequences
end, the pool is compacted, and every step's attention is that of the whole
sequence in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

import mx230_amd as mx
from cache_helpers import Batch, turned, turned_tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("pairs,nh,nkv,hd,dim,bs,interleaved", [
    ([(1, 1)], 1, 1, 64, 64, 16, False), ([(1, 17), (1, 300), (3, 33)], 14, 2, 64, 64, 16, False),
    ([(70, 100), (0, 5), (1, 64), (9, 9)], 4, 2, 128, 96, 1, True), ([(300, 1000), (2, 4000)], 8, 8, 64, 24, 128, False),
    ([(5, 3), (2, 40)], 3, 1, 128, 10, 16, True), ([(40, 60), (1, 2)], 2, 1, 96, 0, 16, False)])
def test_append(pairs, nh, nkv, hd, dim, bs, interleaved, bf16):
    """Q, K and V land turned at their positions, nothing else changes: rows of no
    sequence, positions below 0, and the rest of the caches."""
    b = Batch(pairs, nh, nkv, hd, bs, bf16, seed=dim, extra_rows=2, wide=1)
    k0, v0, table, cu, lens, qkv = b.cuda("k", "v", "table", "cu_q", "lens", "qkv")
    f = mx.rotary_frequencies(dim)[0] if dim else None
    out = torch.full((b.n_tok, nh * hd), 7.0, dtype=b.dt, device="cuda")
    kc, vc = k0.clone(), v0.clone()
    mx.run_cache_append(qkv, out, kc, vc, table, bs, cu, lens, nh, nkv, hd, f, interleaved, 0.75)
    wk, wv, wo = b.k.double(), b.v.double(), torch.full((b.n_tok, nh * hd), 7.0, dtype=torch.float64)
    tol = [torch.zeros_like(x) for x in (wk, wv, wo)]
    t0 = 0
    for s, (n, ln) in enumerate(pairs):
        for i in range(n):
            at = ln - n + i
            if at < 0:
                continue
            x = b.qkv[t0 + i].view(nh + 2 * nkv, hd)
            w, e = x.double(), torch.zeros(x.shape, dtype=torch.float64)
            if dim:
                w = turned(x, torch.tensor(at), f.cpu(), interleaved, 0.75)
                e = turned_tolerance(x, w, dim // 2, interleaved, 0.75)
            row = b.rows[s][at]
            wo[t0 + i], tol[2][t0 + i] = w[:nh].flatten(), e[:nh].flatten()
            wk[row], tol[0][row] = w[nh:nh + nkv].flatten(), e[nh:nh + nkv].flatten()
            wv[row] = x[nh + nkv:].double().flatten()
        t0 += n
    for got, want, e in zip((kc, vc, out), (wk, wv, wo), tol):
        got = got.cpu().double()
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(got), nan)
        assert bool(((got - want).abs()[~nan] <= e[~nan]).all())
    # in place, and by the Python path
    mine = qkv.clone()
    mx.run_cache_append(mine, mine, k0, v0, table, bs, cu, lens, nh, nkv, hd, f, interleaved, 0.75,
                        stream=torch.cuda.current_stream())
    rows = [i for i in range(b.n_tok) if not bool((wo[i] == 7.0).all())]
    assert torch.equal(mine[rows, :nh * hd], out[rows]) and torch.equal(mine[:, nh * hd:], qkv[:, nh * hd:])
    assert torch.equal(k0.view(torch.uint8), kc.view(torch.uint8)) and torch.equal(v0.view(torch.uint8), vc.view(torch.uint8))


def test_append_bad_tables():
    """Blocks outside the pool and positions past the table are left out."""
    b = Batch([(2, 30), (2, 20)], 2, 1, 64, 16, True, seed=1)
    b.table[0, 1] = b.n_blocks
    b.lens[1] = 1000
    k, v, table, cu, lens, qkv = b.cuda("k", "v", "table", "cu_q", "lens", "qkv")
    kc, vc, out = k.clone(), v.clone(), torch.empty(4, 128, dtype=b.dt, device="cuda")
    mx.run_cache_append(qkv, out, kc, vc, table, 16, cu, lens, 2, 1, 64)
    assert torch.equal(kc.view(torch.uint8), k.view(torch.uint8)) and torch.equal(out, qkv[:, :128])
    b.cu_q[1] = 10 ** 9
    mx.run_cache_append(qkv, out, kc, vc, table, 16, b.cu_q.cuda(), lens, 2, 1, 64)


class Engine:
    """A cache of one layer, its tables, and beside them every sequence's own rows of
    Q, K and V as they came."""

    def __init__(self, nh, nkv, hd, bs, n_blocks, rows, entries, bf16, seed):
        self.nh, self.nkv, self.hd, self.bs, self.n_blocks = nh, nkv, hd, bs, n_blocks
        self.dt = torch.bfloat16 if bf16 else torch.float32
        self.pools = torch.full((2, n_blocks * bs, nkv * hd), math.nan, dtype=self.dt, device="cuda")
        self.table = torch.full((rows, entries), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.refs = torch.zeros(n_blocks, dtype=torch.int32, device="cuda")
        self.f, self.a = mx.rotary_frequencies(hd, scaling="yarn", factor=8.0, original_length=64)
        self.g = torch.Generator().manual_seed(seed)
        self.said = {}

    def grow(self, new):
        """Room for new[s] more tokens of row s: the host's part, as an engine has it."""
        t, ln, rf = self.table.tolist(), self.lens.tolist(), self.refs.tolist()
        for s, n in new.items():
            for j in range(-(-ln[s] // self.bs), -(-(ln[s] + n) // self.bs)):
                t[s][j] = rf.index(0)
                rf[t[s][j]] = 1
            ln[s] += n
        for x, y in ((self.table, t), (self.lens, ln), (self.refs, rf)):
            x.copy_(torch.tensor(y, dtype=torch.int32))

    def step(self, new):
        """Tokens enter and attend; every output row against the whole sequence's."""
        nh, nkv, hd = self.nh, self.nkv, self.hd
        self.grow(new)
        n_seq = self.table.shape[0]
        count = [new.get(s, 0) for s in range(n_seq)]
        qkv = torch.randn(sum(count), (nh + 2 * nkv) * hd, generator=self.g).to(self.dt)
        x = qkv.cuda()
        cu = torch.tensor([0] + count).cumsum(0).to(torch.int32).cuda()
        mx.run_cache_append(x, x, self.pools[0], self.pools[1], self.table, self.bs, cu, self.lens, nh, nkv, hd, self.f,
                            factor=self.a)
        out = torch.empty(sum(count), nh * hd, dtype=self.dt, device="cuda")
        mx.run_prefill_batch(x[:, :nh * hd], self.pools[0], self.pools[1], out, self.table, self.bs, cu, self.lens,
                             max(count), nh, nkv, hd)
        got, t0 = out.cpu().double(), 0
        for s, n in enumerate(count):
            if n == 0:
                continue
            self.said[s] = torch.cat([self.said.get(s, qkv[:0]), qkv[t0:t0 + n]])
            whole = self.said[s].double().view(-1, nh + 2 * nkv, hd)
            at, rnd = torch.arange(len(whole)), (lambda z: z.to(self.dt).double())
            q = rnd(turned(whole[:, :nh], at[:, None], self.f.cpu(), False, self.a))
            k = rnd(turned(whole[:, nh:nh + nkv], at[:, None], self.f.cpu(), False, self.a))
            for h in range(nh):
                kh, vh = k[:, h // (nh // nkv)], whole[:, nh + nkv + h // (nh // nkv)]
                p = q[-n:, h] @ kh.T / math.sqrt(hd)
                p = p.masked_fill(at[None] > at[-n:, None], -math.inf).softmax(-1)
                off = (got[t0:t0 + n, h * hd:(h + 1) * hd] - p @ vh).abs()
                # weights and result rounded (2^-8 each) as in the attention tests; where Q
                # or K round the other way here than there, by a step (2^-7 of one product
                # in a score of |q| |k| sqrt(hd)), a weight moves by some 2^-7 more
                u = 2.0 ** -8 if self.dt == torch.bfloat16 else 2.0 ** -16
                assert bool((off <= 4 * u * (p @ vh.abs()) + 1e-12).all()), (s, h, float(off.max()))
            t0 += n


@pytest.mark.parametrize("bf16", [True, False])
def test_engine(bf16):
    e = Engine(4, 2, 64, 16, 200, 10, 12, bf16, seed=3)
    e.step({0: 100, 1: 37, 2: 5})           # prompts
    e.step({0: 1, 1: 40, 2: 1, 3: 64})      # tokens beside chunks
    pairs = torch.zeros(100, 2, dtype=torch.int32, device="cuda")
    status = torch.zeros(4, dtype=torch.int32, device="cuda")
    counts = torch.zeros(2, dtype=torch.int32, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    mx.run_pages_fork(e.table, 16, e.lens, e.refs, i32(0, 0, 1, 3), i32(4, 5, 6, 7), pairs, status, counts)
    mx.run_pages_copy(e.pools, 16, pairs, counts)
    assert status.tolist() == [0] * 4 and counts.tolist() == [3, 0]
    for p, c in ((0, 4), (0, 5), (1, 6), (3, 7)):
        e.said[c] = e.said[p]
    e.step({s: 1 for s in (0, 1, 4, 5, 6, 7)})  # beams go their own ways
    mx.run_pages_free(e.table, 16, e.lens, e.refs, i32(0, 3, 6))
    for s in (0, 3, 6):
        del e.said[s]
    e.step({1: 3, 2: 1, 4: 1, 5: 20, 7: 1})
    mx.run_pages_free(e.table, 16, e.lens, e.refs, i32(1))  # leaves holes below the others
    del e.said[1]
    nt, nr = torch.empty_like(e.table), torch.empty_like(e.refs)
    mx.run_pages_compact(e.table, 16, e.lens, e.refs, nt, nr, pairs, counts)
    mx.run_pages_copy(e.pools, 16, pairs, counts)
    moved, live = counts.tolist()
    assert moved > 0 and bool((nr[live:] == 0).all()) and bool((nr[:live] > 0).all())
    e.pools[:, live * 16:] = math.nan  # the pool's end is not used any more
    e.table, e.refs = nt, nr
    e.step({2: 1, 4: 1, 5: 1, 7: 1})
    e.step({8: 90, 4: 2, 5: 1})
