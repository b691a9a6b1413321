"""The microscaled cache as it is used: serving steps of append and attention over pages
that are forked, freed and compacted, beside the same steps over an ordinary cache of
what it holds; captured and replayed, on streams of their own, and with lengths, blocks
and counts on the device that change between replays."""
from __future__ import annotations

import math

import pytest
import torch

import mx230_amd as mx
from mx_helpers import MxBatch, held

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def near(a, b):
    """Both round each weight and the result once: 2^-7 of the values' size apart."""
    return float((a.float() - b.float()).abs().max()) <= 2.0 ** -6 * max(1.0, float(b.float().abs().max()))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("bf16,hd", [(True, 64), (True, 128), (False, 64)])
def test_steps_with_pages(bf16, hd, bits):
    """A prompt, two beams forked from it, some steps, one beam ended, the pool
    compacted: at each step attention is that over an ordinary cache of the values
    read back."""
    nh, nkv, bs, n_blocks = 6, 2, 16, 40
    dt = torch.bfloat16 if bf16 else torch.float32
    g = torch.Generator(device="cuda").manual_seed(bits)
    wide = mx.mx_block_bytes(bs, nkv, hd, bits)
    pools = torch.zeros(2, n_blocks, wide, dtype=torch.uint8, device="cuda")
    table, lens, refs = torch.full((3, 12), -1, dtype=torch.int32, device="cuda"), ints([70, 0, 0]), ints([0] * n_blocks)
    table[0, :5] = ints([30, 7, 39, 2, 11])
    refs[[30, 7, 39, 2, 11]] = 1
    f, factor = mx.rotary_frequencies(hd)

    def step(new):
        """Appends and attends; the read rows of all sequences."""
        n = sum(new)
        cu = ints([0] + torch.tensor(new).cumsum(0).tolist())
        qkv = torch.randn(n, (nh + 2 * nkv) * hd, generator=g, device="cuda").to(dt)
        q, out, plain = (torch.zeros(n, nh * hd, dtype=dt, device="cuda") for _ in range(3))
        print(f"\n[mx step] {new} lens {lens.tolist()} d {hd} bits {bits}", flush=True)
        mx.run_cache_append_mx(qkv, q, pools[0], pools[1], bits, table, bs, cu, lens, nh, nkv, hd, frequencies=f, factor=factor)
        mx.run_prefill_batch_mx(q, pools[0], pools[1], bits, out, table, bs, cu, lens, max(new), nh, nkv, hd)
        # the same over ordinary rows: the cache's values at the same places
        all_cu = torch.cat([ints([0]), lens.cumsum(0).to(torch.int32)])
        total = int(all_cu[-1])
        k, v = (torch.zeros(total, nkv * hd, dtype=dt, device="cuda") for _ in range(2))
        mx.run_cache_read_mx(pools[0], pools[1], bits, k, v, table, bs, all_cu, lens, nkv, hd)
        kc, vc = (torch.zeros(n_blocks * bs, nkv * hd, dtype=dt, device="cuda") for _ in range(2))
        at = 0
        for s, ln in enumerate(lens.tolist()):
            i = torch.arange(ln, device="cuda")
            rows = table[s].long()[i // bs] * bs + i % bs
            kc[rows], vc[rows] = k[at:at + ln], v[at:at + ln]
            at += ln
        mx.run_prefill_batch(q, kc, vc, plain, table, bs, cu, lens, max(new), nh, nkv, hd)
        assert near(out, plain)
        return k, v

    step([70, 0, 0])
    mx_pairs, status, counts = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), ints([9, 9]), ints([9, 9])
    mx.run_pages_fork(table, bs, lens, refs, ints([0, 0]), ints([1, 2]), mx_pairs, status, counts)
    mx.run_pages_copy(pools, 1, mx_pairs, counts)
    assert status.tolist() == [0, 0] and counts.tolist() == [2, 0] and lens.tolist() == [70, 70, 70]

    def grow():
        """One more position each; a block of its own where one begins."""
        lens.add_(1)
        for s in range(3):
            j = (int(lens[s]) - 1) // bs
            if int(table[s, j]) < 0:
                free = int((refs == 0).nonzero()[0])
                table[s, j] = free
                refs[free] = 1

    for _ in range(11):
        grow()
        k, v = step([1, 1, 1])
        # the beams share the prompt's values and differ after it
        a, b, c = (x.view(3, -1, nkv * hd) for x in (k, v, k))
        assert torch.equal(a[0, :70], a[1, :70]) and torch.equal(b[0, :70], b[2, :70]) and not torch.equal(c[0, 70:], c[1, 70:])
    mx.run_pages_free(table, bs, lens, refs, ints([1]))
    lens_before = lens.tolist()
    k0, v0 = (torch.zeros(2 * 81, nkv * hd, dtype=dt, device="cuda") for _ in range(2))
    mx.run_cache_read_mx(pools[0], pools[1], bits, k0, v0, table, bs, ints([0, 81, 81, 162]), lens, nkv, hd)
    new_refs, pairs = torch.zeros_like(refs), torch.zeros(n_blocks // 2, 2, dtype=torch.int32, device="cuda")
    mx.run_pages_compact(table, bs, lens, refs, table, new_refs, pairs, counts)
    mx.run_pages_copy(pools, 1, pairs, counts)
    assert int(counts[0]) > 0 and lens.tolist() == lens_before == [81, 0, 81]
    k1, v1 = torch.zeros_like(k0), torch.zeros_like(v0)
    mx.run_cache_read_mx(pools[0], pools[1], bits, k1, v1, table, bs, ints([0, 81, 81, 162]), lens, nkv, hd)
    assert torch.equal(k0, k1) and torch.equal(v0, v1)


@pytest.mark.parametrize("bits", [8, 4])
def test_equal_tokens_equal_bytes(bits):
    """A token's bytes do not hang on the call it was written by: a chunk and token by
    token, beside others or alone, give the same pool."""
    nh, nkv, hd, bs = 4, 2, 128, 16
    b = MxBatch([(90, 90), (41, 60)], nh, nkv, hd, bs, bits, True, seed=3)
    qkv, table, lens, cu = b.cuda("qkv", "table", "lens", "cu_q")
    f, factor = mx.rotary_frequencies(hd)
    pools = [torch.zeros_like(b.kp, device="cuda") for _ in range(4)]
    q0, q1 = (torch.zeros(131, nh * hd, dtype=b.dt, device="cuda") for _ in range(2))
    mx.run_cache_append_mx(qkv, q0, pools[0], pools[1], bits, table, bs, cu, lens, nh, nkv, hd, frequencies=f, factor=factor)
    for i in range(131):
        s, at = (0, i + 1) if i < 90 else (1, 19 + i - 90 + 1)
        mx.run_cache_append_mx(qkv[i:i + 1], q1[i:i + 1], pools[2], pools[3], bits, table[s:s + 1], bs, ints([0, 1]), ints([at]),
                               nh, nkv, hd, frequencies=f, factor=factor)
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3]) and torch.equal(q0, q1)


@pytest.mark.parametrize("bits", [8, 4])
def test_captured_step(bits):
    """Append, attention and read in one graph, replayed with other tokens, lengths and
    tables in the same buffers, eager calls between: every replay is the eager result."""
    nh, nkv, hd, bs = 14, 2, 64, 16
    shapes = [[(1, 300), (40, 500), (1, 2000), (3, 90)], [(20, 700), (1, 1), (22, 22), (2, 1500)], [(0, 10), (45, 45), (0, 0), (0, 900)]]
    bs_ = [MxBatch(p, nh, nkv, hd, bs, bits, True, seed=i, spare=5) for i, p in enumerate(shapes)]
    n_blocks, wide = max(b.n_blocks for b in bs_), max(b.table.shape[1] for b in bs_)
    block = bs_[0].kp.shape[1]
    kp, vp = (torch.zeros(n_blocks, block, dtype=torch.uint8, device="cuda") for _ in range(2))
    table = torch.full((4, wide), -1, dtype=torch.int32, device="cuda")
    cu, lens = torch.zeros(5, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    qkv = torch.zeros(45, (nh + 2 * nkv) * hd, dtype=torch.bfloat16, device="cuda")
    q, out = (torch.zeros(45, nh * hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    k, v = (torch.zeros(45, nkv * hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    f, _ = mx.rotary_frequencies(hd)
    ws = torch.empty(mx.prefill_batch_mx_workspace_bytes(45, 4, 45, nh, nkv, hd, True, bits), dtype=torch.uint8, device="cuda")

    def step(workspace):
        mx.run_cache_append_mx(qkv, q, kp, vp, bits, table, bs, cu, lens, nh, nkv, hd, frequencies=f)
        mx.run_prefill_batch_mx(q, kp, vp, bits, out, table, bs, cu, lens, 45, nh, nkv, hd, workspace=workspace)
        mx.run_cache_read_mx(kp, vp, bits, k, v, table, bs, cu, lens, nkv, hd)

    def fill(b):
        kp.zero_(), vp.zero_(), table.fill_(-1)
        kp[:b.n_blocks], vp[:b.n_blocks] = b.kp.cuda(), b.vp.cuda()
        table[:, :b.table.shape[1]] = b.table.cuda()
        cu.copy_(b.cu_q), lens.copy_(b.lens)
        qkv.zero_()
        qkv[:b.n_tok] = b.qkv.cuda()
        for x in (q, out, k, v):
            x.fill_(7.0)

    fill(bs_[0])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(ws)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(ws)
    for b in bs_ + bs_[::-1]:
        fill(b)
        step(None)
        torch.cuda.synchronize()
        want = [x.clone() for x in (q, out, k, v, kp, vp)]
        fill(b)
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip((q, out, k, v, kp, vp), want):
            assert torch.equal(got, w)
        assert bool((out[b.n_new:] == 7.0).all()) and bool((k[b.n_new:] == 7.0).all()) and not bool((out[:b.n_new] == 7.0).all(1).any())


@pytest.mark.parametrize("bits", [8, 4])
def test_given_stream(bits):
    """Calls on a given stream run there, behind its work, whatever stream is current."""
    b = MxBatch([(1, 900), (30, 333)], 4, 2, 64, 16, bits, True, seed=8)
    qkv, table, cu, lens, kp, vp = b.cuda("qkv", "table", "cu_q", "lens", "kp", "vp")
    q, out, k, v = (torch.zeros(31, w, dtype=b.dt, device="cuda") for w in (256, 256, 128, 128))
    mx.run_cache_append_mx(qkv, q, kp, vp, bits, table, 16, cu, lens, 4, 2, 64)
    mx.run_prefill_batch_mx(q, kp, vp, bits, out, table, 16, cu, lens, 30, 4, 2, 64)
    mx.run_cache_read_mx(kp, vp, bits, k, v, table, 16, cu, lens, 2, 64)
    want = [x.clone() for x in (q, out, k, v, kp, vp)]
    src, late = qkv.clone(), torch.zeros_like(qkv)
    kp2, vp2 = b.cuda("kp", "vp")
    for x in (q, out, k, v):
        x.zero_()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        busy = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            busy = busy @ busy * 1e-3
        late.copy_(src)
    kw = dict(stream=s)
    mx.run_cache_append_mx(late, q, kp2, vp2, bits, table, 16, cu, lens, 4, 2, 64, **kw)
    mx.run_prefill_batch_mx(q, kp2, vp2, bits, out, table, 16, cu, lens, 30, 4, 2, 64, **kw)
    mx.run_cache_read_mx(kp2, vp2, bits, k, v, table, 16, cu, lens, 2, 64, **kw)
    s.synchronize()
    for got, w in zip((q, out, k, v, kp2, vp2), want):
        assert torch.equal(got, w)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("bs,entries", [(16, 3), (128, 1)])
def test_lengths_and_blocks_of_any_kind(bs, entries, bits):
    """Whatever lens, cu_q and the tables hold, nothing outside the buffers is touched,
    and a sound sequence beside gets its result."""
    b = MxBatch([(2, 40), (1, 33), (5, 44)], 4, 2, 64, bs, bits, True, seed=9, spare=1)
    qkv, kp, vp = b.cuda("qkv", "kp", "vp")
    table = b.table[:, :entries].contiguous()
    out = torch.zeros(b.n_tok, 256, dtype=b.dt, device="cuda")
    mx.run_prefill_batch_mx(qkv[:, :256], kp, vp, bits, out, table.cuda(), bs, b.cu_q.cuda(), b.lens.cuda(), 5, 4, 2, 64)
    sound = out[:2].clone()
    for lens in ([40, 2 ** 31 - 1, 44], [40, -5, 2 ** 31 - 1], [40, -2 ** 31, 0]):
        for cu in ([0, 2, 3, 8], [0, 2, 100, 8], [0, 2, -7, 2 ** 31 - 1], [0, 2, 2, 2 ** 31 - 1]):
            own = cu[2] >= 2  # (a third sequence from -7 on has the first one's rows too)
            for bad in (-1, -2 ** 31, 2 ** 31 - 1, b.n_blocks):
                t = table.clone()
                t[1:] = bad
                print(f"\n[mx] lens {lens} cu {cu} blocks {bad} size {bs} bits {bits}", flush=True)
                guard = torch.zeros(3, *kp.shape, dtype=torch.uint8, device="cuda")
                guard[1] = kp
                k2, v2 = guard[1], vp.clone()
                got = torch.zeros_like(out)
                mx.run_prefill_batch_mx(qkv[:, :256], k2, v2, bits, got, t.cuda(), bs, ints(cu), ints(lens), 5, 4, 2, 64)
                assert not own or torch.equal(got[:2], sound)
                q, k, v = torch.zeros_like(out), *(torch.zeros(b.n_tok, 128, dtype=b.dt, device="cuda") for _ in range(2))
                mx.run_cache_append_mx(qkv, q, k2, v2, bits, t.cuda(), bs, ints(cu), ints(lens), 4, 2, 64)
                mx.run_cache_read_mx(k2, v2, bits, k, v, t.cuda(), bs, ints(cu), ints(lens), 2, 64)
                assert not guard[0].any() and not guard[2].any()
                rows = [int(table[0, p // bs]) * bs + p % bs for p in (38, 39)]
                assert not own or torch.equal(k[:2].cpu().double(), held(k2.cpu(), rows, 2, bs, 64, bits))
    assert math.isfinite(float(sound.float().sum()))


@pytest.mark.parametrize("bf16,hd,bits", [(True, 64, 8), (True, 128, 4), (False, 64, 4)])
def test_pools_in_one_tensor(bf16, hd, bits):
    """K's and V's blocks as columns of the same wider rows: the bytes and the results of
    pools that lie apart, and nothing else touched; over each other they are refused."""
    nh, nkv, bs, pairs = 6, 2, 16, [(5, 70), (1, 1), (40, 40), (1, 900)]
    b = MxBatch(pairs, nh, nkv, hd, bs, bits, bf16, seed=hd)
    kp, vp, table, cu, lens, qkv = b.cuda("kp", "vp", "table", "cu_q", "lens", "qkv")
    wide = kp.shape[1]
    both = torch.full((kp.shape[0], 2 * wide + 48), 0x5a, dtype=torch.uint8, device="cuda")
    k2, v2 = both[:, 16:16 + wide], both[:, 32 + wide:32 + 2 * wide]
    k2.copy_(kp)
    v2.copy_(vp)
    got = []
    for k, v in ((kp, vp), (k2, v2)):
        q, out = (torch.zeros(b.n_tok, nh * hd, dtype=b.dt, device="cuda") for _ in range(2))
        ko, vo = (torch.zeros(b.n_tok, nkv * hd, dtype=b.dt, device="cuda") for _ in range(2))
        mx.run_cache_append_mx(qkv, q, k, v, bits, table, bs, cu, lens, nh, nkv, hd)
        mx.run_prefill_batch_mx(q, k, v, bits, out, table, bs, cu, lens, b.max_q, nh, nkv, hd)
        mx.run_cache_read_mx(k, v, bits, ko, vo, table, bs, cu, lens, nkv, hd)
        got.append((q, out, ko, vo))
    assert all(torch.equal(x, y) for x, y in zip(*got)) and bool(got[0][1].any())
    assert torch.equal(k2, kp) and torch.equal(v2, vp)
    for c in (slice(0, 16), slice(16 + wide, 32 + wide), slice(32 + 2 * wide, None)):
        assert bool((both[:, c] == 0x5a).all())
    for v in (kp, kp[1:], k2):
        with pytest.raises((mx.MxfaError, ValueError)):
            mx.run_cache_append_mx(qkv, q, k2 if v is k2 else kp, v, bits, table, bs, cu, lens, nh, nkv, hd)
