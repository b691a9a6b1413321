"""The pages of a cache (free, fork, compact, copy) against the same steps in plain
Python, and against what must hold of them: counts that match the tables, data
that follows its sequence."""
from __future__ import annotations

import random

import pytest
import torch

import mx230_amd as mx

pytestmark = pytest.mark.gpu


def make(r, lens, bs, n_blocks, entries, width=64, pools=2, dtype=torch.bfloat16):
    order = list(range(n_blocks))
    r.shuffle(order)
    table = [[-1] * entries for _ in lens]
    refs = [0] * n_blocks
    for s, ln in enumerate(lens):
        for j in range(-(-ln // bs)):
            table[s][j] = order.pop()
            refs[table[s][j]] += 1
    pool = torch.randn(pools, n_blocks * bs, width, generator=torch.Generator().manual_seed(r.randrange(1000))).to(dtype)
    return table, list(lens), refs, pool


def dev(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def plain_fork(table, lens, refs, bs, parents, children):
    """By the definition: (status, pairs, table, lens, refs)."""
    t, ln, rf = [list(x) for x in table], list(lens), list(refs)
    status, pairs, named = [], [], set()
    n, free = len(lens), [b for b, x in enumerate(refs) if x == 0]
    for p, c in zip(parents, children):
        ok = 0 <= p < n and 0 <= c < n and lens[c] == 0
        first = ok and c not in named
        if ok:
            named.add(c)
        part = ok and lens[p] % bs != 0
        if not first or (part and not free):
            status.append(1)
            continue
        status.append(0)
        full = lens[p] // bs
        for j in range(full):
            t[c][j] = table[p][j]
            rf[table[p][j]] += 1
        if part:
            b = free.pop(0)
            t[c][full], rf[b] = b, 1
            pairs.append([table[p][full], b])
        ln[c] = lens[p]
    return status, pairs, t, ln, rf


def fork(table, lens, refs, bs, parents, children):
    n = len(parents)
    t, ln, rf = dev(table), dev(lens), dev(refs)
    pairs = torch.full((n, 2), -9, dtype=torch.int32, device="cuda")
    status, counts = torch.full((n,), -9, dtype=torch.int32, device="cuda"), dev([-9, -9])
    mx.run_pages_fork(t, bs, ln, rf, dev(parents), dev(children), pairs, status, counts)
    torch.cuda.synchronize()
    return t, ln, rf, pairs, status, counts


@pytest.mark.parametrize("seed", range(6))
def test_fork(seed):
    r = random.Random(seed)
    bs = r.choice([1, 16, 64])
    n = r.choice([6, 40, 300])
    lens = [r.choice([0, 0, r.randint(1, 5 * bs), bs * r.randint(1, 5)]) for _ in range(n)]
    table, lens, refs, _ = make(r, lens, bs, 5 * n + r.choice([0, 1, 3, 500]), 6)
    m = r.randint(1, 2 * n)
    parents = [r.randint(-1, n) for _ in range(m)]
    children = [r.randint(-1, n) for _ in range(m)]
    want = plain_fork(table, lens, refs, bs, parents, children)
    t, ln, rf, pairs, status, counts = fork(table, lens, refs, bs, parents, children)
    assert status.tolist() == want[0]
    assert counts.tolist() == [len(want[1]), sum(want[0])]
    assert pairs[:len(want[1])].tolist() == want[1]
    assert (t.tolist(), ln.tolist(), rf.tolist()) == want[2:]


@pytest.mark.parametrize("entries", [1, 255, 256, 257, 700])
def test_fork_long_rows(entries):
    """Rows shared by the plan's own launch (8 pairs of up to 256 entries) and by a second."""
    r = random.Random(entries)
    lens = [16 * entries, max(1, 16 * entries - 5)] + [0] * 8
    table, lens, refs, _ = make(r, lens, 16, 2 * entries + 9, entries)
    parents, children = [0, 1] * 4, list(range(2, 10))
    want = plain_fork(table, lens, refs, 16, parents, children)
    t, ln, rf, pairs, status, counts = fork(table, lens, refs, 16, parents, children)
    assert status.tolist() == want[0] and pairs[:len(want[1])].tolist() == want[1]
    assert (t.tolist(), ln.tolist(), rf.tolist()) == want[2:]


def test_fork_more_pairs_than_threads():
    r = random.Random(9)
    n = 3000
    lens = [100, 37, 0] + [0] * n
    table, lens, refs, _ = make(r, lens, 16, 9000, 7)
    parents = [r.randint(0, 2) for _ in range(n)]
    children = [3 + r.randrange(n) for _ in range(n)]
    want = plain_fork(table, lens, refs, 16, parents, children)
    t, ln, rf, pairs, status, counts = fork(table, lens, refs, 16, parents, children)
    assert status.tolist() == want[0] and pairs[:len(want[1])].tolist() == want[1]
    assert (t.tolist(), ln.tolist(), rf.tolist()) == want[2:]


def test_fork_refusals():
    """No block left, a child named twice, a full child, a child that is its own
    parent, a chain over an empty row, a parent longer than its row, no pairs."""
    table, lens, refs = [[0, 1], [2, -1], [-1, -1], [-1, -1], [-1, -1], [-1, -1]], [20, 16, 0, 0, 0, 50], [1, 1, 1, 0]
    pairs_ = [(0, 2), (0, 3), (1, 4), (1, 4), (0, 1), (2, 2), (5, 3), (4, 3)]
    t, ln, rf, pairs, status, counts = fork(table, lens, refs, 16, *zip(*pairs_))
    # (0, 3) claims row 3 and finds no block; row 4 was empty when the call began, but 3 is claimed
    assert status.tolist() == [0, 1, 0, 1, 1, 1, 1, 1] and counts.tolist() == [1, 6]
    assert pairs[0].tolist() == [1, 3]
    assert t.tolist() == [[0, 1], [2, -1], [0, 3], [-1, -1], [2, -1], [-1, -1]]
    assert ln.tolist() == [20, 16, 20, 0, 16, 50] and rf.tolist() == [2, 1, 2, 1]
    t, ln, rf, pairs, status, counts = fork(table, lens, refs, 16, [], [])
    assert counts.tolist() == [0, 0] and rf.tolist() == refs


def test_free():
    table, lens, refs = [[0, 1, -1], [2, 0, 3], [4, -1, -1], [-1, -1, -1]], [30, 33, 16, 0], [2, 1, 1, 1, 1, 0]
    t, ln, rf = dev(table), dev(lens), dev(refs)
    mx.run_pages_free(t, 16, ln, rf, dev([1, 3, 1, -1, 4, 2 ** 31 - 1]))
    assert t.tolist() == [[0, 1, -1], [-1, -1, -1], [4, -1, -1], [-1, -1, -1]]
    assert ln.tolist() == [30, 0, 16, 0] and rf.tolist() == [1, 1, 0, 0, 1, 0]
    mx.run_pages_free(t, 16, ln, rf, dev([]))
    mx.run_pages_free(t, 16, ln, rf, dev([0, 2]), stream=torch.cuda.current_stream())
    assert rf.tolist() == [0] * 6 and ln.tolist() == [0] * 4
    # a length past the row, and entries that are no blocks
    t, ln, rf = dev([[7, -3]]), dev([2 ** 31 - 1]), dev([1, 1])
    mx.run_pages_free(t, 16, ln, rf, dev([0]))
    assert t.tolist() == [[-1, -1]] and rf.tolist() == [1, 1] and ln.tolist() == [0]


def test_free_long_rows():
    r = random.Random(1)
    table, lens, refs, _ = make(r, [9000, 5000, 8192], 16, 1500, 600)
    t, ln, rf = dev(table), dev(lens), dev(refs)
    mx.run_pages_free(t, 16, ln, rf, dev([2, 0]))
    held = [0] * 1500
    for b in table[1]:
        if b >= 0:
            held[b] += 1
    assert rf.tolist() == held and ln.tolist() == [0, 5000, 0]


@pytest.mark.parametrize("n_blocks,dtype,width", [(1, torch.bfloat16, 64), (2, torch.float32, 4), (50, torch.bfloat16, 72),
                                                  (1025, torch.bfloat16, 8), (20000, torch.float32, 4)])
@pytest.mark.parametrize("bs", [2, 16])
def test_compact(n_blocks, bs, dtype, width):
    """Some sequences end, the rest moves down: every sequence reads what it read."""
    r = random.Random(n_blocks)
    entries = max(1, n_blocks // 10)
    lens = [r.randint(1, entries * bs) for _ in range(8)] if n_blocks > 1 else [1]
    while sum(-(-x // bs) for x in lens) > n_blocks:
        lens.pop()
    table, lens, refs, pool = make(r, lens, bs, n_blocks, entries, width, 3, dtype)
    t, ln, rf, pl = dev(table), dev(lens), dev(refs), pool.cuda()
    mx.run_pages_free(t, bs, ln, rf, dev(list(range(0, len(lens), 2)) if len(lens) > 1 else []))
    table, lens, refs = t.tolist(), ln.tolist(), rf.tolist()

    def read(tab, data):
        return [data[:, [tab[s][i // bs] * bs + i % bs for i in range(x)]] for s, x in enumerate(lens)]
    before = read(table, pool)
    nt, nr = torch.empty_like(t), torch.empty_like(rf)
    pairs, counts = torch.empty(max(1, n_blocks // 2), 2, dtype=torch.int32, device="cuda"), dev([-1, -1])
    mx.run_pages_compact(t, bs, ln, rf, nt, nr, pairs, counts)
    mx.run_pages_copy(pl, bs, pairs, counts)
    torch.cuda.synchronize()
    moves, live = counts.tolist()
    assert live == sum(1 for x in refs if x) and nr.tolist() == sorted(nr.tolist(), key=lambda x: x == 0)
    src = [b for b, x in enumerate(refs) if x and b >= live]
    dst = [b for b, x in enumerate(refs) if not x and b < live]
    assert pairs[:moves].tolist() == [list(x) for x in zip(src, dst)]
    held = [0] * n_blocks
    for s, x in enumerate(lens):
        for j in range(entries):
            used = j < -(-x // bs)
            assert (nt[s, j] >= 0) == used
            if used:
                held[int(nt[s, j])] += 1
    assert nr.tolist() == held
    after = read(nt.tolist(), pl.cpu())
    assert all(torch.equal(a, b) for a, b in zip(before, after))
    assert t.tolist() == table and rf.tolist() == refs  # what came in stays
    # the table in its own place, and a pool that is compact already
    mx.run_pages_compact(nt, bs, ln, nr, nt, rf, pairs, counts)
    assert counts.tolist() == [0, live] and rf.tolist() == held and read(nt.tolist(), pl.cpu())[0].shape == before[0].shape


@pytest.mark.parametrize("bs,width,dtype", [(1, 8, torch.bfloat16), (16, 24, torch.float32), (16, 1024, torch.bfloat16),
                                            (64, 33, torch.float32), (16, 128, torch.uint8)])
def test_copy(bs, width, dtype):
    g = torch.Generator().manual_seed(bs)
    n = 23
    pool = torch.randint(0, 255, (3, n * bs, width), generator=g).to(dtype)
    order = torch.randperm(n, generator=g)
    pairs = torch.stack([order[:8], order[8:16]], 1).to(torch.int32)
    pairs[2, 0], pairs[3, 1], pairs[4, 0], pairs[5, 1] = -1, n, 2 ** 31 - 1, -2 ** 31
    for count in (None, 7, 0, 100, -4):
        k = 8 if count is None else max(0, min(8, count))
        want = pool.clone().view(3, n, bs, width)
        for i, (a, b) in enumerate(pairs.tolist()):
            if i < k and 0 <= a < n and 0 <= b < n:
                want[:, b] = pool.view(3, n, bs, width)[:, a]
        got = pool.cuda()
        mx.run_pages_copy(got, bs, pairs.cuda(), None if count is None else dev([count, 5]))
        assert torch.equal(got.cpu(), want.view_as(pool))
    # one pool by itself, and pools further apart than they are long
    one = pool[0].cuda()
    mx.run_pages_copy(one, bs, pairs.cuda(), stream=torch.cuda.current_stream())
    far = torch.zeros(3, n * bs + 16, width, dtype=dtype, device="cuda")
    far[:, :n * bs] = pool.cuda()
    mx.run_pages_copy(far[:, :n * bs], bs, pairs.cuda())
    want = pool.clone().view(3, n, bs, width)
    for a, b in pairs.tolist():
        if 0 <= a < n and 0 <= b < n:
            want[:, b] = pool.view(3, n, bs, width)[:, a]
    assert torch.equal(one.cpu(), want[0].view(n * bs, width)) and torch.equal(far[:, :n * bs].cpu(), want.view_as(pool))
    assert not far[:, n * bs:].any()
    with pytest.raises((ValueError, mx.MxfaError)):
        mx.run_pages_copy(got.transpose(1, 2), bs, pairs.cuda())


def test_copy_large_blocks_past_32_bits():
    """Blocks at offsets past 2^32 bytes, of more than one piece."""
    bs, width, n = 64, 1024, 33000
    pool = torch.zeros(n * bs, width, dtype=torch.bfloat16, device="cuda")
    assert pool.numel() * 2 > 2 ** 32
    pool[(n - 1) * bs:] = torch.randn(bs, width, device="cuda").bfloat16()
    mx.run_pages_copy(pool, bs, dev([[n - 1, 3], [n - 2, 5]]))
    assert torch.equal(pool[3 * bs:4 * bs], pool[(n - 1) * bs:]) and not pool[5 * bs:6 * bs].any()


def test_graph():
    """free, fork and copy captured as one step and replayed: the same result each time."""
    r = random.Random(2)
    table, lens, refs, pool = make(r, [100, 55, 30, 9, 80], 16, 60, 8)
    t, ln, rf, pl = dev(table), dev(lens), dev(refs), pool.cuda()
    parents, children, rows = dev([0, 0, 1]), dev([2, 3, 4]), dev([2, 3, 4])
    pairs, status, counts = (torch.zeros(3, 2, dtype=torch.int32, device="cuda"), dev([0] * 3), dev([0, 0]))

    def step():
        mx.run_pages_free(t, 16, ln, rf, rows)
        mx.run_pages_fork(t, 16, ln, rf, parents, children, pairs, status, counts)
        mx.run_pages_copy(pl, 16, pairs, counts)
    step()
    torch.cuda.synchronize()
    want = [x.clone() for x in (t, ln, rf, pl, pairs, status, counts)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for _ in range(3):
        pairs.fill_(-7)
        g.replay()
        torch.cuda.synchronize()
        pl.view(-1)[:4].add_(0.0)
        assert all(torch.equal(a, b) for a, b in zip(want, (t, ln, rf, pl, pairs, status, counts)))
    assert status.tolist() == [0, 0, 0]
