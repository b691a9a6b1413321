"""Large calls of the append into a microscaled cache and of the read out of it, whose
threads walk several heads (the launcher gives a thread n_tok U heads / 2^17 of them in the
append, / 2^18 in the read, U being the threads of a token's row): the bytes of small
calls, in which each thread has one."""
from __future__ import annotations

import pytest
import torch

import mx230_amd as mx

pytestmark = pytest.mark.gpu

BS = 16


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pages(lens, g):
    """A table of blocks in any order, and their count."""
    need = [-(-n // BS) for n in lens]
    order = torch.randperm(sum(need) + 3, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table.cuda(), sum(need) + 3


def append_small(qkv, q, kp, vp, bits, table, new, lens, nh, nkv, hd, step, **kw):
    """The same tokens, `step` at a time, each sequence by itself."""
    t0 = 0
    for s, (n, ln) in enumerate(zip(new, lens)):
        for i in range(0, n, step):
            m = min(step, n - i)
            mx.run_cache_append_mx(qkv[t0 + i:t0 + i + m], q[t0 + i:t0 + i + m], kp, vp, bits, table[s:s + 1], BS, ints([0, m]),
                                   ints([ln - n + i + m]), nh, nkv, hd, **kw)
        t0 += n


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("turn", ["halves", "interleaved", "part", "none"])
@pytest.mark.parametrize("nh,nkv,hd,n_tok,each", [
    (14, 2, 128, 3000, 3),   # 14 heads of Q by 3 (the last group has 2), both KV heads (halves; the others by 6)
    (9, 3, 128, 2500, 2),    # 9 by 2, 3 KV heads by 2
    (32, 8, 64, 4100, 6),    # 32 by 6, 8 KV heads by 6
    (5, 1, 64, 20000, 4)])
def test_append(nh, nkv, hd, n_tok, each, turn, bf16, bits):
    units = hd // (16 if turn == "halves" else 8)
    got = n_tok * units * (nh + 2 * nkv) >> 17
    assert got >= each >= 2  # heads to a thread
    assert 250 * units * (nh + 2 * nkv) >> 17 == 0  # and one in the small calls
    g = torch.Generator().manual_seed(n_tok + bits)
    dt = torch.bfloat16 if bf16 else torch.float32
    new = [n_tok // 2, 1, n_tok - n_tok // 2 - 1]
    lens = [n_tok // 2, 700, n_tok]
    table, n_blocks = pages(lens, g)
    qkv = torch.randn(n_tok, (nh + 2 * nkv) * hd, generator=g).to(dt).cuda()
    kw = {}
    if turn != "none":
        dim = hd // 2 if turn == "part" else hd
        kw = dict(frequencies=mx.rotary_frequencies(dim)[0], interleaved=turn == "interleaved", factor=1.25)
    wide = mx.mx_block_bytes(BS, nkv, hd, bits)
    noise = [torch.randint(0, 256, (n_blocks, wide), generator=g, dtype=torch.uint8).cuda() for _ in range(2)]
    want = [x.clone() for x in noise]
    q1 = torch.zeros(n_tok, nh * hd, dtype=dt, device="cuda")
    cu = ints([0, new[0], new[0] + 1, n_tok])
    print(f"\n[append mx] {n_tok} tokens, heads {nh}/{nkv} d {hd} bits {bits} {dt} {turn}: {got} heads a thread", flush=True)
    append_small(qkv, q1, *want, bits, table, new, lens, nh, nkv, hd, 250, **kw)
    for inplace in (False, True):
        pools = [x.clone() for x in noise]
        src = qkv.clone()
        q0 = src[:, :nh * hd] if inplace else torch.zeros_like(q1)
        mx.run_cache_append_mx(src, q0, *pools, bits, table, BS, cu, ints(lens), nh, nkv, hd, **kw)
        torch.cuda.synchronize()
        assert torch.equal(q0, q1) and torch.equal(src[:, nh * hd:], qkv[:, nh * hd:])
        for x, y, z in zip(pools, want, noise):
            assert torch.equal(x, y) and not torch.equal(x, z)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("nkv,hd,n_tok,each", [
    (8, 128, 4000, 3),    # K's and V's 16 heads by 3: a group has heads of both
    (8, 128, 13000, 11),  # by 11: more than the 8 that are loaded together, and 5
    (3, 64, 20000, 3), (2, 64, 40000, 4)])
def test_read(nkv, hd, n_tok, each, bf16, bits):
    got = min(n_tok * (hd // 8) * 2 * nkv >> 18, 2 * nkv)
    assert got >= each >= 2 and 1000 * (hd // 8) * 2 * nkv >> 18 == 0
    g = torch.Generator().manual_seed(n_tok)
    dt = torch.bfloat16 if bf16 else torch.float32
    lens = [n_tok // 3, n_tok - n_tok // 3]
    table, n_blocks = pages(lens, g)
    wide = mx.mx_block_bytes(BS, nkv, hd, bits)
    kp, vp = (torch.randint(0, 256, (n_blocks, wide), generator=g, dtype=torch.uint8).cuda() for _ in range(2))
    k0, v0, k1, v1 = (torch.full((n_tok + 2, nkv * hd), 7.0, dtype=dt, device="cuda") for _ in range(4))
    print(f"\n[read mx] {n_tok} tokens, {nkv} heads d {hd} bits {bits} {dt}: {got} heads a thread", flush=True)
    mx.run_cache_read_mx(kp, vp, bits, k0, v0, table, BS, ints([0, lens[0], n_tok]), ints(lens), nkv, hd)
    t0 = 0
    for s, n in enumerate(lens):
        for i in range(0, n, 1000):
            m = min(1000, n - i)
            mx.run_cache_read_mx(kp, vp, bits, k1[t0 + i:t0 + i + m], v1[t0 + i:t0 + i + m], table[s:s + 1], BS, ints([0, m]),
                                 ints([i + m]), nkv, hd)
        t0 += n
    torch.cuda.synchronize()
    for x, y in ((k0, k1), (v0, v1)):
        # (noise has NaN among its values)
        a, b = (t.view(torch.int16 if bf16 else torch.int32) for t in (x, y))
        assert torch.equal(a, b)
        assert bool((x[n_tok:] == 7.0).all()) and not bool((x[:n_tok] == 7.0).all(1).any())
