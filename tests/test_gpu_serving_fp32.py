"""Append and attention in fp32 one after the other, as exactly as their own roundings
allow: prompts in chunks and single tokens, long enough for keys to be split, against
the whole sequences in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

import mx230_amd as mx
from cache_helpers import turned

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("steps,nh,nkv,bs", [
    ([[100, 37, 5], [1, 40, 1], [1, 1, 64]], 4, 2, 16),      # chunks beside tokens
    ([[600, 20], [1, 300], [1, 1]], 2, 1, 16),
    ([[1], [1], [1]], 14, 2, 1), ([[3000, 500], [1, 1], [70, 1]], 2, 1, 128)])
def test_steps(steps, nh, nkv, bs, interleaved):
    hd, n_seq, g = 64, len(steps[0]), torch.Generator().manual_seed(7)
    f, a = mx.rotary_frequencies(hd, scaling="yarn", factor=8.0, original_length=64)
    ends = [sum(s[i] for s in steps) for i in range(n_seq)]
    wide = max(-(-e // bs) for e in ends)
    n_blocks = n_seq * wide
    table = torch.randperm(n_blocks, generator=g).to(torch.int32).view(n_seq, wide).cuda()
    k, v = (torch.full((n_blocks * bs, nkv * hd), math.nan, device="cuda") for _ in range(2))
    lens, said = [0] * n_seq, [torch.zeros(0, (nh + 2 * nkv) * hd) for _ in range(n_seq)]
    for new in steps:
        qkv = torch.randn(sum(new), (nh + 2 * nkv) * hd, generator=g)
        lens = [x + n for x, n in zip(lens, new)]
        cu, ln = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0] + torch.tensor(new).cumsum(0).tolist(), lens))
        x = qkv.cuda()
        mx.run_cache_append(x, x, k, v, table, bs, cu, ln, nh, nkv, hd, f, interleaved, a)
        out = torch.empty(sum(new), nh * hd, device="cuda")
        mx.run_prefill_batch(x[:, :nh * hd], k, v, out, table, bs, cu, ln, max(new), nh, nkv, hd)
        got, t0 = out.cpu().double(), 0
        for s, n in enumerate(new):
            said[s] = torch.cat([said[s], qkv[t0:t0 + n]])
            whole = said[s].double().view(-1, nh + 2 * nkv, hd)
            at = torch.arange(len(whole))
            t = turned(whole[:, :nh + nkv], at[:, None], f.cpu(), interleaved, a)
            # an element of a turned row: 9 roundings of (|x1| + |x2|) factor (cosine and
            # sine within 6, the products and their sum), as the append's own test counts them
            x = whole[:, :nh + nkv].abs()
            pairs = x.view(*x.shape[:2], hd // 2, 2) if interleaved else x.view(*x.shape[:2], 2, hd // 2).transpose(2, 3)
            size = pairs.sum(-1)
            size = a * (size.repeat_interleave(2, -1) if interleaved else size.repeat(1, 1, 2))
            for h in range(nh):
                c, kv = slice(h * hd, (h + 1) * hd), nh + h // (nh // nkv)
                q, ks, vs = t[-n:, h], t[:, kv], whole[:, kv + nkv]
                hide = at[None] > at[-n:, None]
                p = (q @ ks.T / math.sqrt(hd)).masked_fill(hide, -math.inf).softmax(-1)
                # a score: Q and K off by that, and hd products and sums rounded hd + 2 times
                off = 9 * U * (size[-n:, h] @ ks.abs().T + q.abs() @ size[:, kv].T) + (hd + 2) * U * (q.abs() @ ks.abs().T)
                delta = off.masked_fill(hide, 0.0).amax(-1, keepdim=True) / math.sqrt(hd)
                # a weight moves by e^(2 delta), numerator and sum; sums over the keys, and 64 at the joins
                mag = p @ vs.abs()
                tol = mag * (4 * delta + 2 * (len(whole) + 64) * U) + 1e-30
                err = (got[t0:t0 + n, c] - p @ vs).abs()
                if n == len(whole):
                    # the first position sees itself alone, by a weight of 1: V in its three
                    # parts (2^-9 of the rest each), added twice, and the division
                    tol[0] = 4 * U * vs[0].abs() + 1e-30
                assert bool((err <= tol).all()), (s, h, float((err / tol).max()))
            t0 += n
