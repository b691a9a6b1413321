"""What the tests of the paged-cache operators share: a batch of sequences over a
pool with its blocks in any order, and attention in 64 bits."""
from __future__ import annotations

import math

import torch


class Batch:
    """Sequences of (new tokens, length) with their cache, tables and inputs, on the
    CPU in the kernels' type; blocks that nobody holds, and the rows past a
    sequence's end in its last block, are NaN."""

    def __init__(self, pairs, nh, nkv, hd, bs, bf16=True, seed=0, extra_rows=0, wide=0, scale_kv=1.0, spare=5):
        g = torch.Generator().manual_seed(seed)
        self.pairs, self.nh, self.nkv, self.hd, self.bs = pairs, nh, nkv, hd, bs
        self.dt = torch.bfloat16 if bf16 else torch.float32
        need = [-(-max(ln, 0) // bs) for _, ln in pairs]
        self.n_blocks = sum(need) + spare
        order = torch.randperm(self.n_blocks, generator=g).tolist()
        entries = max(max(need), 1) + wide
        self.table = torch.full((len(pairs), entries), -1, dtype=torch.int32)
        self.k, self.v = (torch.full((self.n_blocks * bs, nkv * hd), math.nan, dtype=self.dt) for _ in range(2))
        self.rows = []
        for s, (_, ln) in enumerate(pairs):
            mine = [order.pop() for _ in range(need[s])]
            self.table[s, :need[s]] = torch.tensor(mine, dtype=torch.int32)
            at = torch.arange(max(ln, 0))
            rows = torch.tensor(mine, dtype=torch.long)[at // bs] * bs + at % bs if ln > 0 else at
            for x in (self.k, self.v):
                x[rows] = (torch.randn(len(rows), nkv * hd, generator=g) * scale_kv).to(self.dt)
            self.rows.append(rows)
        self.n_new = sum(n for n, _ in pairs)
        self.n_tok = self.n_new + extra_rows
        self.qkv = torch.randn(self.n_tok, (nh + 2 * nkv) * hd, generator=g).to(self.dt)
        ends = torch.tensor([n for n, _ in pairs]).cumsum(0)
        self.cu_q = torch.cat([torch.zeros(1), ends]).to(torch.int32)
        self.lens = torch.tensor([ln for _, ln in pairs], dtype=torch.int32)
        self.max_q = max(max(n for n, _ in pairs), 1)

    def cuda(self, *names):
        return [getattr(self, n).cuda() for n in names]

    def attention(self, scale=None):
        """(out, sum of |p v|, lse, largest sum of |q k| scale) in 64 bits; rows of
        no sequence are NaN."""
        nh, nkv, hd = self.nh, self.nkv, self.hd
        scale = scale or 1.0 / math.sqrt(hd)
        out, mag = (torch.full((self.n_tok, nh * hd), math.nan, dtype=torch.float64) for _ in range(2))
        lse = torch.full((self.n_tok, nh), math.nan, dtype=torch.float64)
        reach, t0 = 0.0, 0
        for s, (n, ln) in enumerate(self.pairs):
            q = self.qkv[t0:t0 + n, :nh * hd].double().view(n, nh, hd)
            k, v = (x[self.rows[s]].double().view(-1, nkv, hd) for x in (self.k, self.v))
            for h in range(nh):
                kh, vh = k[:, h // (nh // nkv)], v[:, h // (nh // nkv)]
                for i in range(n):
                    seen = max(ln - n + i + 1, 0)
                    c = slice(h * hd, (h + 1) * hd)
                    if seen == 0:
                        out[t0 + i, c], mag[t0 + i, c], lse[t0 + i, h] = 0.0, 0.0, -math.inf
                        continue
                    x = kh[:seen] @ q[i, h] * scale
                    reach = max(reach, float((kh[:seen].abs() @ q[i, h].abs()).max()) * scale)
                    lse[t0 + i, h] = torch.logsumexp(x, 0)
                    p = torch.softmax(x, 0)
                    out[t0 + i, c], mag[t0 + i, c] = p @ vh[:seen], p @ vh[:seen].abs()
            t0 += n
        return out, mag, lse, reach

    def tolerance(self, out, mag, reach):
        """What rounding may do to each output. A score is a sum of hd products
        rounded hd + 2 times at most (2^-24 of `reach` each), which moves every
        weight by e^(2 delta) at most, numerator and sum; a sum over n keys is
        rounded n times and 64 times at the joins. bf16: each weight is also
        rounded to 2^-8 of itself before it meets V, and the result once."""
        longest = max(ln for _, ln in self.pairs)
        delta = (self.hd + 2) * 2.0 ** -24 * reach
        tol = mag * (4 * delta + 2 * (longest + 64) * 2.0 ** -24)
        if self.dt == torch.bfloat16:
            tol = tol + 2.0 ** -8 * (mag + out.abs() + tol)
        return tol + 1e-30

    def lse_tolerance(self, reach):
        longest = max(ln for _, ln in self.pairs)
        # the logarithm's own rounding and that of m ln 2, beside the scores'
        return 2 * (self.hd + 2) * 2.0 ** -24 * reach + (longest + 64) * 2.0 ** -24 + 8 * 2.0 ** -24 * (reach + 12)


def turned(x, positions, frequencies, interleaved=False, factor=1.0, sign=1.0):
    """x [..., d] turned at positions (broadcast against x's other dimensions), in 64
    bits, one pair at a time."""
    y = x.double().clone()
    n = frequencies.numel()
    a = positions.double()[..., None] * frequencies
    c, s = factor * a.cos(), sign * factor * a.sin()
    i, j = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    u, v = x[..., i].double(), x[..., j].double()
    y[..., i], y[..., j] = u * c - v * s, v * c + u * s
    return y


def turned_tolerance(x, want, n, interleaved=False, factor=1.0):
    """cos and sin are within 6 x 2^-24 of the exact ones (the angle and its factor
    rounded once, the series a few times), the two products and their sum are
    rounded once each; bf16: the result once more."""
    i, j = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    tol = torch.zeros_like(want)
    size = (x[..., i].double().abs() + x[..., j].double().abs()) * factor
    tol[..., i] = tol[..., j] = size * 9 * 2.0 ** -24
    if x.dtype == torch.bfloat16:
        tol[..., :2 * n] += 2.0 ** -8 * (want[..., :2 * n].abs() + tol[..., :2 * n])
    return tol
