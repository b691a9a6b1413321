"""Attention over a microscaled cache whose KV heads hold the same rows and whose
sequences share blocks (each block `times` in a row of the table), so that work-groups
have many stages of keys and the 64-bit result is still quickly made."""
from __future__ import annotations

import math

import torch

import mx230_amd as mx
from mx_helpers import block_bytes, packed, parts, quantised, stands_for

TYPES = [(True, 64, 8), (True, 64, 4), (True, 128, 8), (True, 128, 4), (False, 64, 8), (False, 64, 4)]
BS = 16
# The launcher gives the few-row form 256 work-groups for all KV heads, which cut the
# sequences' stages of 64 keys into equal runs, shared by the waves of each (8, beside
# chunks 4): KV heads and single tokens by which a run is one sequence or a good part
# of one. A chunk alone has the many-row form to itself.
FORMS = {"one": (64, [1]), "few": (8, [1] * 31 + [2]), "both": (8, [1] * 31 + [40]), "many": (2, [300])}


class Shared:
    def __init__(self, k, v, q, news, nkv, bits, bf16, times=1):
        """k, v: rows [L, d] of every head; q: [new tokens, heads, d]; news: the sequences'
        new tokens."""
        self.news, self.nkv, self.bits, self.times = news, nkv, bits, times
        self.dt = torch.bfloat16 if bf16 else torch.float32
        n, hd = k.shape
        self.hd, self.nh, self.lens = hd, q.shape[1], n * times
        self.q = q.to(self.dt)
        need = n // BS
        order = torch.randperm(need, generator=torch.Generator().manual_seed(n))
        self.pools, held = [], []
        for x in (k, v):
            pool = torch.zeros(need, block_bytes(BS, nkv, hd, bits), dtype=torch.uint8)
            codes, E = parts(pool, nkv, BS, hd, bits)
            c, e = quantised(x, bits)
            codes[order] = packed(c, bits).view(need, 1, BS, -1)
            E[order] = e.to(torch.uint8).view(need, 1, BS, -1)
            self.pools.append(pool)
            held.append(stands_for(c, e, bits))
        self.k, self.v = held  # in 64 bits
        self.table = order.to(torch.int32).repeat(len(news), times)

    def run(self, **kw):
        n_tok, nh, hd = self.q.shape
        ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in
                ([0] + torch.tensor(self.news).cumsum(0).tolist(), [self.lens] * len(self.news))]
        out = torch.full((n_tok, nh * hd), 7.0, dtype=self.dt, device="cuda")
        lse = torch.full((n_tok, nh), 7.0, device="cuda")
        print(f"\n[prefill batch mx] {len(self.news)} sequences, new {self.news[-1]} of {self.lens} heads {nh}/{self.nkv} d {hd} "
              f"bits {self.bits} {self.dt}", flush=True)
        mx.run_prefill_batch_mx(self.q.flatten(1).cuda(), *(p.cuda() for p in self.pools), self.bits, out, self.table.cuda(), BS,
                                *ints, max(self.news), nh, self.nkv, hd, lse=lse, **kw)
        torch.cuda.synchronize()
        return out.cpu(), lse.cpu()

    def check(self, out, lse, few=0.0):
        """Against 64 bits. A score is a sum of hd products rounded hd + 2 times at most, 2^-24
        of the sum of their sizes each, which moves every weight by e^(2 delta) at most,
        numerator and sum; a sum over n keys is rounded n times, and 64 times at the
        joins; bf16: each weight is rounded by 2^-8 of itself before it meets V, and the
        result once. `few`: an absolute error beside those."""
        hd, scale = self.hd, 1.0 / math.sqrt(self.hd)
        q = self.q.double()
        t0 = 0
        for n in self.news:
            for i in range(n):
                # all keys `times`, but for the last n - 1 - i positions once less
                count = torch.full((self.k.shape[0],), float(self.times), dtype=torch.float64)
                count[self.k.shape[0] - (n - 1 - i):] -= 1.0
                x = q[t0 + i] @ self.k.T * scale + torch.log(count)
                there = x > -1e30  # (keys past fp32's range, at the other end, weigh nothing)
                x = torch.where(there, x, -math.inf)
                p = torch.softmax(x, -1)
                want, mag = p @ self.v, p @ self.v.abs()
                reach = (q[t0 + i].abs() @ self.k.abs().T * scale).where(there, torch.zeros(())).amax(-1)
                delta = (hd + 2) * 2.0 ** -24 * reach[:, None]
                tol = mag * (4 * delta + 2 * (self.lens + 64) * 2.0 ** -24)
                if self.dt == torch.bfloat16:
                    tol = tol + 2.0 ** -8 * (mag + want.abs() + tol)
                off = (out[t0 + i].double().view(-1, hd) - want).abs()
                assert bool((off <= tol + few).all()), (t0 + i, float((off / (tol + few)).max()))
                wide = 2 * delta[:, 0] + (self.lens + 64) * 2.0 ** -24 + 8 * 2.0 ** -24 * (reach + 12)
                assert bool(((lse[t0 + i].double() - torch.logsumexp(x, -1)).abs() <= wide).all()), t0 + i
            t0 += n
