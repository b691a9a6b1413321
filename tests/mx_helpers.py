"""What the tests of the microscaled cache share: its format on the CPU in 64 bits, and
a batch of sequences whose cache is in it."""
from __future__ import annotations

import math

import torch

from cache_helpers import Batch

GROUP, LEAST = 32, 10


def levels(bits):
    """Values of the non-negative codes, by code (e4m3 without its NaN, e2m1)."""
    man, bias, n = (3, 7, 127) if bits == 8 else (1, 1, 8)
    got = []
    for c in range(n):
        e, f = c >> man, (c & ((1 << man) - 1)) / (1 << man)
        got.append(f * 2.0 ** (1 - bias) if e == 0 else (1 + f) * 2.0 ** (e - bias))
    return torch.tensor(got, dtype=torch.float64)


def quantised(x, bits):
    """(codes, one to an element, and E) of rows x [..., d], from their values rounded
    to 32 bits; elements above 1.75 2^127 count as that."""
    x = x.float().double()
    x = torch.where(torch.isfinite(x), x.clamp(-1.75 * 2.0 ** 127, 1.75 * 2.0 ** 127), x)
    x = x.unflatten(-1, (-1, GROUP))
    most = x.abs().amax(-1)
    top, lv = (448.0 if bits == 8 else 7.0), levels(bits)
    E = torch.full(most.shape, LEAST, dtype=torch.long)
    for e in range(LEAST, 254):  # the least power that holds the largest element
        E = torch.where(most > top * 2.0 ** (e - 127), e + 1, E)
    bad = ~torch.isfinite(x).all(-1)
    z = torch.where(bad[..., None], torch.zeros_like(x), x) * torch.exp2(127.0 - E.double())[..., None]
    a = z.abs().clamp(max=float(lv[-1]))
    hi = torch.searchsorted(lv, a.contiguous()).clamp(1, lv.numel() - 1)
    down, up = a - lv[hi - 1], lv[hi] - a
    c = torch.where((down < up) | ((down == up) & (hi % 2 == 1)), hi - 1, hi)
    c = c | (torch.signbit(z).long() << (bits - 1))
    return c.flatten(-2), torch.where(bad, 255, E)


def stands_for(codes, E, bits):
    """The values of codes [..., d] with E [..., d / 32], in 64 bits."""
    lv = levels(bits)
    if bits == 8:
        lv = torch.cat([lv, torch.tensor([math.nan], dtype=torch.float64)])
    lv = torch.cat([lv, -lv])
    power = torch.where(E == 255, torch.full((), math.nan, dtype=torch.float64), torch.exp2(E.double() - 127.0))
    return (lv[codes].unflatten(-1, (-1, GROUP)) * power[..., None]).flatten(-2)


def packed(codes, bits):
    """Codes [..., d], one to an element, as bytes."""
    if bits == 8:
        return codes.to(torch.uint8)
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).to(torch.uint8)


def unpacked(b, bits):
    b = b.long()
    return b if bits == 8 else torch.stack([b & 15, b >> 4], -1).flatten(-2)


def parts(pool, nkv, bs, hd, bits):
    """A pool's codes and E as views [blocks, KV head, token, bytes]."""
    cb, sb = hd * bits // 8, hd // GROUP
    return (pool[:, :nkv * bs * cb].unflatten(1, (nkv, bs, cb)),
            pool[:, nkv * bs * cb:nkv * bs * (cb + sb)].unflatten(1, (nkv, bs, sb)))


def block_bytes(bs, nkv, hd, bits):
    return -(-nkv * bs * (hd * bits // 8 + hd // GROUP) // 16) * 16


def held(pool, rows, nkv, bs, hd, bits):
    """The values of a pool's rows (block bs + token), [rows, nkv hd] in 64 bits."""
    codes, E = parts(pool, nkv, bs, hd, bits)
    r = torch.as_tensor(rows, dtype=torch.long)
    c, e = codes[r // bs, :, r % bs], E[r // bs, :, r % bs]
    return stands_for(unpacked(c, bits), e.long(), bits).flatten(1)


class MxBatch(Batch):
    """A Batch whose cache is microscaled: kp and vp are the pools, k and v what they
    hold. Rows that nobody holds are NaN by E and, in 8 bits, by their codes."""

    def __init__(self, pairs, nh, nkv, hd, bs, bits, bf16=True, seed=0, gap=0, **kw):
        super().__init__(pairs, nh, nkv, hd, bs, bf16, seed, **kw)
        self.bits, self.gap = bits, gap
        self.kp, self.k = self.pool(self.k)
        self.vp, self.v = self.pool(self.v)

    def pool(self, x):
        """The pool of rows x, and what it holds of them."""
        nkv, bs, hd, bits = self.nkv, self.bs, self.hd, self.bits
        pool = torch.full((self.n_blocks, block_bytes(bs, nkv, hd, bits) + self.gap), 0xff, dtype=torch.uint8)
        codes, E = parts(pool, nkv, bs, hd, bits)
        x = x.unflatten(1, (nkv, hd)).unflatten(0, (self.n_blocks, bs)).transpose(1, 2)
        c, e = quantised(x, bits)
        fine = e[..., :1] != 255  # (a row is all there or all NaN)
        codes.copy_(torch.where(fine, packed(c, bits), codes))
        E.copy_(e)
        got = stands_for(c, e, bits).transpose(1, 2).flatten(0, 1).flatten(1)
        return pool, got.to(self.dt)  # (exact in either type)

    def again(self):
        """The pools of k and v as they are now."""
        self.kp, self.k = self.pool(self.k)
        self.vp, self.v = self.pool(self.v)
