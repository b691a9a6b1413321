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
