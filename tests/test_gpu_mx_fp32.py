"""The fp32 microscaled cache to fp32's own roundings, where other tests hold both types to
bf16's: the steps of a serving loop over forked pages, and rows beside keys that they do
not see and that are NaN."""
from __future__ import annotations

import math

import pytest
import torch

import mx230_amd as mx
from mx_helpers import MxBatch, parts
from test_gpu_mx_attention import run

pytestmark = pytest.mark.gpu


# A score's partial sums are of size 1 here, so its some 66 independent roundings of up to
# half of 2^-23 move it, and its key's weight, by some sqrt(66 / 3) 2^-24 = 2.8e-7 (rms), and
# the sums over the keys less. Without the last of the three parts of q or p each would be
# off by up to 2^-17, 4.4e-6 rms: in the 2-norm 2^-19 = 1.9e-6 lies between.
NORM = 2.0 ** -19


def off_by(got, want):
    return float((got.double() - want).norm() / want.norm())


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def attention(q, k, v, ln, nh, nkv, hd):
    """One sequence's new rows q [n, nh hd] over its k, v [ln, nkv hd] in 64 bits: the result,
    and what fp32's roundings may move it by (as Batch.tolerance has it)."""
    n, scale = q.shape[0], 1.0 / math.sqrt(hd)
    q = q.double().cpu().view(n, nh, hd)
    k, v = (x.double().cpu().view(ln, nkv, hd) for x in (k, v))
    want, tol = torch.zeros(n, nh, hd, dtype=torch.float64), torch.zeros(n, nh, hd, dtype=torch.float64)
    for h in range(nh):
        kh, vh = k[:, h // (nh // nkv)], v[:, h // (nh // nkv)]
        for i in range(n):
            seen = ln - n + i + 1
            p = torch.softmax(kh[:seen] @ q[i, h] * scale, 0)
            reach = float((kh[:seen].abs() @ q[i, h].abs()).max()) * scale
            want[i, h] = p @ vh[:seen]
            tol[i, h] = (p @ vh[:seen].abs()) * (4 * (hd + 2) * 2.0 ** -24 * reach + 2 * (ln + 64) * 2.0 ** -24) + 1e-30
    return want.flatten(1), tol.flatten(1)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("nh,nkv", [(6, 2), (14, 2)])
def test_steps_over_forked_pages(nh, nkv, bits):
    """A prompt in two chunks, two beams forked from it, some tokens of each."""
    hd, bs, n_blocks = 64, 16, 40
    g = torch.Generator(device="cuda").manual_seed(bits)
    pools = torch.zeros(2, n_blocks, mx.mx_block_bytes(bs, nkv, hd, bits), dtype=torch.uint8, device="cuda")
    table, lens, refs = torch.full((3, 12), -1, dtype=torch.int32, device="cuda"), ints([40, 0, 0]), ints([0] * n_blocks)
    table[0, :5] = ints([30, 7, 39, 2, 11])
    refs[[30, 7, 39, 2, 11]] = 1
    f, factor = mx.rotary_frequencies(hd)

    def step(new):
        n, each = sum(new), lens.tolist()
        cu = ints([0] + torch.tensor(new).cumsum(0).tolist())
        qkv = torch.randn(n, (nh + 2 * nkv) * hd, generator=g, device="cuda")
        q, out = (torch.zeros(n, nh * hd, device="cuda") for _ in range(2))
        print(f"\n[mx fp32 step] {new} lens {each} bits {bits}", flush=True)
        mx.run_cache_append_mx(qkv, q, pools[0], pools[1], bits, table, bs, cu, lens, nh, nkv, hd, frequencies=f, factor=factor)
        mx.run_prefill_batch_mx(q, pools[0], pools[1], bits, out, table, bs, cu, lens, max(new), nh, nkv, hd)
        k, v = (torch.zeros(sum(each), nkv * hd, device="cuda") for _ in range(2))
        mx.run_cache_read_mx(pools[0], pools[1], bits, k, v, table, bs, torch.cat([ints([0]), lens.cumsum(0).to(torch.int32)]),
                             lens, nkv, hd)
        t0 = at = 0
        for m, ln in zip(new, each):
            if m:
                want, tol = attention(q[t0:t0 + m], k[at:at + ln], v[at:at + ln], ln, nh, nkv, hd)
                off = (out[t0:t0 + m].cpu().double() - want).abs()
                assert bool((off <= tol).all()), float((off / tol).max())
                assert off_by(out[t0:t0 + m].cpu(), want) <= NORM
            t0, at = t0 + m, at + ln

    step([40, 0, 0])
    lens[0] = 70
    step([30, 0, 0])
    pairs, status, counts = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), ints([9, 9]), ints([9, 9])
    mx.run_pages_fork(table, bs, lens, refs, ints([0, 0]), ints([1, 2]), pairs, status, counts)
    mx.run_pages_copy(pools, 1, pairs, counts)
    assert status.tolist() == [0, 0] and lens.tolist() == [70, 70, 70]
    for _ in range(12):
        lens.add_(1)
        for s in range(3):
            j = (int(lens[s]) - 1) // bs
            if int(table[s, j]) < 0:
                free = int((refs == 0).nonzero()[0])
                table[s, j] = free
                refs[free] = 1
        step([1, 1, 1])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("pairs", [[(4, 40), (80, 100)], [(40, 3000), (3, 2900)], [(5, 2000)]])
def test_values_a_row_does_not_see(pairs, bits):
    """As the test of that name in both types: rows that see no NaN are as exact as ever."""
    b = MxBatch(pairs, 4, 2, 64, 16, bits, False, seed=12)
    want, mag, wlse, reach = b.attention()
    tol = b.tolerance(want, mag, reach)
    ke, ve = parts(b.kp, 2, 16, 64, bits)[1], parts(b.vp, 2, 16, 64, bits)[1]
    for s, (_, ln) in enumerate(pairs):
        last, one = int(b.rows[s][ln - 1]), int(b.rows[s][ln - 2])
        ve[one // 16, 0, one % 16], ke[last // 16, 1, last % 16] = 255, 255
    out, lse = run(b)
    t0 = 0
    for n, _ in pairs:
        for h in range(4):
            c, fine = slice(h * 64, (h + 1) * 64), n - 2 if h < 2 else n - 1
            off = (out[t0:t0 + fine, c].double() - want[t0:t0 + fine, c]).abs()
            assert bool((off <= tol[t0:t0 + fine, c]).all())
            assert off_by(out[t0:t0 + fine, c], want[t0:t0 + fine, c]) <= NORM
            assert float((lse[t0:t0 + fine, h].double() - wlse[t0:t0 + fine, h]).abs().max()) <= b.lse_tolerance(reach)
            assert bool(torch.isnan(out[t0 + fine:t0 + n, c]).all())
        t0 += n
