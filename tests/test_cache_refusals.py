"""More argument checks of the operators around the paged cache (no GPU needed, nothing
is launched): outputs that lie over inputs, tables of the largest width, rows that do
not begin on 16 bytes, and frequencies worked out by hand."""
from __future__ import annotations

import ctypes

import pytest
import torch

import mx230_amd as mx
from mx230_amd.autograd import _rows16
from test_cache_abi import OK, SHAPE, UNSUPPORTED, P, batch_shape, lib, pages_shape  # noqa: F401

BASE = 1 << 30
FAR = [BASE + (i << 28) for i in range(1, 6)]  # nothing is there


def attend(lib, s, q=FAR[0], k=FAR[1], v=FAR[2], out=FAR[3], lse=None, ws=FAR[4]):
    """The status of a call that has to be refused."""
    n = lib.mxfa_prefill_batch_workspace_bytes(ctypes.byref(s))
    p = [None if x is None else ctypes.c_void_p(x) for x in (q, k, v, out, lse)]
    return lib.mxfa_run_prefill_batch(ctypes.byref(s), *p, P, P, P, ctypes.c_void_p(ws), n, None)


# bf16, 4/2 heads of 64, 8 tokens, a pool of 160 rows: a row of Q or out 512 bytes, of K or V 256
@pytest.mark.parametrize("q_stride,out_stride,off", [
    (512, 512, 16), (512, 512, -16), (512, 512, 1024), (512, 512, 256), (256, 512, 0), (512, 256, 0), (512, 256, 1024 * 7 + 496),
    (256, 512, -1024 * 7), (512, 512, 1024 + 256), (512, 512, 1024 - 496), (256, 264, 512 * 7)])
def test_output_over_the_queries(lib, q_stride, out_stride, off):  # noqa: F811
    s = batch_shape(q_stride=q_stride, out_stride=out_stride)
    assert attend(lib, s, out=FAR[0] + off) == UNSUPPORTED


@pytest.mark.parametrize("off,n_tok", [(16, 1), (-16, 1), (496, 1), (-496, 1)])
def test_output_over_one_query_row(lib, off, n_tok):  # noqa: F811
    s = batch_shape(n_tok=n_tok, n_seq=1, max_q=1)
    assert attend(lib, s, out=FAR[0] + off) == UNSUPPORTED


def test_output_over_the_caches(lib):  # noqa: F811
    for which in ("k", "v"):
        at = dict(k=FAR[1], v=FAR[2])[which]
        for off in (0, 256 * 159 + 240, 16, 256 * 80, -512 * 7 - 16):
            assert attend(lib, batch_shape(), out=at + off) == UNSUPPORTED, off
        # columns of the same wide rows that the cache has itself
        s = batch_shape(kv_stride=1024, out_stride=1024)
        for off in (0, 240, -496, 2048 * 5 + 240, 2048 * 159 + 16):
            assert attend(lib, s, out=at + off) == UNSUPPORTED, off
        # one token's row inside a wide cache row's columns
        s = batch_shape(n_tok=1, n_seq=1, max_q=1, kv_stride=1024)
        assert attend(lib, s, out=at + 2048 * 7 + 240) == UNSUPPORTED


def test_lse_and_workspace_over_the_rest(lib):  # noqa: F811
    s = batch_shape()
    n = lib.mxfa_prefill_batch_workspace_bytes(ctypes.byref(s))
    for x in (FAR[0], FAR[1], FAR[2], FAR[3]):
        assert attend(lib, s, ws=x) == UNSUPPORTED
        assert attend(lib, s, ws=x - n // 16 * 16 + 16) == UNSUPPORTED
        assert attend(lib, s, lse=x + 4) == UNSUPPORTED
    assert attend(lib, s, lse=FAR[4]) == UNSUPPORTED
    assert attend(lib, s, lse=FAR[4] + n - 4) == UNSUPPORTED


def test_widest_table(lib):  # noqa: F811
    """A table's entries are counted in ints, a work-group past the last."""
    for wide, want in ((2 ** 31 - 1, SHAPE), (2 ** 31 - 255, SHAPE), (2 ** 31 - 256, OK)):
        s = pages_shape(n_seq=1, max_blocks=wide, table_stride=wide)
        assert lib.mxfa_check_pages(ctypes.byref(s)) == want


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_rows_begin_on_16_bytes(dt):
    base = torch.zeros(2 * 3 * 5 * 64 + 8, dtype=dt)
    for off in range(8):
        x = base[off:off + 2 * 3 * 5 * 64].view(2, 3, 5, 64)
        y = _rows16(x)
        assert y.data_ptr() % 16 == 0 and torch.equal(x, y) and (y is x) == (x.data_ptr() % 16 == 0)


def test_yarn_between_its_ends():
    """dim 64, base 10^4, 4096 positions: a pair that turns 32 times is number 10.5 and
    one that turns once 22.5, so the ramp goes from 10 to 23: pair i is divided by 8 to
    (i - 10) / 13."""
    f, _ = mx.rotary_frequencies(64, 10000.0, "yarn", 8.0, 4096, device="cpu")
    for i in (10, 11, 12, 16, 20, 22, 23):
        part = (i - 10) / 13
        assert f[i].item() == pytest.approx(10.0 ** (-i / 8) * (1 - part * 7 / 8), rel=1e-14)
    assert f[16].item() == pytest.approx(0.01 * 62 / 104, rel=1e-14)
    assert f[9].item() == pytest.approx(10.0 ** (-9 / 8), rel=1e-14)
    assert f[24].item() == pytest.approx(10.0 ** -3 / 8, rel=1e-14)
