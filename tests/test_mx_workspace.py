"""The workspaces of batches whose tables may have any width (no GPU needed)."""
from __future__ import annotations

import ctypes

import pytest

import mx230_amd as mx
from test_cache_abi import batch_shape, lib  # noqa: F401

WIDTHS = (1, 64, 500, 1000, 1280, 1281, 1344, 2304, 3000, 8000, 32000, 60000, 100000, 130880, 1 << 17, 1 << 20)


def most(lib, bits, n_tok, n_seq, max_q, nh, nkv, hd, bf16):  # noqa: F811
    """The most that a call of such a batch needs, by the widths that are taken."""
    got = 0
    for wide in WIDTHS:
        for bs in (1, 16):
            n = -(-wide // bs)
            s = batch_shape(n_tok=n_tok, n_seq=n_seq, max_q=max_q, n_head=nh, n_kv_head=nkv, head_dim=hd, block_size=bs,
                            max_blocks=n, table_stride=n, q_stride=nh * hd, out_stride=nh * hd,
                            kv_stride=1 << 20 if bits else nkv * hd, dtype=mx.MXFA_BF16 if bf16 else mx.MXFA_F32)
            got = max(got, lib.mxfa_prefill_batch_mx_workspace_bytes(ctypes.byref(s), bits) if bits else
                      lib.mxfa_prefill_batch_workspace_bytes(ctypes.byref(s)))
    return got


@pytest.mark.parametrize("bits", [0, 8, 4])
@pytest.mark.parametrize("bf16,hd", [(True, 64), (True, 128), (False, 64)])
@pytest.mark.parametrize("n_tok,n_seq,max_q", [
    (1, 1, 1), (64, 64, 1), (600, 4, 512), (2000, 1, 2000), (1000, 3, 4096),
    # so many sequences (nearly all without new tokens) that the widest tables are refused
    (60, 1 << 20, 1), (60, (1 << 20) + 1, 1), (60, 1300000, 2), (1, 1 << 22, 1), (50, 30000000, 1)])
def test_enough_for_any_table(lib, n_tok, n_seq, max_q, bf16, hd, bits):  # noqa: F811
    for nh, nkv in ((14, 2), (32, 8), (1, 1), (40, 1)):
        need = most(lib, bits, n_tok, n_seq, max_q, nh, nkv, hd, bf16)
        got = (mx.prefill_batch_mx_workspace_bytes(n_tok, n_seq, max_q, nh, nkv, hd, bf16, bits) if bits else
               mx.prefill_batch_workspace_bytes(n_tok, n_seq, max_q, nh, nkv, hd, bf16))
        assert got >= need, (nh, nkv, need, got)
        assert (got > 0) == (need > 0)
