"""Argument checks of the microscaled cache's calls (no GPU needed, nothing is launched),
and its format on the CPU, by hand and against torch's 8-bit type."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import mx230_amd as mx
from mx_helpers import levels, quantised, stands_for
from test_cache_abi import ALIGN, DTYPE, NULL, OK, SHAPE, UNSUPPORTED, WORKSPACE, P, batch_shape, lib  # noqa: F401

BASE = 1 << 30
FAR = [BASE + (i << 28) for i in range(1, 6)]  # nothing is there
WIDE = {8: 2112, 4: 1088}  # blocks of 16 tokens of 2 heads of 64


def shape(bits, **kw):
    return batch_shape(**{"kv_stride": WIDE[bits], **kw})


@pytest.mark.parametrize("args,want", [
    ((16, 2, 64, 8), 2112), ((16, 2, 64, 4), 1088), ((16, 8, 128, 4), 8704), ((1, 1, 64, 4), 48), ((1, 1, 32, 8), 48),
    ((2, 3, 96, 4), 320), ((16, 2, 64, 5), 0), ((16, 2, 64, 16), 0), ((16, 2, 80, 8), 0), ((16, 2, 288, 8), 0), ((16, 2, 0, 8), 0),
    ((12, 2, 64, 8), 0), ((0, 2, 64, 8), 0), ((16, 0, 64, 8), 0), ((1 << 24, 1, 128, 8), 0), ((1 << 24, 1, 64, 8), 1107296256),
    ((1 << 25, 1, 32, 4), 0)])
def test_block_bytes(lib, args, want):  # noqa: F811
    assert lib.mxfa_mx_block_bytes(*args) == want
    if want:
        assert mx.mx_block_bytes(*args) == want
    else:
        with pytest.raises(ValueError):
            mx.mx_block_bytes(*args)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("kw,want", [
    (dict(), OK), (dict(dtype=mx.MXFA_F32, out_stride=256), OK), (dict(dtype=9), DTYPE), (dict(n_tok=0), SHAPE), (dict(max_q=0), SHAPE),
    (dict(block_size=24), UNSUPPORTED), (dict(kv_stride=1024), SHAPE), (dict(kv_stride=4098), ALIGN), (dict(kv_stride=4096), OK),
    (dict(head_dim=96, q_stride=768, out_stride=384, kv_stride=4096), UNSUPPORTED), (dict(head_dim=128, q_stride=1024, out_stride=512, kv_stride=8192), OK),
    (dict(head_dim=128, dtype=mx.MXFA_F32, q_stride=1024, out_stride=512, kv_stride=8192), UNSUPPORTED),
    (dict(scale=-1.0), SHAPE), (dict(scale=math.nan), SHAPE), (dict(n_head=5), SHAPE), (dict(q_stride=516), ALIGN),
    (dict(out_stride=128), SHAPE), (dict(n_blocks=1 << 30, block_size=16, kv_stride=4096), SHAPE)])
def test_check_batch(lib, bits, kw, want):  # noqa: F811
    s = shape(bits, **kw)
    assert lib.mxfa_check_batch_mx(ctypes.byref(s), bits) == want
    assert (lib.mxfa_prefill_batch_mx_workspace_bytes(ctypes.byref(s), bits) > 0) == (want == OK)


def test_bits(lib):  # noqa: F811
    s = shape(8)
    r = mx.MxfaAppendRotaryMx(0, 0, 1.0, None)
    for bits in (0, 1, 2, 5, 16, -8):
        assert lib.mxfa_check_batch_mx(ctypes.byref(s), bits) == UNSUPPORTED
        assert lib.mxfa_run_cache_append_mx(ctypes.byref(s), bits, ctypes.byref(r), P, P, P, P, P, P, P, None) == UNSUPPORTED
        assert lib.mxfa_run_cache_read_mx(ctypes.byref(s), bits, P, P, P, P, P, P, P, None) == UNSUPPORTED
    assert lib.mxfa_check_batch_mx(None, 8) == NULL


def attend(lib, s, bits, q=FAR[0], k=FAR[1], v=FAR[2], out=FAR[3], lse=None, ws=FAR[4], n=None):  # noqa: F811
    need = lib.mxfa_prefill_batch_mx_workspace_bytes(ctypes.byref(s), bits)
    p = [None if x is None else ctypes.c_void_p(x) for x in (q, k, v, out, lse)]
    return lib.mxfa_run_prefill_batch_mx(ctypes.byref(s), bits, *p, P, P, P, ctypes.c_void_p(ws), need if n is None else n, None)


@pytest.mark.parametrize("bits", [8, 4])
def test_attention_buffers(lib, bits):  # noqa: F811
    s = shape(bits)
    need, w = lib.mxfa_prefill_batch_mx_workspace_bytes(ctypes.byref(s), bits), WIDE[bits]
    assert attend(lib, s, bits, n=need - 1) == WORKSPACE
    assert attend(lib, s, bits, q=None) == NULL and attend(lib, s, bits, k=FAR[1] + 8) == ALIGN
    for at in (FAR[1], FAR[2]):
        for off in (0, 10 * w - 16, w // 2 // 16 * 16, -512 * 7 - 16):
            assert attend(lib, s, bits, out=at + off) == UNSUPPORTED, off
        assert attend(lib, s, bits, ws=at + 16) == UNSUPPORTED and attend(lib, s, bits, lse=at + 4) == UNSUPPORTED
    assert attend(lib, s, bits, out=FAR[0] + 16) == UNSUPPORTED and attend(lib, s, bits, ws=FAR[0]) == UNSUPPORTED
    # in the gap that wider blocks leave, columns of equal rows
    s = shape(bits, kv_stride=4096, out_stride=2048)
    assert attend(lib, s, bits, out=FAR[1] + 16) == UNSUPPORTED


@pytest.mark.parametrize("bits", [8, 4])
def test_append_and_read_buffers(lib, bits):  # noqa: F811
    s, w = shape(bits), WIDE[bits]
    p = [ctypes.c_void_p(x) for x in FAR]
    f = ctypes.c_void_p(4096)
    run = lib.mxfa_run_cache_append_mx

    def append(rot=(64, 0, 1.0, f), q_out=p[1], qkv=p[0], k=p[2], sh=s, v=p[3]):
        r = mx.MxfaAppendRotaryMx(*rot)
        return run(ctypes.byref(sh), bits, ctypes.byref(r), qkv, q_out, k, v, P, P, P, None)
    assert append(rot=(64, 0, 1.0, None)) == NULL and append(rot=(66, 0, 1.0, f)) == SHAPE
    assert append(rot=(7, 0, 1.0, f)) == UNSUPPORTED and append(rot=(64, 2, 1.0, f)) == SHAPE
    for x in (math.inf, math.nan, 1e300):
        assert append(rot=(64, 0, x, f)) == SHAPE
    assert append(rot=(64, 0, 1.0, ctypes.c_void_p(4100))) == ALIGN
    assert append(q_out=None) == NULL and append(k=ctypes.c_void_p(FAR[2] + 4)) == ALIGN
    assert append(q_out=ctypes.c_void_p(FAR[0] + 512)) == UNSUPPORTED  # over K's columns
    for at in (FAR[2], FAR[2] + w // 32 * 16, FAR[2] + 9 * w + 16):  # V, q_out or qkv over K
        assert append(v=ctypes.c_void_p(at)) == UNSUPPORTED and append(q_out=ctypes.c_void_p(at)) == UNSUPPORTED
        assert append(qkv=ctypes.c_void_p(at)) == UNSUPPORTED
    assert append(q_out=ctypes.c_void_p(FAR[3] + 16)) == UNSUPPORTED
    assert append(sh=shape(bits, q_stride=256)) == SHAPE and append(sh=shape(bits, kv_stride=w - 16)) == SHAPE
    assert append(sh=shape(bits, head_dim=48, kv_stride=4096)) == UNSUPPORTED

    def read(ko=FAR[2], vo=FAR[3], sh=s):
        return lib.mxfa_run_cache_read_mx(ctypes.byref(sh), bits, p[0], p[1], None if ko is None else ctypes.c_void_p(ko),
                                          ctypes.c_void_p(vo), P, P, P, None)
    assert read(ko=None) == NULL and read(vo=FAR[3] + 2) == ALIGN
    for a, b in ((FAR[2], FAR[2]), (FAR[2], FAR[2] + 128), (FAR[2], FAR[2] + 512 * 7), (FAR[0], FAR[3]), (FAR[2], FAR[1] + 9 * w),
                 (FAR[0] - 512 * 7 - 16, FAR[3])):
        assert read(a, b) == UNSUPPORTED
    assert read(sh=shape(bits, out_stride=64)) == SHAPE
    assert lib.mxfa_run_cache_read_mx(None, bits, P, P, P, P, P, P, P, None) == NULL


def test_python_refuses():
    x = torch.zeros(8, 512, dtype=torch.bfloat16)
    pool, t = torch.zeros(4, 2112, dtype=torch.uint8), torch.zeros(1, 4, dtype=torch.int32)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensor"):
        mx.run_cache_append_mx(x, x, pool, pool, 8, t, 16, i, i[:1], 4, 2)
    with pytest.raises(ValueError, match="device tensor"):
        mx.run_cache_read_mx(pool, pool, 8, x, x, t, 16, i, i[:1], 2)
    with pytest.raises(ValueError, match="device tensor"):
        mx.run_prefill_batch_mx(x, pool, pool, 8, x, t, 16, i, i[:1], 1, 4, 2)
    assert mx.prefill_batch_mx_workspace_bytes(64, 64, 1, 32, 8, 128, True, 4) > 0
    assert mx.prefill_batch_mx_workspace_bytes(64, 64, 1, 32, 8, 96, True, 4) == 0
    with pytest.raises(ValueError):
        mx.prefill_batch_mx_workspace_bytes(64, 64, 1, 32, 8, 128, True, 6)


def test_format_by_hand():
    """The oracle's own: the codes of 4 bits in order, ties to the even one, the power
    that 7 and what is just above it get, and 8 bits as torch rounds them."""
    assert levels(4).tolist() == [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0] and levels(8)[-1] == 448.0
    x = torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0] + [0.0] * 24])
    c, e = quantised(x, 4)
    assert c[0, :8].tolist() == [0, 2, 2, 4, 4, 6, 6, 7] and e.tolist() == [[127]]
    assert quantised(x * (1 + 2.0 ** -22), 4)[1].tolist() == [[128]] and quantised(x / 2, 4)[1].tolist() == [[126]]
    g = torch.Generator().manual_seed(0)
    x = torch.randn(50, 64, generator=g)
    c, e = quantised(x, 8)
    p = torch.exp2(127.0 - e.float()).repeat_interleave(32, -1)
    assert torch.equal(c.to(torch.uint8), (x * p).to(torch.float8_e4m3fn).view(torch.uint8))
    assert torch.equal(stands_for(c, e, 8).float(), (x * p).to(torch.float8_e4m3fn).float() / p)
    assert bool((x * p).abs().unflatten(-1, (-1, 32)).amax(-1).gt(224).all())


@pytest.mark.parametrize("bf16,hd", [(True, 64), (True, 128), (False, 64)])
def test_workspace_for_tables_of_any_width(lib, bf16, hd):  # noqa: F811
    """prefill_batch_mx_workspace_bytes holds what a call needs, whatever its table."""
    for n_tok, n_seq, max_q in ((1, 1, 1), (64, 64, 1), (96, 24, 4), (500, 1, 500), (700, 4, 512), (2000, 1, 2000), (4000, 8, 700),
                                (1000, 3, 4096), (30, 30, 7)):
        for nh, nkv in ((14, 2), (32, 8), (4, 1), (40, 1)):
            got = mx.prefill_batch_mx_workspace_bytes(n_tok, n_seq, max_q, nh, nkv, hd, bf16, 4)
            for wide in (1, 64, 256, 500, 700, 1000, 1280, 1281, 1500, 2000, 2304, 2305, 3000, 4000, 6000, 10 ** 4, 10 ** 5, 10 ** 6):
                for bs in (1, 16):
                    n = -(-wide // bs)
                    s = shape(4, n_tok=n_tok, n_seq=n_seq, max_q=max_q, n_head=nh, n_kv_head=nkv, head_dim=hd, block_size=bs,
                              max_blocks=n, table_stride=n, q_stride=nh * hd, out_stride=nh * hd, kv_stride=1 << 20,
                              dtype=mx.MXFA_BF16 if bf16 else mx.MXFA_F32)
                    need = lib.mxfa_prefill_batch_mx_workspace_bytes(ctypes.byref(s), 4)
                    assert 0 < need <= got, (n_tok, n_seq, max_q, nh, nkv, wide, bs, need, got)
