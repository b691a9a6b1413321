"""Argument checks of the operators around the paged cache and of rotary positions
(no GPU needed, nothing is launched): the status codes of the C ABI, and what the
Python layer refuses."""
from __future__ import annotations

import ctypes
import math
import os
import subprocess

import pytest

import mx230_amd as mx

P = ctypes.c_void_p(4096)  # an aligned address, never read


@pytest.fixture(scope="module")
def lib():
    return mx.load_library()


def code(name):
    return next(k for k, v in mx.STATUS.items() if v == name)


OK, NULL, SHAPE, DTYPE = 0, code("MXFA_ERR_NULL"), code("MXFA_ERR_SHAPE"), code("MXFA_ERR_DTYPE")
UNSUPPORTED, ALIGN, WORKSPACE = code("MXFA_ERR_UNSUPPORTED"), code("MXFA_ERR_ALIGN"), code("MXFA_ERR_WORKSPACE")


def rotary_shape(**kw):
    B, Hq, Hkv, N, d = (kw.get(k, v) for k, v in (("B", 2), ("Hq", 4), ("Hkv", 2), ("N", 10), ("head_dim", 64)))
    base = dict(B=B, Hq=Hq, Hkv=Hkv, N=N, head_dim=d, rotary_dim=d, interleaved=0, inverse=0, dtype=mx.MXFA_BF16,
                pos0=0, factor=1.0, pos_bs=N)
    for t, h in (("q", Hq), ("k", Hkv), ("qo", Hq), ("ko", Hkv)):
        base.update({f"{t}_bs": h * N * d, f"{t}_hs": N * d, f"{t}_ts": d})
    base.update(kw)
    return mx.MxfaRotaryShape(**base)


@pytest.mark.parametrize("kw,want", [
    (dict(), OK), (dict(Hkv=0), OK), (dict(dtype=mx.MXFA_F32), OK), (dict(rotary_dim=2), OK), (dict(rotary_dim=24), OK),
    (dict(dtype=5), DTYPE), (dict(B=0), SHAPE), (dict(N=0), SHAPE), (dict(Hq=0), SHAPE), (dict(Hkv=-1), SHAPE),
    (dict(inverse=2), SHAPE), (dict(interleaved=-1), SHAPE), (dict(rotary_dim=0), SHAPE), (dict(rotary_dim=66), SHAPE),
    (dict(rotary_dim=7), UNSUPPORTED), (dict(head_dim=68, rotary_dim=68), UNSUPPORTED),
    (dict(head_dim=512, rotary_dim=64), UNSUPPORTED), (dict(factor=float("nan")), SHAPE),
    (dict(factor=float("inf")), SHAPE), (dict(pos0=2 ** 31 - 5), SHAPE), (dict(pos0=-7), OK),
    (dict(q_ts=68), ALIGN), (dict(qo_ts=68, qo_hs=680, qo_bs=6800), ALIGN),
    (dict(q_hs=0), OK),                       # an input may repeat rows
    (dict(qo_hs=0), SHAPE), (dict(qo_ts=32), SHAPE),  # an output may not
    (dict(qo_hs=64, qo_ts=64), SHAPE),        # heads over tokens
    (dict(qo_hs=64, qo_ts=512, qo_bs=5120), OK),  # tokens first, columns of wider rows
    (dict(N=1, q_ts=-1, qo_ts=0), OK),        # no stride to a single token
    (dict(B=70000), SHAPE),
    (dict(N=2 ** 29, B=1), SHAPE),            # 4 threads a row: more than a launch counts
])
def test_check_rotary(lib, kw, want):
    assert lib.mxfa_check_rotary(ctypes.byref(rotary_shape(**kw))) == want


def test_rotary_pointers(lib):
    s = rotary_shape()
    run = lib.mxfa_run_rotary
    assert lib.mxfa_check_rotary(None) == NULL
    assert run(ctypes.byref(s), P, None, P, P, None, P, None) == NULL
    assert run(ctypes.byref(s), P, P, P, P, None, None, None) == NULL
    odd = ctypes.c_void_p(4096 + 4)
    assert run(ctypes.byref(s), odd, P, P, P, None, P, None) == ALIGN
    assert run(ctypes.byref(s), P, P, P, P, ctypes.c_void_p(4098), P, None) == ALIGN
    assert run(ctypes.byref(s), P, P, P, P, None, odd, None) == ALIGN
    # an output over its input with other strides, or a row further on
    near = ctypes.c_void_p(4096 + 128)
    assert run(ctypes.byref(s), P, P, near, P, None, P, None) == UNSUPPORTED
    s = rotary_shape(qo_hs=64, qo_ts=256)
    assert run(ctypes.byref(s), P, P, P, P, None, P, None) == UNSUPPORTED


def batch_shape(**kw):
    base = dict(n_tok=8, n_seq=3, max_q=4, n_head=4, n_kv_head=2, head_dim=64, block_size=16, n_blocks=10, max_blocks=5,
                table_stride=5, q_stride=512, kv_stride=128, out_stride=256, dtype=mx.MXFA_BF16, scale=0.0)
    base.update(kw)
    return mx.MxfaBatchShape(**base)


@pytest.mark.parametrize("kw,want", [
    (dict(), OK), (dict(head_dim=128, q_stride=1024, kv_stride=256, out_stride=512), OK),
    (dict(dtype=mx.MXFA_F32), OK), (dict(dtype=9), DTYPE), (dict(n_tok=0), SHAPE), (dict(n_seq=0), SHAPE),
    (dict(max_q=0), SHAPE), (dict(n_head=3), SHAPE), (dict(n_blocks=0), SHAPE), (dict(max_blocks=0), SHAPE),
    (dict(table_stride=4), SHAPE), (dict(block_size=24), UNSUPPORTED), (dict(block_size=0), UNSUPPORTED),
    (dict(block_size=1), OK), (dict(head_dim=32), UNSUPPORTED),
    (dict(head_dim=128, dtype=mx.MXFA_F32, q_stride=1024, kv_stride=256, out_stride=512), UNSUPPORTED),
    (dict(q_stride=128), SHAPE), (dict(kv_stride=64), SHAPE), (dict(out_stride=128), SHAPE),
    (dict(q_stride=513), ALIGN), (dict(kv_stride=132), ALIGN), (dict(out_stride=260), ALIGN),
    (dict(scale=-1.0), SHAPE), (dict(scale=float("inf")), SHAPE), (dict(n_tok=2 ** 31 - 1), SHAPE),
])
def test_check_batch(lib, kw, want):
    s = batch_shape(**kw)
    assert lib.mxfa_check_batch(ctypes.byref(s)) == want
    assert (lib.mxfa_prefill_batch_workspace_bytes(ctypes.byref(s)) > 0) == (want == OK)


def test_prefill_batch_pointers(lib):
    s = batch_shape()
    n = lib.mxfa_prefill_batch_workspace_bytes(ctypes.byref(s))
    run = lib.mxfa_run_prefill_batch
    odd = ctypes.c_void_p(4096 + 8)
    args = [P, P, P, P, None, P, P, P, P, n, None]
    for i in (0, 1, 2, 3, 8):
        for bad, want in ((None, NULL), (odd, ALIGN)):
            assert run(ctypes.byref(s), *(bad if j == i else a for j, a in enumerate(args))) == want
    for i in (5, 6, 7):
        for bad, want in ((None, NULL), (ctypes.c_void_p(4097), ALIGN)):
            assert run(ctypes.byref(s), *(bad if j == i else a for j, a in enumerate(args))) == want
    assert run(ctypes.byref(s), P, P, P, P, ctypes.c_void_p(4098), P, P, P, P, n, None) == ALIGN
    assert run(ctypes.byref(s), P, P, P, P, None, P, P, P, P, n - 1, None) == WORKSPACE


def test_append_arguments(lib):
    run = lib.mxfa_run_cache_append

    def go(rot, s=None, frequencies=P, **kw):
        s = s or batch_shape(**kw)
        return run(ctypes.byref(s), ctypes.byref(mx.MxfaAppendRotary(*rot, frequencies)), P, P, P, P, P, P, None, None)
    assert run(ctypes.byref(batch_shape()), None, P, P, P, P, P, P, P, None) == NULL
    assert go((64, 0, 1.0)) == NULL  # lens
    assert go((64, 0, 1.0), frequencies=None) == NULL
    assert go((64, 0, 1.0), q_stride=256) == SHAPE  # no room for K and V beside Q
    assert go((65, 0, 1.0)) == SHAPE
    assert go((63, 0, 1.0)) == UNSUPPORTED
    assert go((64, 2, 1.0)) == SHAPE
    assert go((64, 0, math.nan)) == SHAPE
    assert go((0, 0, 1.0), frequencies=None, head_dim=12, q_stride=96, kv_stride=24, out_stride=48) == UNSUPPORTED
    assert go((64, 0, 1.0), n_tok=2 ** 29) == SHAPE


def test_append_over_its_input(lib):
    """q_out may be qkv or other columns of its rows; otherwise it lies apart."""
    def go(off, stride, n_tok=4):  # (bf16, 4/2 heads of 64: Q 512 bytes, a row of qkv 1024)
        s = batch_shape(n_tok=n_tok, n_head=4, n_kv_head=2, head_dim=64, q_stride=1024, out_stride=stride, kv_stride=128)
        base = 1 << 20
        return lib.mxfa_run_cache_append(ctypes.byref(s), ctypes.byref(mx.MxfaAppendRotary(64, 0, 1.0, P)),
                                         ctypes.c_void_p(base), ctypes.c_void_p(base + off), P, P, P, P, P, None)
    for off, stride, n in ((512, 1024, 4), (-256, 1024, 4), (0, 512, 4), (1024, 512, 4), (16, 1024, 4), (1536 + 16, 1024, 4),
                           (2048 + 512, 1024, 4), (512, 512, 1), (16, 256, 1), (-16, 256, 1)):
        assert go(off, stride, n) == UNSUPPORTED, (off, stride, n)


def pages_shape(**kw):
    base = dict(n_seq=3, max_blocks=5, table_stride=5, block_size=16, n_blocks=10)
    base.update(kw)
    return mx.MxfaPagesShape(**base)


@pytest.mark.parametrize("kw,want", [
    (dict(), OK), (dict(n_seq=0), SHAPE), (dict(n_seq=70000), SHAPE), (dict(max_blocks=0), SHAPE),
    (dict(table_stride=4), SHAPE), (dict(n_blocks=0), SHAPE), (dict(n_blocks=2 ** 30 + 1), SHAPE),
    (dict(block_size=12), UNSUPPORTED), (dict(block_size=-16), UNSUPPORTED)])
def test_check_pages(lib, kw, want):
    assert lib.mxfa_check_pages(ctypes.byref(pages_shape(**kw))) == want


def test_pages_arguments(lib):
    s = ctypes.byref(pages_shape())
    far = ctypes.c_void_p(1 << 20)
    assert lib.mxfa_run_pages_free(s, P, P, P, None, 1, None) == NULL
    assert lib.mxfa_run_pages_free(s, P, P, P, P, -1, None) == SHAPE
    assert lib.mxfa_run_pages_free(s, P, P, P, P, 0, None) == OK  # nothing to do
    assert lib.mxfa_run_pages_fork(s, P, P, P, P, P, -1, P, P, P, None) == SHAPE
    assert lib.mxfa_run_pages_fork(s, P, P, P, P, P, 1, None, P, P, None) == NULL
    assert lib.mxfa_run_pages_compact(s, P, P, P, P, 4, far, P, P, None) == SHAPE
    assert lib.mxfa_run_pages_compact(s, P, P, P, P, 5, P, P, P, None) == UNSUPPORTED  # counts over counts
    assert lib.mxfa_run_pages_compact(s, P, P, P, P, 5, ctypes.c_void_p(4097), P, P, None) == ALIGN
    # a new table over the old one in any way but as the same rows
    assert lib.mxfa_run_pages_compact(s, P, P, P, P, 6, far, P, P, None) == UNSUPPORTED
    assert lib.mxfa_run_pages_compact(s, P, P, P, ctypes.c_void_p(4096 + 40), 5, far, P, P, None) == UNSUPPORTED
    copy = lib.mxfa_run_pages_copy
    assert copy(P, 1, 0, 10, 0, P, 1, None, None) == SHAPE
    assert copy(P, 1, 0, 10, 24, P, 1, None, None) == ALIGN
    assert copy(None, 1, 0, 10, 32, P, 1, None, None) == NULL
    assert copy(P, 1, 0, 10, 32, None, 1, None, None) == NULL
    assert copy(P, 2, 300, 10, 32, P, 1, None, None) == SHAPE   # pools over each other
    assert copy(P, 2, 328, 10, 32, P, 1, None, None) == ALIGN
    assert copy(P, 1, 0, 10, 32, P, 0, None, None) == OK
    assert copy(P, 1, 0, 10, 32, P, 1, ctypes.c_void_p(4097), None) == ALIGN


def test_python_layer_refuses_host_tensors():
    import torch
    z = torch.zeros
    q, i = z(1, 2, 4, 64), z(4, dtype=torch.int32)
    f = mx.rotary_frequencies(64, device="cpu")[0]
    for call in (lambda: mx.run_rotary(q, None, q, None, f),
                 lambda: mx.run_cache_append(z(4, 256), z(4, 128), z(16, 64), z(16, 64), i[None], 16, i, i, 2, 1, 64),
                 lambda: mx.run_prefill_batch(z(4, 128), z(16, 64), z(16, 64), z(4, 128), i[None], 16, i, i, 1, 2, 1, 64),
                 lambda: mx.run_pages_free(i[None], 16, i, i, i),
                 lambda: mx.run_pages_fork(i[None], 16, i, i, i, i, i[None], i, i),
                 lambda: mx.run_pages_compact(i[None], 16, i, i, i[None], i, i[None], i),
                 lambda: mx.run_pages_copy(z(32, 64), 16, i[None])):
        with pytest.raises(ValueError, match="device tensor"):
            call()
    with pytest.raises(TypeError):
        mx.run_rotary(None, None, None, None, f)


def test_numbers_past_32_bits():
    with pytest.raises(ValueError, match="past 32 bits"):
        mx.prefill_batch_workspace_bytes(2 ** 32 + 1, 1, 1, 4, 2)
    with pytest.raises(TypeError):
        mx.prefill_batch_workspace_bytes(5, 1, 1.5, 4, 2)
    assert mx.prefill_batch_workspace_bytes(150000, 150000, 1, 1, 1) > 0


def test_rotary_frequencies():
    """The formulas, from their definitions in Python's own arithmetic."""
    f, a = mx.rotary_frequencies(8, 10000.0, device="cpu")
    assert f.tolist() == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-15) and a == 1.0
    f, a = mx.rotary_frequencies(8, 10000.0, "linear", 4.0, device="cpu")
    assert f.tolist() == pytest.approx([0.25, 0.025, 0.0025, 0.00025], rel=1e-15) and a == 1.0
    f, a = mx.rotary_frequencies(8, 10000.0, "base", 16.0, device="cpu")
    assert f[0] == 1.0 and f[3].item() == pytest.approx(0.001 / 16.0, rel=1e-14)
    f, a = mx.rotary_frequencies(64, 10000.0, "yarn", 8.0, 4096, device="cpu")
    plain = mx.rotary_frequencies(64, device="cpu")[0]
    turns = (4096 * plain / (2 * math.pi)).tolist()
    assert a == pytest.approx(0.1 * math.log(8.0) + 1.0)
    for x, y, t in zip(f.tolist(), plain.tolist(), turns):
        if t > 40:
            assert x == y
        if t < 0.7:
            assert x == pytest.approx(y / 8, rel=1e-15)
        assert y / 8 <= x <= y
    for bad in (dict(dim=7), dict(dim=0), dict(dim=8, base=1.0), dict(dim=8, scaling="cubic"),
                dict(dim=2, scaling="base"), dict(dim=8, factor=0.5)):
        with pytest.raises(ValueError):
            mx.rotary_frequencies(device="cpu", **bad)


def test_binding_leaves_other_calls():
    import torch
    c = mx._calls()
    z = torch.zeros(2, 2)
    for name, n in (("rotary", 10), ("cache_append", 14), ("prefill_batch", 15), ("pages_free", 5), ("pages_fork", 9),
                    ("pages_compact", 8), ("pages_copy", 4)):
        assert getattr(c, name)(*[z] * n) is NotImplemented
        assert getattr(c, name)() is NotImplemented
        assert getattr(c, name)(*[None] * n) is NotImplemented


@pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc"), reason="hipcc is not installed")
def test_batch_items():
    """The items of the attention over a batch (fa_batch_items.h) on the host, with
    sanitizers: they cover every row and stage once, their workspace slots are
    theirs alone, and nothing lies outside the buffers, whatever the arrays hold."""
    here = os.path.join(os.path.dirname(os.path.abspath(__file__)), "sanitize")
    subprocess.run(["make", "-s", "-j8", "-C", here], check=True)
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=1", UBSAN_OPTIONS="print_stacktrace=1")
    r = subprocess.run([os.path.join(here, "_build", "items_selftest")], capture_output=True, text=True, env=env,
                       timeout=300)
    assert r.returncode == 0 and "all checks passed" in r.stdout, r.stderr[-2000:]
