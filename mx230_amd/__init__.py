"""MI355X-native flash-attention training path (forward O + LSE, FA-2 backward).

The compute lives in ``libmxfa.so`` (HIP kernels for gfx950 behind the C ABI of
``include/mxfa.h``, built from ``mx230_amd/csrc``). This module is the host-side
mirror of the reference crate's Rust wrappers
(02-flash-attention/src/main.rs:32-210): the same entry points, the same argument
meaning (caller-owned device buffers, ``n`` implied by the shapes, ``causal``
flag), the same ownership (the caller allocates O, LSE, Delta, dQ, dK, dV) and the
same "wrappers only enqueue work" contract. Where the reference panics on a
launch failure, these raise :class:`MxfaError`.

PyTorch is only plumbing here: tensors provide device memory and the current
stream. There is no CPU or PyTorch fallback: if ``libmxfa.so`` is missing or the
tensors are not on a GPU, every call raises.

Tensor layouts (contiguous): Q, O, dO, dQ ``[B, Hq, N, d]``; K, V, dK, dV
``[B, Hkv, N, d]``; LSE, Delta ``[B, Hq, N]`` float32. A 2-D ``[N, d]`` tensor is
read as B = H = 1, i.e. the reference's single-head layout.
"""
from __future__ import annotations

import ctypes
import os
import warnings
from dataclasses import dataclass

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libmxfa.so")
# the kernels: one gfx950 code object the library loads per device
CODE_OBJECT_PATH = os.path.join(_HERE, "mxfa_gfx950.hsaco")
# the same kernels with per-work-group timestamps in the backward bodies
# (make -C mx230_amd/csrc timeline; read with probe_wg_times)
TIMELINE_CODE_OBJECT_PATH = os.path.join(_HERE, "mxfa_gfx950_timeline.hsaco")

MXFA_F32, MXFA_BF16 = 0, 1

STATUS = {
    0: "MXFA_OK",
    -1: "MXFA_ERR_NULL",
    -2: "MXFA_ERR_SHAPE",
    -3: "MXFA_ERR_DTYPE",
    -4: "MXFA_ERR_UNSUPPORTED",
    -5: "MXFA_ERR_ALIGN",
    -6: "MXFA_ERR_LAUNCH",
    -7: "MXFA_ERR_DEVICE",
    -8: "MXFA_ERR_WORKSPACE",
    -9: "MXFA_ERR_CODE_OBJECT",
    -10: "MXFA_ERR_SCRATCH",
}

# Every symbol include/mxfa.h declares (the tests check the library exports them).
EXPORTS = (
    "mxfa_version", "mxfa_strerror", "mxfa_init", "mxfa_shutdown", "mxfa_set_code_object",
    "mxfa_check_code_object", "mxfa_check_shape",
    "mxfa_run_flash", "mxfa_run_flash_lse", "mxfa_run_preprocess", "mxfa_run_bwd_dq",
    "mxfa_run_bwd_dkv", "mxfa_run_bwd_flash", "mxfa_run_bwd_dq_delta", "mxfa_run_bwd", "mxfa_bwd_one_launch", "mxfa_bwd_workspace_bytes",
    "mxfa_run_bwd_dkv_ws", "mxfa_run_bwd_ws", "mxfa_run_bwd_naive",
    "mxfa_naive_scratch_bytes", "mxfa_run_naive_fwd", "mxfa_check_prefill", "mxfa_run_prefill",
    "mxfa_run_prefill_paged", "mxfa_prefill_workspace_bytes", "mxfa_run_prefill_ws", "mxfa_run_prefill_paged_ws",
    "mxfa_set_bwd_options", "mxfa_get_bwd_options", "mxfa_bwd_delta_fallbacks", "mxfa_bwd_reduce_timeouts",
    "mxfa_run_bwd_noalloc", "mxfa_bwd_noalloc_scratch_bytes",
    "mxfa_check_rotary", "mxfa_run_rotary", "mxfa_check_batch", "mxfa_prefill_batch_workspace_bytes",
    "mxfa_run_prefill_batch", "mxfa_run_cache_append", "mxfa_check_pages", "mxfa_run_pages_free",
    "mxfa_run_pages_fork", "mxfa_run_pages_compact", "mxfa_run_pages_copy",
    "mxfa_mx_block_bytes", "mxfa_run_cache_append_mx", "mxfa_run_cache_read_mx", "mxfa_check_batch_mx",
    "mxfa_prefill_batch_mx_workspace_bytes", "mxfa_run_prefill_batch_mx",
)
# Every symbol include/mxfa_probes.h declares.
PROBE_EXPORTS = (
    "mxfa_probe_sink_len", "mxfa_probe_mfma", "mxfa_probe_mfma32", "mxfa_probe_mix", "mxfa_probe_read",
    "mxfa_probe_copy", "mxfa_probe_dq_atomic", "mxfa_probe_wg_times",
)


class MxfaError(RuntimeError):
    """A non-zero status from libmxfa."""

    def __init__(self, func: str, status: int, text: str):
        super().__init__(f"{func}: {STATUS.get(status, status)} ({text})")
        self.status = status


class MxfaShape(ctypes.Structure):
    _fields_ = [("B", ctypes.c_int), ("Hq", ctypes.c_int), ("Hkv", ctypes.c_int), ("N", ctypes.c_int),
                ("d", ctypes.c_int), ("causal", ctypes.c_int), ("dtype", ctypes.c_int),
                ("scale", ctypes.c_float)]


class MxfaBwdOptions(ctypes.Structure):
    _fields_ = [("one_launch", ctypes.c_int), ("delta_wait_us", ctypes.c_int), ("reduce_wait_us", ctypes.c_int)]


class MxfaPrefillShape(ctypes.Structure):
    _fields_ = [("n_tok", ctypes.c_int), ("n_head", ctypes.c_int), ("n_kv_head", ctypes.c_int),
                ("head_dim", ctypes.c_int), ("pos0", ctypes.c_int), ("q_stride", ctypes.c_int),
                ("kv_stride", ctypes.c_int), ("out_stride", ctypes.c_int), ("dtype", ctypes.c_int),
                ("scale", ctypes.c_float)]


class MxfaRotaryShape(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("B", "Hq", "Hkv", "N", "head_dim", "rotary_dim", "interleaved", "inverse",
                                            "dtype", "pos0")] + [("factor", ctypes.c_float)] + \
               [(n, ctypes.c_longlong) for n in ("q_bs", "q_hs", "q_ts", "k_bs", "k_hs", "k_ts", "qo_bs", "qo_hs",
                                                 "qo_ts", "ko_bs", "ko_hs", "ko_ts", "pos_bs")]


class MxfaBatchShape(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("n_tok", "n_seq", "max_q", "n_head", "n_kv_head", "head_dim", "block_size",
                                            "n_blocks", "max_blocks", "table_stride", "q_stride", "kv_stride",
                                            "out_stride", "dtype")] + [("scale", ctypes.c_float)]


class MxfaAppendRotary(ctypes.Structure):
    _fields_ = [("rotary_dim", ctypes.c_int), ("interleaved", ctypes.c_int), ("factor", ctypes.c_float),
                ("frequencies", ctypes.c_void_p)]


class MxfaAppendRotaryMx(ctypes.Structure):
    _fields_ = [("rotary_dim", ctypes.c_int), ("interleaved", ctypes.c_int), ("factor", ctypes.c_double),
                ("frequencies", ctypes.c_void_p)]


class MxfaPagesShape(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("n_seq", "max_blocks", "table_stride", "block_size", "n_blocks")]


_lib = None


def load_library(path: str | None = None):
    """Loads libmxfa.so (raises if it has not been built)."""
    global _lib
    if path is None and _lib is not None:
        return _lib
    p = path or LIB_PATH
    # torch first: libmxfa then binds to the HIP runtime torch already loaded, so
    # the device pointers and streams it receives from torch are valid for it
    # (loading libmxfa first would pull in a second HIP runtime)
    try:
        import torch  # noqa: F401
    except ImportError:
        pass
    if not os.path.exists(p):
        raise ImportError(f"{p} is missing: build it with `make -C mx230_amd/csrc` "
                          "(or __graft_entry__.build()); there is no fallback path")
    if path is None and not os.path.exists(CODE_OBJECT_PATH):
        raise ImportError(f"{CODE_OBJECT_PATH} (the kernels) is missing: build it with "
                          "`make -C mx230_amd/csrc`; there is no fallback path")
    lib = ctypes.CDLL(p)
    vp, sp, fp = ctypes.c_void_p, ctypes.POINTER(MxfaShape), ctypes.c_void_p
    lib.mxfa_version.restype = ctypes.c_int
    lib.mxfa_strerror.restype = ctypes.c_char_p
    lib.mxfa_strerror.argtypes = [ctypes.c_int]
    lib.mxfa_init.argtypes = [ctypes.c_int]
    lib.mxfa_set_code_object.argtypes = [ctypes.c_char_p]
    lib.mxfa_check_code_object.argtypes = [ctypes.c_char_p]
    lib.mxfa_check_shape.argtypes = [sp]
    lib.mxfa_run_flash.argtypes = [sp, vp, vp, vp, vp, vp]
    lib.mxfa_run_flash_lse.argtypes = [sp, vp, vp, vp, vp, fp, vp]
    lib.mxfa_run_preprocess.argtypes = [sp, vp, vp, fp, vp]
    lib.mxfa_run_bwd_dq.argtypes = [sp, vp, vp, vp, vp, fp, fp, vp, vp]
    lib.mxfa_run_bwd_dkv.argtypes = [sp, vp, vp, vp, vp, fp, fp, vp, vp, vp]
    lib.mxfa_run_bwd_flash.argtypes = [sp, vp, vp, vp, vp, fp, fp, vp, vp, vp, vp]
    lib.mxfa_run_bwd.argtypes = [sp, vp, vp, vp, vp, vp, fp, fp, vp, vp, vp, vp]
    lib.mxfa_run_bwd_dq_delta.argtypes = [sp, vp, vp, vp, vp, vp, fp, fp, vp, vp]
    lib.mxfa_run_bwd_naive.argtypes = [sp, vp, vp, vp, vp, fp, fp, vp, vp, vp, vp]
    lib.mxfa_bwd_one_launch.argtypes = [sp]
    lib.mxfa_bwd_workspace_bytes.argtypes = [sp]
    lib.mxfa_bwd_workspace_bytes.restype = ctypes.c_size_t
    lib.mxfa_run_bwd_dkv_ws.argtypes = [sp, vp, vp, vp, vp, fp, fp, vp, vp, vp, ctypes.c_size_t, vp]
    lib.mxfa_run_bwd_ws.argtypes = [sp, vp, vp, vp, vp, vp, fp, fp, vp, vp, vp, vp, ctypes.c_size_t, vp]
    lib.mxfa_run_bwd_noalloc.argtypes = [sp, vp, vp, vp, vp, vp, fp, fp, vp, vp, vp, vp]
    lib.mxfa_bwd_noalloc_scratch_bytes.argtypes = []
    lib.mxfa_bwd_noalloc_scratch_bytes.restype = ctypes.c_size_t
    lib.mxfa_naive_scratch_bytes.argtypes = [sp]
    lib.mxfa_naive_scratch_bytes.restype = ctypes.c_size_t
    lib.mxfa_run_naive_fwd.argtypes = [sp, vp, vp, vp, fp, vp, vp]
    pp = ctypes.POINTER(MxfaPrefillShape)
    lib.mxfa_check_prefill.argtypes = [pp]
    lib.mxfa_run_prefill.argtypes = [pp, vp, vp, vp, vp, vp]
    lib.mxfa_run_prefill_paged.argtypes = [pp, vp, vp, vp, vp, vp, ctypes.c_int, vp]
    lib.mxfa_prefill_workspace_bytes.argtypes = [pp]
    lib.mxfa_prefill_workspace_bytes.restype = ctypes.c_size_t
    lib.mxfa_run_prefill_ws.argtypes = [pp, vp, vp, vp, vp, vp, ctypes.c_size_t, vp]
    lib.mxfa_run_prefill_paged_ws.argtypes = [pp, vp, vp, vp, vp, vp, ctypes.c_int, vp, ctypes.c_size_t, vp]
    lib.mxfa_probe_sink_len.argtypes = []
    lib.mxfa_probe_mfma.argtypes = [ctypes.c_int, ctypes.c_int, fp, ctypes.POINTER(ctypes.c_double), vp]
    lib.mxfa_probe_mfma32.argtypes = [ctypes.c_int, fp, ctypes.POINTER(ctypes.c_double), vp]
    lib.mxfa_probe_mix.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_int, fp, ctypes.POINTER(ctypes.c_double), vp]
    lib.mxfa_probe_wg_times.argtypes = [vp, ctypes.c_size_t, ctypes.POINTER(ctypes.c_size_t)]
    lib.mxfa_probe_read.argtypes = [vp, ctypes.c_size_t, fp, vp]
    lib.mxfa_probe_copy.argtypes = [vp, vp, ctypes.c_size_t, vp]
    lib.mxfa_probe_dq_atomic.argtypes = [fp, ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                         ctypes.POINTER(ctypes.c_double), vp]
    rp, bp, gp = (ctypes.POINTER(t) for t in (MxfaRotaryShape, MxfaBatchShape, MxfaPagesShape))
    ci, cl = ctypes.c_int, ctypes.c_longlong
    lib.mxfa_check_rotary.argtypes = [rp]
    lib.mxfa_run_rotary.argtypes = [rp, vp, vp, vp, vp, vp, vp, vp]
    lib.mxfa_check_batch.argtypes = [bp]
    lib.mxfa_prefill_batch_workspace_bytes.argtypes = [bp]
    lib.mxfa_prefill_batch_workspace_bytes.restype = ctypes.c_size_t
    lib.mxfa_run_prefill_batch.argtypes = [bp, vp, vp, vp, vp, vp, vp, vp, vp, vp, ctypes.c_size_t, vp]
    lib.mxfa_run_cache_append.argtypes = [bp, ctypes.POINTER(MxfaAppendRotary), vp, vp, vp, vp, vp, vp, vp, vp]
    lib.mxfa_check_pages.argtypes = [gp]
    lib.mxfa_run_pages_free.argtypes = [gp, vp, vp, vp, vp, ci, vp]
    lib.mxfa_run_pages_fork.argtypes = [gp, vp, vp, vp, vp, vp, ci, vp, vp, vp, vp]
    lib.mxfa_run_pages_compact.argtypes = [gp, vp, vp, vp, vp, ci, vp, vp, vp, vp]
    lib.mxfa_run_pages_copy.argtypes = [vp, ci, cl, ci, cl, vp, ci, vp, vp]
    lib.mxfa_mx_block_bytes.argtypes = [ci, ci, ci, ci]
    lib.mxfa_mx_block_bytes.restype = ctypes.c_size_t
    lib.mxfa_run_cache_append_mx.argtypes = [bp, ci, ctypes.POINTER(MxfaAppendRotaryMx), vp, vp, vp, vp, vp, vp, vp, vp]
    lib.mxfa_run_cache_read_mx.argtypes = [bp, ci, vp, vp, vp, vp, vp, vp, vp, vp]
    lib.mxfa_check_batch_mx.argtypes = [bp, ci]
    lib.mxfa_prefill_batch_mx_workspace_bytes.argtypes = [bp, ci]
    lib.mxfa_prefill_batch_mx_workspace_bytes.restype = ctypes.c_size_t
    lib.mxfa_run_prefill_batch_mx.argtypes = [bp, ci, vp, vp, vp, vp, vp, vp, vp, vp, vp, ctypes.c_size_t, vp]
    op = ctypes.POINTER(MxfaBwdOptions)
    lib.mxfa_set_bwd_options.argtypes = [op]
    lib.mxfa_get_bwd_options.argtypes = [op]
    lib.mxfa_bwd_delta_fallbacks.argtypes = [ctypes.POINTER(ctypes.c_ulonglong)]
    lib.mxfa_bwd_reduce_timeouts.argtypes = [ctypes.POINTER(ctypes.c_ulonglong)]
    for name in EXPORTS + PROBE_EXPORTS:
        if name not in ("mxfa_version", "mxfa_strerror", "mxfa_bwd_workspace_bytes",
                        "mxfa_naive_scratch_bytes", "mxfa_bwd_noalloc_scratch_bytes",
                        "mxfa_prefill_workspace_bytes", "mxfa_prefill_batch_workspace_bytes",
                        "mxfa_mx_block_bytes", "mxfa_prefill_batch_mx_workspace_bytes"):
            getattr(lib, name).restype = ctypes.c_int
    if path is None:
        _lib = lib
    return lib


_native = None


class _NoBinding:
    """In the place of csrc/binding.cpp where it cannot be loaded: leaves every
    call to the Python path."""

    @staticmethod
    def _other(*args):
        return NotImplemented
    attention_fwd = attention_bwd = prefill = _other
    rotary = rotary_embedding = cache_append = prefill_batch = pages_free = pages_fork = pages_compact = pages_copy = _other
    cache_append_mx = cache_read_mx = prefill_batch_mx = _other


def _calls():
    """The call path in C++ (csrc/binding.cpp), bound to the loaded libmxfa: its
    functions take plain GPU tensors on torch's current stream and return
    NotImplemented for every other call, which the Python below then takes.
    Where the module is not built or cannot be loaded (another torch), it
    warns once, and every call goes the Python way."""
    global _native
    if _native is None:
        lib = load_library()
        _torch()  # whose libraries the module is linked with
        try:
            from . import _binding as ext
        except ImportError as e:
            warnings.warn(f"{os.path.join(_HERE, '_binding.so')} cannot be loaded ({e}); calls cost 10-30 us more on "
                          "the host. Build it with `make -C mx230_amd/csrc` (or __graft_entry__.build())",
                          RuntimeWarning, stacklevel=3)
            _native = _NoBinding
            return _native
        ext.bind(*(ctypes.cast(getattr(lib, f), ctypes.c_void_p).value for f in (
            "mxfa_run_flash_lse", "mxfa_run_bwd_ws", "mxfa_bwd_workspace_bytes", "mxfa_run_prefill",
            "mxfa_run_prefill_ws", "mxfa_run_prefill_paged", "mxfa_run_prefill_paged_ws", "mxfa_run_rotary",
            "mxfa_run_cache_append", "mxfa_run_prefill_batch", "mxfa_prefill_batch_workspace_bytes",
            "mxfa_run_pages_free", "mxfa_run_pages_fork", "mxfa_run_pages_compact", "mxfa_run_pages_copy",
            "mxfa_mx_block_bytes", "mxfa_run_cache_append_mx", "mxfa_run_cache_read_mx", "mxfa_run_prefill_batch_mx",
            "mxfa_prefill_batch_mx_workspace_bytes")))
        _native = ext
    return _native


def _check(func: str, rc: int):
    if rc != 0:
        raise MxfaError(func, rc, load_library().mxfa_strerror(rc).decode())


def _invoke(func: str, args):
    _check(func, getattr(load_library(), func)(*args))


@dataclass(frozen=True)
class Shape:
    B: int
    Hq: int
    Hkv: int
    N: int
    d: int
    causal: bool
    bf16: bool
    scale: float = 0.0

    def c(self) -> MxfaShape:
        return MxfaShape(self.B, self.Hq, self.Hkv, self.N, self.d, int(self.causal),
                         MXFA_BF16 if self.bf16 else MXFA_F32, self.scale)


# --------------------------------------------------------------- torch glue --

def _torch():
    import torch
    return torch


def _dims(t, name):
    if t.dim() == 2:
        return 1, 1, t.shape[0], t.shape[1]
    if t.dim() == 4:
        return tuple(t.shape)
    raise ValueError(f"{name}: expected [N, d] or [B, H, N, d], got {tuple(t.shape)}")


def _ptr(t, name, dtype):
    torch = _torch()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name}: must be a device tensor (got {t.device}); there is no CPU path")
    if t.dtype != dtype:
        raise ValueError(f"{name}: dtype {t.dtype}, expected {dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    return ctypes.c_void_p(t.data_ptr())


def _stream(stream):
    torch = _torch()
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def _scratch(nbytes: int, device, stream):
    """Device bytes for a launch on `stream` (None: the current one), of that stream's
    own memory: what another stream's pool gives may still be in use there."""
    torch = _torch()
    if stream is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    if not isinstance(stream, torch.cuda.Stream):  # anything with a cuda_stream, as _stream takes it
        stream = torch.cuda.ExternalStream(stream.cuda_stream, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(nbytes, dtype=torch.uint8, device=device)


def shape_of(q, k, causal: bool, scale: float = 0.0) -> Shape:
    """Shape of an attention call from Q [B,Hq,N,d] and K [B,Hkv,N,d]."""
    torch = _torch()
    B, Hq, N, d = _dims(q, "q")
    Bk, Hkv, Nk, dk = _dims(k, "k")
    if (Bk, Nk, dk) != (B, N, d):
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} disagree")
    if q.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"dtype {q.dtype} not supported (float32 or bfloat16)")
    return Shape(B, Hq, Hkv, N, d, bool(causal), q.dtype == torch.bfloat16, float(scale))


def _expect(t, name, shape4, dtype):
    dims = _dims(t, name)
    if tuple(dims) != tuple(shape4):
        raise ValueError(f"{name}: shape {tuple(t.shape)} does not match {tuple(shape4)}")
    return _ptr(t, name, dtype)


def _io(sh: Shape):
    torch = _torch()
    dt = torch.bfloat16 if sh.bf16 else torch.float32
    qs = (sh.B, sh.Hq, sh.N, sh.d)
    ks = (sh.B, sh.Hkv, sh.N, sh.d)
    return dt, qs, ks


def _vec_ptr(t, name, sh: Shape):
    torch = _torch()
    if t.numel() != sh.B * sh.Hq * sh.N:
        raise ValueError(f"{name}: expected {sh.B * sh.Hq * sh.N} elements, got {t.numel()}")
    return _ptr(t, name, torch.float32)


# ------------------------------------------- reference-shaped entry points --

def _call_flash(q, k, v, o, causal: bool, scale: float = 0.0, stream=None):
    sh = shape_of(q, k, causal, scale)
    dt, qs, ks = _io(sh)
    args = (_expect(q, "q", qs, dt), _expect(k, "k", ks, dt), _expect(v, "v", ks, dt),
            _expect(o, "o", qs, dt))
    return "mxfa_run_flash", (ctypes.byref(sh.c()), *args, _stream(stream))


def run_flash(q, k, v, o, causal: bool, scale: float = 0.0, stream=None):
    """Forward, O only (main.rs:68-88)."""
    _invoke(*_call_flash(q, k, v, o, causal, scale, stream))


def _call_flash_lse(q, k, v, o, lse, causal: bool, scale: float = 0.0, stream=None):
    sh = shape_of(q, k, causal, scale)
    dt, qs, ks = _io(sh)
    args = (_expect(q, "q", qs, dt), _expect(k, "k", ks, dt), _expect(v, "v", ks, dt),
            _expect(o, "o", qs, dt), _vec_ptr(lse, "lse", sh))
    return "mxfa_run_flash_lse", (ctypes.byref(sh.c()), *args, _stream(stream))


def run_flash_lse(q, k, v, o, lse, causal: bool, scale: float = 0.0, stream=None):
    """Forward with the log-sum-exp the backward needs (main.rs:102-123)."""
    _invoke(*_call_flash_lse(q, k, v, o, lse, causal, scale, stream))


def _call_preprocess(do, o, delta, stream=None):
    sh = shape_of(do, do, False)
    dt, qs, _ = _io(sh)
    args = (_expect(do, "do", qs, dt), _expect(o, "o", qs, dt), _vec_ptr(delta, "delta", sh))
    return "mxfa_run_preprocess", (ctypes.byref(sh.c()), *args, _stream(stream))


def run_preprocess(do, o, delta, stream=None):
    """Delta = rowsum(dO * O) (main.rs:126-143)."""
    _invoke(*_call_preprocess(do, o, delta, stream))


def _bwd_args(q, k, v, do, lse, delta, causal, scale):
    sh = shape_of(q, k, causal, scale)
    dt, qs, ks = _io(sh)
    args = [_expect(q, "q", qs, dt), _expect(k, "k", ks, dt), _expect(v, "v", ks, dt),
            _expect(do, "do", qs, dt), _vec_ptr(lse, "lse", sh), _vec_ptr(delta, "delta", sh)]
    return sh, dt, qs, ks, args


def _call_bwd_flash(q, k, v, do, lse, delta, dq, dk, dv, causal: bool, scale: float = 0.0,
                  stream=None):
    sh, dt, qs, ks, args = _bwd_args(q, k, v, do, lse, delta, causal, scale)
    args += [_expect(dq, "dq", qs, dt), _expect(dk, "dk", ks, dt), _expect(dv, "dv", ks, dt)]
    return "mxfa_run_bwd_flash", (ctypes.byref(sh.c()), *args, _stream(stream))


def run_bwd_flash(q, k, v, do, lse, delta, dq, dk, dv, causal: bool, scale: float = 0.0,
                  stream=None):
    """Tiled atomic-free backward: dK/dV pass then dQ pass (main.rs:179-210).
    Outputs are overwritten."""
    _invoke(*_call_bwd_flash(q, k, v, do, lse, delta, dq, dk, dv, causal, scale, stream))


def _call_bwd(q, k, v, o, do, lse, delta, dq, dk, dv, causal: bool, scale: float = 0.0, stream=None):
    sh = shape_of(q, k, causal, scale)
    dt, qs, ks = _io(sh)
    args = [_expect(q, "q", qs, dt), _expect(k, "k", ks, dt), _expect(v, "v", ks, dt), _expect(o, "o", qs, dt),
            _expect(do, "do", qs, dt), _vec_ptr(lse, "lse", sh), _vec_ptr(delta, "delta", sh),
            _expect(dq, "dq", qs, dt), _expect(dk, "dk", ks, dt), _expect(dv, "dv", ks, dt)]
    return "mxfa_run_bwd", (ctypes.byref(sh.c()), *args, _stream(stream))


def run_bwd(q, k, v, o, do, lse, delta, dq, dk, dv, causal: bool, scale: float = 0.0, stream=None):
    """The whole backward from O (mxfa_run_bwd): the dQ work computes
    Delta = rowsum(dO * O) itself and writes it to ``delta`` for the dK/dV
    work (run_preprocess + run_bwd_flash with the preprocess launch folded in);
    one launch for bf16 (bwd_one_launch) and small fp32 grids, else two.
    Outputs are overwritten."""
    _invoke(*_call_bwd(q, k, v, o, do, lse, delta, dq, dk, dv, causal, scale, stream))


def bwd_one_launch(q, k, causal: bool) -> bool:
    """True if run_bwd runs the backward as one launch for this shape
    (mxfa_bwd_one_launch; set_bwd_options(one_launch=False) selects two
    launches)."""
    sh = shape_of(q, k, causal)
    return bool(load_library().mxfa_bwd_one_launch(ctypes.byref(sh.c())))


def get_bwd_options() -> dict:
    """The one-launch backward's process-wide settings (mxfa_get_bwd_options)."""
    o = MxfaBwdOptions()
    _check("mxfa_get_bwd_options", load_library().mxfa_get_bwd_options(ctypes.byref(o)))
    return {"one_launch": bool(o.one_launch), "delta_wait_us": o.delta_wait_us, "reduce_wait_us": o.reduce_wait_us}


def set_bwd_options(one_launch: bool | None = None, delta_wait_us: int | None = None,
                    reduce_wait_us: int | None = None) -> dict:
    """Changes the given settings (mxfa_set_bwd_options) and returns the
    previous ones. one_launch=False: always two launches; delta_wait_us < 0:
    the dK/dV work-groups never wait for Delta and compute it themselves;
    reduce_wait_us: the bound of a GQA split's reduce wait (>= 0)."""
    old = get_bwd_options()
    o = MxfaBwdOptions(int(old["one_launch"] if one_launch is None else one_launch),
                       old["delta_wait_us"] if delta_wait_us is None else int(delta_wait_us),
                       old["reduce_wait_us"] if reduce_wait_us is None else int(reduce_wait_us))
    _check("mxfa_set_bwd_options", load_library().mxfa_set_bwd_options(ctypes.byref(o)))
    return old


def bwd_delta_fallbacks() -> int:
    """Delta blocks the one-launch backward computed in its dK/dV work-groups
    on the current device since load (mxfa_bwd_delta_fallbacks; synchronise the
    launches of interest first)."""
    n = ctypes.c_ulonglong(0)
    _check("mxfa_bwd_delta_fallbacks", load_library().mxfa_bwd_delta_fallbacks(ctypes.byref(n)))
    return int(n.value)


def bwd_reduce_timeouts() -> int:
    """Work-groups of the one-launch backward that add a GQA split's partial
    sums and whose wait for them ran out (their dK/dV rows are NaN), on the
    current device since load (mxfa_bwd_reduce_timeouts; 0 in normal operation;
    synchronise the launches of interest first)."""
    n = ctypes.c_ulonglong(0)
    _check("mxfa_bwd_reduce_timeouts", load_library().mxfa_bwd_reduce_timeouts(ctypes.byref(n)))
    return int(n.value)


def bwd_workspace_bytes(q, k, causal: bool) -> int:
    """Bytes of workspace run_bwd_ws / run_bwd_dkv_ws can use for this shape
    (mxfa_bwd_workspace_bytes): nonzero only for GQA shapes whose dK/dV pass
    splits each group's query heads over several work-groups."""
    sh = shape_of(q, k, causal)
    return int(load_library().mxfa_bwd_workspace_bytes(ctypes.byref(sh.c())))


def _ws_args(workspace):
    if workspace is None:
        return [None, 0]
    torch = _torch()
    if workspace.device.type != "cuda" or not workspace.is_contiguous():
        raise ValueError("workspace: must be a contiguous device tensor")
    return [ctypes.c_void_p(workspace.data_ptr()), workspace.numel() * workspace.element_size()]


def _call_bwd_ws(q, k, v, o, do, lse, delta, dq, dk, dv, workspace, causal: bool, scale: float = 0.0,
               stream=None):
    sh = shape_of(q, k, causal, scale)
    dt, qs, ks = _io(sh)
    args = [_expect(q, "q", qs, dt), _expect(k, "k", ks, dt), _expect(v, "v", ks, dt), _expect(o, "o", qs, dt),
            _expect(do, "do", qs, dt), _vec_ptr(lse, "lse", sh), _vec_ptr(delta, "delta", sh),
            _expect(dq, "dq", qs, dt), _expect(dk, "dk", ks, dt), _expect(dv, "dv", ks, dt)]
    args += _ws_args(workspace)
    return "mxfa_run_bwd_ws", (ctypes.byref(sh.c()), *args, _stream(stream))


def run_bwd_ws(q, k, v, o, do, lse, delta, dq, dk, dv, workspace, causal: bool, scale: float = 0.0,
               stream=None):
    """run_bwd with a workspace (a device tensor of at least
    bwd_workspace_bytes(q, k, causal) bytes, or None) for the split dK/dV pass
    of GQA shapes (mxfa_run_bwd_ws)."""
    _invoke(*_call_bwd_ws(q, k, v, o, do, lse, delta, dq, dk, dv, workspace, causal, scale, stream))


def _call_bwd_noalloc(q, k, v, o, do, lse, delta, dq, dk, dv, causal: bool, scale: float = 0.0, stream=None):
    sh = shape_of(q, k, causal, scale)
    dt, qs, ks = _io(sh)
    args = [_expect(q, "q", qs, dt), _expect(k, "k", ks, dt), _expect(v, "v", ks, dt), _expect(o, "o", qs, dt),
            _expect(do, "do", qs, dt), _vec_ptr(lse, "lse", sh), _vec_ptr(delta, "delta", sh),
            _expect(dq, "dq", qs, dt), _expect(dk, "dk", ks, dt), _expect(dv, "dv", ks, dt)]
    return "mxfa_run_bwd_noalloc", (ctypes.byref(sh.c()), *args, _stream(stream))


def run_bwd_noalloc(q, k, v, o, do, lse, delta, dq, dk, dv, causal: bool, scale: float = 0.0, stream=None):
    """run_bwd_ws with the library's static scratch in place of a workspace
    (mxfa_run_bwd_noalloc): allocates nothing; calls overlapping on one device
    race on the scratch."""
    _invoke(*_call_bwd_noalloc(q, k, v, o, do, lse, delta, dq, dk, dv, causal, scale, stream))


def _call_bwd_dq_delta(q, k, v, o, do, lse, delta, dq, causal: bool, scale: float = 0.0, stream=None):
    sh = shape_of(q, k, causal, scale)
    dt, qs, ks = _io(sh)
    args = [_expect(q, "q", qs, dt), _expect(k, "k", ks, dt), _expect(v, "v", ks, dt), _expect(o, "o", qs, dt),
            _expect(do, "do", qs, dt), _vec_ptr(lse, "lse", sh), _vec_ptr(delta, "delta", sh),
            _expect(dq, "dq", qs, dt)]
    return "mxfa_run_bwd_dq_delta", (ctypes.byref(sh.c()), *args, _stream(stream))


def run_bwd_dq_delta(q, k, v, o, do, lse, delta, dq, causal: bool, scale: float = 0.0, stream=None):
    """dQ pass that computes Delta from O itself and writes it to ``delta``."""
    _invoke(*_call_bwd_dq_delta(q, k, v, o, do, lse, delta, dq, causal, scale, stream))


def _call_bwd_dq(q, k, v, do, lse, delta, dq, causal: bool, scale: float = 0.0, stream=None):
    sh, dt, qs, ks, args = _bwd_args(q, k, v, do, lse, delta, causal, scale)
    args += [_expect(dq, "dq", qs, dt)]
    return "mxfa_run_bwd_dq", (ctypes.byref(sh.c()), *args, _stream(stream))


def run_bwd_dq(q, k, v, do, lse, delta, dq, causal: bool, scale: float = 0.0, stream=None):
    """dQ pass alone (attention_bwd.cu:96-158)."""
    _invoke(*_call_bwd_dq(q, k, v, do, lse, delta, dq, causal, scale, stream))


def _call_bwd_dkv(q, k, v, do, lse, delta, dk, dv, causal: bool, scale: float = 0.0, stream=None):
    sh, dt, qs, ks, args = _bwd_args(q, k, v, do, lse, delta, causal, scale)
    args += [_expect(dk, "dk", ks, dt), _expect(dv, "dv", ks, dt)]
    return "mxfa_run_bwd_dkv", (ctypes.byref(sh.c()), *args, _stream(stream))


def run_bwd_dkv(q, k, v, do, lse, delta, dk, dv, causal: bool, scale: float = 0.0, stream=None):
    """dK/dV pass alone (attention_bwd.cu:165-243)."""
    _invoke(*_call_bwd_dkv(q, k, v, do, lse, delta, dk, dv, causal, scale, stream))


def _call_bwd_dkv_ws(q, k, v, do, lse, delta, dk, dv, workspace, causal: bool, scale: float = 0.0,
                   stream=None):
    sh, dt, qs, ks, args = _bwd_args(q, k, v, do, lse, delta, causal, scale)
    args += [_expect(dk, "dk", ks, dt), _expect(dv, "dv", ks, dt)] + _ws_args(workspace)
    return "mxfa_run_bwd_dkv_ws", (ctypes.byref(sh.c()), *args, _stream(stream))


def run_bwd_dkv_ws(q, k, v, do, lse, delta, dk, dv, workspace, causal: bool, scale: float = 0.0,
                   stream=None):
    """dK/dV pass with a workspace for the split GQA form (mxfa_run_bwd_dkv_ws)."""
    _invoke(*_call_bwd_dkv_ws(q, k, v, do, lse, delta, dk, dv, workspace, causal, scale, stream))


def _call_bwd_naive(q, k, v, do, lse, delta, dq, dk, dv, causal: bool, scale: float = 0.0,
                  stream=None):
    sh, dt, qs, ks, args = _bwd_args(q, k, v, do, lse, delta, causal, scale)
    args += [_expect(dq, "dq", qs, dt), _expect(dk, "dk", ks, dt), _expect(dv, "dv", ks, dt)]
    return "mxfa_run_bwd_naive", (ctypes.byref(sh.c()), *args, _stream(stream))


def run_bwd_naive(q, k, v, do, lse, delta, dq, dk, dv, causal: bool, scale: float = 0.0,
                  stream=None):
    """Naive atomic backward baseline, fp32; outputs must be zeroed (main.rs:147-173)."""
    _invoke(*_call_bwd_naive(q, k, v, do, lse, delta, dq, dk, dv, causal, scale, stream))


class Prepared:
    """One entry point with its arguments checked and marshalled once
    (prepare()): calling it enqueues the same launch again (the same tensors,
    shape, scale and stream) for the cost of one foreign call. It keeps the
    tensors referenced; they must keep their storage (no resize or
    reallocation) while it is in use, as their device addresses are fixed
    in it. The library validates the call again each time, as for any call."""
    __slots__ = ("func", "_fn", "_args", "_keep")

    def __init__(self, func: str, args, keep):
        self.func = func
        self._fn = getattr(load_library(), func)
        self._args = tuple(args)
        self._keep = keep

    def __call__(self):
        rc = self._fn(*self._args)
        if rc != 0:
            _check(self.func, rc)


def prepare(fn, *args, **kwargs) -> Prepared:
    """fn(*args, **kwargs) as a Prepared call, for one of run_flash,
    run_flash_lse, run_preprocess, run_bwd, run_bwd_ws, run_bwd_noalloc,
    run_bwd_flash, run_bwd_dq, run_bwd_dq_delta, run_bwd_dkv, run_bwd_dkv_ws
    and run_bwd_naive: the argument checks of fn run here, once (and raise
    here), so a loop of calls pays only the launch."""
    marshal = _MARSHAL.get(fn)
    if marshal is None:
        raise ValueError(f"prepare: {getattr(fn, '__name__', fn)!r} is not a preparable entry point")
    func, cargs = marshal(*args, **kwargs)
    return Prepared(func, cargs, (args, kwargs))


_MARSHAL = {run_flash: _call_flash, run_flash_lse: _call_flash_lse, run_preprocess: _call_preprocess,
            run_bwd: _call_bwd, run_bwd_ws: _call_bwd_ws, run_bwd_noalloc: _call_bwd_noalloc,
            run_bwd_flash: _call_bwd_flash, run_bwd_dq: _call_bwd_dq, run_bwd_dq_delta: _call_bwd_dq_delta,
            run_bwd_dkv: _call_bwd_dkv, run_bwd_dkv_ws: _call_bwd_dkv_ws, run_bwd_naive: _call_bwd_naive}


def naive_scratch_bytes(q, k, causal: bool) -> int:
    sh = shape_of(q, k, causal)
    return int(load_library().mxfa_naive_scratch_bytes(ctypes.byref(sh.c())))


def naive_run(q, k, v, s, o, causal: bool, scale: float = 0.0, stream=None):
    """Naive forward with the materialised N x N scores ``s`` (Naive::run, main.rs:32-66)."""
    torch = _torch()
    sh = shape_of(q, k, causal, scale)
    dt, qs, ks = _io(sh)
    if s.numel() * 4 < naive_scratch_bytes(q, k, causal):
        raise ValueError("s: scratch too small (needs B*Hq*N*N float32)")
    args = (_expect(q, "q", qs, dt), _expect(k, "k", ks, dt), _expect(v, "v", ks, dt),
            _ptr(s, "s", torch.float32), _expect(o, "o", qs, dt))
    _check("mxfa_run_naive_fwd",
           load_library().mxfa_run_naive_fwd(ctypes.byref(sh.c()), *args, _stream(stream)))


# ------------------------------------------------------------------ prefill --

def _rows(t, name, dtype, min_rows, min_cols):
    """A 2-D device tensor whose rows are contiguous (any row stride): returns
    (pointer, row stride in elements)."""
    torch = _torch()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name}: must be a device tensor (got {t.device}); there is no CPU path")
    if t.dtype != dtype:
        raise ValueError(f"{name}: dtype {t.dtype}, expected {dtype}")
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{name}: expected a 2-D tensor with contiguous rows, got shape {tuple(t.shape)} "
                         f"strides {t.stride()}")
    if t.shape[0] < min_rows or t.shape[1] < min_cols:
        raise ValueError(f"{name}: needs at least {min_rows} rows x {min_cols} columns, got {tuple(t.shape)}")
    return ctypes.c_void_p(t.data_ptr()), (t.stride(0) if t.shape[0] > 1 else max(t.shape[1], min_cols))


def run_prefill(q, kcache, vcache, out, pos0: int, n_head: int, n_kv_head: int, head_dim: int = 64,
                scale: float = 0.0, stream=None):
    """mxfa_run_prefill, the flash forward over a KV cache with token-major rows
    (attn_prefill, 03-llm-engine/kernels/llm.cu:3806-3815): query row i sits at
    position pos0 + i and attends to cache rows 0..pos0 + i.

    q: [n_tok, >= n_head*head_dim] (head h at columns h*head_dim..; may be a
    view into a fused QKV buffer); kcache, vcache: [>= pos0 + n_tok,
    >= n_kv_head*head_dim], same row stride, rows 0..pos0 + n_tok - 1 filled;
    out: [n_tok, >= n_head*head_dim]. All bf16, or fp32 with head_dim 64."""
    torch = _torch()
    if stream is None:
        rc = _calls().prefill(q, kcache, vcache, out, None, 0, pos0, n_head, n_kv_head, head_dim, scale, False, None)
        if rc is not NotImplemented:
            return _check("mxfa_run_prefill", rc)
    if q.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"q: dtype {q.dtype}; bf16 or float32 expected")
    n_tok = q.shape[0] if q.dim() == 2 else -1
    qp, qs = _rows(q, "q", q.dtype, 1, n_head * head_dim)
    kp, ks = _rows(kcache, "kcache", q.dtype, pos0 + n_tok, n_kv_head * head_dim)
    vp, vs = _rows(vcache, "vcache", q.dtype, pos0 + n_tok, n_kv_head * head_dim)
    if ks != vs:
        raise ValueError(f"kcache and vcache must share a row stride ({ks} != {vs})")
    op, os_ = _rows(out, "out", q.dtype, n_tok, n_head * head_dim)
    sh = MxfaPrefillShape(n_tok, n_head, n_kv_head, head_dim, pos0, qs, ks, os_,
                          MXFA_BF16 if q.dtype == torch.bfloat16 else MXFA_F32, scale)
    _check("mxfa_run_prefill", load_library().mxfa_run_prefill(ctypes.byref(sh), qp, kp, vp, op, _stream(stream)))


def run_prefill_paged(q, kcache, vcache, out, block_table, block_size: int, pos0: int, n_head: int,
                      n_kv_head: int, head_dim: int = 64, scale: float = 0.0, stream=None, split: bool = False,
                      workspace=None):
    """mxfa_run_prefill_paged, run_prefill over a paged KV cache
    (attn_prefill_paged, 03-llm-engine/kernels/llm.cu:3827-3836): logical
    position t sits in cache row block_table[t // block_size] * block_size +
    t % block_size (kv_row<true>, llm.cu:959-963).

    kcache, vcache: [pool rows, >= n_kv_head*head_dim], same row stride, the
    pool holding every block the table names; block_table: int32 device tensor
    with at least ceil((pos0 + n_tok) / block_size) entries; block_size: a power
    of two. The rest as run_prefill; the outputs equal run_prefill's over the
    gathered cache bit for bit.

    split=True: mxfa_run_prefill_paged_ws, the keys split as run_prefill_split
    does (workspace as there, allocated here when None and returned); its
    outputs equal run_prefill_split's over the gathered cache bit for bit."""
    torch = _torch()
    if stream is None and (workspace is not None or not split):
        rc = _calls().prefill(q, kcache, vcache, out, block_table, block_size, pos0, n_head, n_kv_head, head_dim,
                                scale, split, workspace)
        if rc is not NotImplemented:
            _check("mxfa_run_prefill_paged_ws" if split else "mxfa_run_prefill_paged", rc)
            return workspace if split else None
    if q.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"q: dtype {q.dtype}; bf16 or float32 expected")
    n_tok = q.shape[0] if q.dim() == 2 else -1
    qp, qs = _rows(q, "q", q.dtype, 1, n_head * head_dim)
    kp, ks = _rows(kcache, "kcache", q.dtype, 1, n_kv_head * head_dim)
    vp, vs = _rows(vcache, "vcache", q.dtype, 1, n_kv_head * head_dim)
    if ks != vs:
        raise ValueError(f"kcache and vcache must share a row stride ({ks} != {vs})")
    op, os_ = _rows(out, "out", q.dtype, n_tok, n_head * head_dim)
    if not isinstance(block_table, torch.Tensor) or block_table.device.type != "cuda" or \
            block_table.dtype != torch.int32 or block_table.dim() != 1 or block_table.stride(0) != 1:
        raise ValueError("block_table: expected a contiguous 1-D int32 device tensor")
    if block_size < 1:
        raise ValueError(f"block_size {block_size}: must be positive")
    need = -(-(pos0 + n_tok) // block_size)
    if block_table.numel() < need:
        raise ValueError(f"block_table: {block_table.numel()} entries, positions 0..{pos0 + n_tok - 1} need {need}")
    sh = MxfaPrefillShape(n_tok, n_head, n_kv_head, head_dim, pos0, qs, ks, os_,
                          MXFA_BF16 if q.dtype == torch.bfloat16 else MXFA_F32, scale)
    lib = load_library()
    if not split:
        _check("mxfa_run_prefill_paged",
               lib.mxfa_run_prefill_paged(ctypes.byref(sh), qp, kp, vp, op, ctypes.c_void_p(block_table.data_ptr()),
                                          int(block_size), _stream(stream)))
        return None
    workspace = _split_workspace(lib, sh, workspace, q.device, stream)
    _check("mxfa_run_prefill_paged_ws",
           lib.mxfa_run_prefill_paged_ws(ctypes.byref(sh), qp, kp, vp, op, ctypes.c_void_p(block_table.data_ptr()),
                                         int(block_size), ctypes.c_void_p(workspace.data_ptr()),
                                         workspace.numel() * workspace.element_size(), _stream(stream)))
    return workspace


def _split_workspace(lib, sh, workspace, device, stream):
    """The split prefill's workspace: `workspace` checked, or a new one of the size the shape needs."""
    torch = _torch()
    if workspace is None:
        need = int(lib.mxfa_prefill_workspace_bytes(ctypes.byref(sh)))
        workspace = _scratch(max(need, 16), device, stream)
    if not isinstance(workspace, torch.Tensor) or workspace.device.type != "cuda" or not workspace.is_contiguous():
        raise ValueError("workspace: expected a contiguous device tensor")
    return workspace


def prefill_workspace_bytes(n_tok: int, pos0: int, n_head: int, n_kv_head: int, head_dim: int = 64,
                            bf16: bool = True) -> int:
    """mxfa_prefill_workspace_bytes for contiguous rows: the fp32 partials
    run_prefill_split needs (0: the shape runs unsplit)."""
    w = n_head * head_dim
    sh = MxfaPrefillShape(n_tok, n_head, n_kv_head, head_dim, pos0, w, n_kv_head * head_dim, w,
                          MXFA_BF16 if bf16 else MXFA_F32, 0.0)
    return int(load_library().mxfa_prefill_workspace_bytes(ctypes.byref(sh)))


def run_prefill_split(q, kcache, vcache, out, pos0: int, n_head: int, n_kv_head: int, head_dim: int = 64,
                      scale: float = 0.0, workspace=None, stream=None):
    """mxfa_run_prefill_ws: run_prefill with the cache's keys split over
    work-groups when the chunk's query blocks would not fill the GPU (the same
    attn_prefill launch, 03-llm-engine/kernels/llm.cu:3806-3815). Arguments as
    run_prefill; workspace: a device tensor of at least the size
    mxfa_prefill_workspace_bytes reports (allocated here when None). Results
    equal run_prefill's to fp32 rounding, not bitwise."""
    torch = _torch()
    if stream is None and workspace is not None:
        rc = _calls().prefill(q, kcache, vcache, out, None, 0, pos0, n_head, n_kv_head, head_dim, scale, True,
                                workspace)
        if rc is not NotImplemented:
            _check("mxfa_run_prefill_ws", rc)
            return workspace
    if q.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"q: dtype {q.dtype}; bf16 or float32 expected")
    n_tok = q.shape[0] if q.dim() == 2 else -1
    qp, qs = _rows(q, "q", q.dtype, 1, n_head * head_dim)
    kp, ks = _rows(kcache, "kcache", q.dtype, pos0 + n_tok, n_kv_head * head_dim)
    vp, vs = _rows(vcache, "vcache", q.dtype, pos0 + n_tok, n_kv_head * head_dim)
    if ks != vs:
        raise ValueError(f"kcache and vcache must share a row stride ({ks} != {vs})")
    op, os_ = _rows(out, "out", q.dtype, n_tok, n_head * head_dim)
    sh = MxfaPrefillShape(n_tok, n_head, n_kv_head, head_dim, pos0, qs, ks, os_,
                          MXFA_BF16 if q.dtype == torch.bfloat16 else MXFA_F32, scale)
    lib = load_library()
    workspace = _split_workspace(lib, sh, workspace, q.device, stream)
    have = workspace.numel() * workspace.element_size()
    _check("mxfa_run_prefill_ws",
           lib.mxfa_run_prefill_ws(ctypes.byref(sh), qp, kp, vp, op, ctypes.c_void_p(workspace.data_ptr()),
                                   have, _stream(stream)))
    return workspace


# ------------------------------------------------------------ rotary positions --

def rotary_frequencies(dim: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                       original_length: int = 4096, fast_turns: float = 32.0, slow_turns: float = 1.0, device="cuda"):
    """The angles per position (radians, float64, dim / 2 of them) that run_rotary
    and run_cache_append take, and the factor of the rotation, as (frequencies,
    factor): base^(-2i / dim), and for contexts `factor` times as long as
    the model's own

    * scaling="linear": positions compressed, every frequency divided by factor;
    * "base": base times factor^(dim / (dim - 2)), which leaves the fastest pair
      as it is and divides the slowest by factor;
    * "yarn": divided by factor where a pair turns at most slow_turns times over
      original_length positions, left where it turns fast_turns times or more,
      in between in proportion to the pair's index; the rotation's factor is
      0.1 ln(factor) + 1.

    Computed on the host, once per model."""
    import math
    torch = _torch()
    if dim < 2 or dim % 2:
        raise ValueError(f"dim {dim}: must be even and positive")
    if not base > 1.0 or not factor >= 1.0:
        raise ValueError("base must be above 1 and factor at least 1")
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    if scaling == "base":
        if dim == 2:
            raise ValueError('scaling="base" needs more than one pair')
        base = base * factor ** (dim / (dim - 2))
    f = base ** (-i / dim)
    amount = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        def pair(turns):  # the pair that turns so often over original_length
            return dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(pair(fast_turns)), 0), min(math.ceil(pair(slow_turns)), dim - 1)
        ramp = ((torch.arange(dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        amount = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "base"):
        raise ValueError(f"scaling {scaling!r}: None, 'linear', 'base' or 'yarn' expected")
    return f.to(device), amount


def _on(device):
    """Runs launches on `device` (its current stream) where it is not the
    calling thread's."""
    torch = _torch()
    import contextlib
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _dev(t, name, dtype=None, like=None):
    """A device tensor of the dtype, on `like`'s device."""
    torch = _torch()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name}: must be a device tensor (got {t.device}); there is no CPU path")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name}: dtype {t.dtype}, expected {dtype}")
    if like is not None and t.device != like.device:
        raise ValueError(f"{name}: on {t.device}, the other tensors on {like.device}")
    return t


def _c_int(**values):
    """The values, which must be whole numbers that a C int holds (ctypes would cut
    them)."""
    import operator
    for name, v in values.items():
        if not -2 ** 31 <= operator.index(v) < 2 ** 31:
            raise ValueError(f"{name} {v}: past 32 bits")


def _ints(t, name, n, like):
    """A contiguous int32 vector of at least n elements."""
    torch = _torch()
    _dev(t, name, torch.int32, like)
    if t.dim() != 1 or (t.numel() > 1 and t.stride(0) != 1) or t.numel() < n:
        raise ValueError(f"{name}: expected a contiguous int32 vector of at least {n} elements, got shape "
                         f"{tuple(t.shape)} strides {t.stride()}")
    return ctypes.c_void_p(t.data_ptr())


def _freqs(frequencies, dim_max, like):
    """(pointer, rotary_dim) of a frequencies vector."""
    torch = _torch()
    _dev(frequencies, "frequencies", torch.float64, like)
    if frequencies.dim() != 1 or not frequencies.is_contiguous() or not 1 <= frequencies.numel() <= dim_max // 2:
        raise ValueError(f"frequencies: expected a contiguous vector of 1 to {dim_max // 2} elements (half of what is "
                         f"rotated), got shape {tuple(frequencies.shape)}")
    return ctypes.c_void_p(frequencies.data_ptr()), 2 * frequencies.numel()


def _heads(t, name):
    """[B, H, N, d], or [N, H, d] (tokens first) as B = 1: (pointer, sizes, strides)."""
    if t.dim() == 3:
        n, h, d = t.shape
        sizes, strides = (1, h, n, d), (0, t.stride(1), t.stride(0))
    elif t.dim() == 4:
        sizes, strides = tuple(t.shape), t.stride()[:3]
    else:
        raise ValueError(f"{name}: expected [B, H, N, d] or [N, H, d], got {tuple(t.shape)}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: rows must be contiguous (strides {t.stride()})")
    return ctypes.c_void_p(t.data_ptr()), sizes, strides


def run_rotary(q, k, q_out, k_out, frequencies, positions=None, pos0: int = 0, interleaved: bool = False,
               factor: float = 1.0, inverse: bool = False, stream=None):
    """mxfa_run_rotary: rotary positions of Q and K (k and k_out None: Q alone)
    in one launch. Pair i of a head's first 2 len(frequencies) elements, (x[i],
    x[i + len(frequencies)]) or with interleaved (x[2i], x[2i + 1]), turns by
    position * frequencies[i] and is multiplied by factor; the rest is copied.

    q, k and their outputs: [B, H, N, d], or [N, H, d] with the tokens first;
    rows contiguous, any other strides (views of a fused QKV buffer; an output
    may be its input), starting on 16 bytes. bf16 or fp32, d a multiple of 8 up
    to 256. frequencies: float64 on the device (rotary_frequencies).
    positions: int32, [N] or [B, N]; None: token n at pos0 + n. inverse: the
    transpose (gradients of the outputs to gradients of the inputs)."""
    torch = _torch()
    if stream is None:
        rc = _calls().rotary(q, k, q_out, k_out, frequencies, positions, pos0, interleaved, factor, inverse)
        if rc is not NotImplemented:
            return _check("mxfa_run_rotary", rc)
    _dev(q, "q")
    if q.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"q: dtype {q.dtype}; bf16 or float32 expected")
    qp, (B, Hq, N, d), qs = _heads(q, "q")
    qop, osz, qos = _heads(_dev(q_out, "q_out", q.dtype, q), "q_out")
    if osz != (B, Hq, N, d):
        raise ValueError(f"q_out: shape {tuple(q_out.shape)} does not match q's {tuple(q.shape)}")
    if (k is None) != (k_out is None):
        raise ValueError("k and k_out: both or neither")
    kp = kop = None
    Hkv, ks, kos = 0, (0, 0, 0), (0, 0, 0)
    if k is not None:
        kp, (Bk, Hkv, Nk, dk), ks = _heads(_dev(k, "k", q.dtype, q), "k")
        if (Bk, Nk, dk) != (B, N, d):
            raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} disagree")
        kop, osz, kos = _heads(_dev(k_out, "k_out", q.dtype, q), "k_out")
        if osz != (B, Hkv, N, d):
            raise ValueError(f"k_out: shape {tuple(k_out.shape)} does not match k's {tuple(k.shape)}")
    fp, dim = _freqs(frequencies, d, q)
    pp, pbs = None, 0
    if positions is not None:
        _dev(positions, "positions", torch.int32, q)
        if tuple(positions.shape) not in ((N,), (B, N)) or (N > 1 and positions.stride(-1) != 1):
            raise ValueError(f"positions: expected [{N}] or [{B}, {N}] with contiguous rows, got "
                             f"{tuple(positions.shape)} strides {positions.stride()}")
        pp, pbs = ctypes.c_void_p(positions.data_ptr()), positions.stride(0) if positions.dim() == 2 else 0
    _c_int(pos0=pos0, B=B, Hq=Hq, Hkv=Hkv, N=N)
    sh = MxfaRotaryShape(B, Hq, Hkv, N, d, dim, int(bool(interleaved)), int(bool(inverse)),
                         MXFA_BF16 if q.dtype == torch.bfloat16 else MXFA_F32, pos0, factor, *qs, *ks, *qos, *kos, pbs)
    with _on(q.device):
        _check("mxfa_run_rotary", load_library().mxfa_run_rotary(ctypes.byref(sh), qp, kp, qop, kop, pp, fp,
                                                                 _stream(stream)))


# ------------------------------------------------- a batch over a paged cache --

def _block_table(block_table, n_seq, like):
    """A 2-D int32 table of contiguous rows: (pointer, entries of a row, row stride)."""
    torch = _torch()
    _dev(block_table, "block_table", torch.int32, like)
    if block_table.dim() != 2 or block_table.shape[1] < 1 or \
            (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError(f"block_table: expected a 2-D int32 tensor with contiguous rows, got shape "
                         f"{tuple(block_table.shape)} strides {block_table.stride()}")
    if block_table.shape[0] != n_seq:
        raise ValueError(f"block_table: {block_table.shape[0]} rows for {n_seq} sequences")
    wide = block_table.shape[1]
    return ctypes.c_void_p(block_table.data_ptr()), wide, block_table.stride(0) if n_seq > 1 else wide


def _batch_args(q, q_cols, kcache, vcache, out, block_table, block_size, cu_q, lens, max_q, n_head, n_kv_head,
                head_dim, scale, bits=None):
    """bits: None for a cache of rows in q's type, else blocks of bytes of so many bits a value."""
    torch = _torch()
    _dev(q, "q")
    if q.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"q: dtype {q.dtype}; bf16 or float32 expected")
    _c_int(max_q=max_q, n_head=n_head, n_kv_head=n_kv_head, head_dim=head_dim, block_size=block_size)
    if n_head < 1 or n_kv_head < 1 or head_dim < 1 or block_size < 1:
        raise ValueError("n_head, n_kv_head, head_dim and block_size must be positive")
    n_tok = q.shape[0] if q.dim() == 2 else -1
    qp, qs = _rows(q, "q", q.dtype, 1, q_cols * head_dim)
    kt, least, wide = q.dtype, block_size, n_kv_head * head_dim
    if bits is not None:
        kt, least, wide = torch.uint8, 1, mx_block_bytes(block_size, n_kv_head, head_dim, bits)
    kp, ks = _rows(_dev(kcache, "kcache", kt, q), "kcache", kt, least, wide)
    vp, vs = _rows(_dev(vcache, "vcache", kt, q), "vcache", kt, least, wide)
    if ks != vs or kcache.shape[0] != vcache.shape[0]:
        raise ValueError(f"kcache and vcache must share their rows and row stride ({kcache.shape[0]}, {ks} and "
                         f"{vcache.shape[0]}, {vs})")
    op, os_ = _rows(_dev(out, "out", q.dtype, q), "out", q.dtype, n_tok, n_head * head_dim)
    n_seq = lens.numel() if isinstance(lens, torch.Tensor) else 0
    lp = _ints(lens, "lens", 1, q)
    cp = _ints(cu_q, "cu_q", n_seq + 1, q)
    tp, wide, ts = _block_table(block_table, n_seq, q)
    n_blocks = kcache.shape[0] // least
    _c_int(n_tok=n_tok, n_blocks=n_blocks, table_stride=ts, q_stride=qs, kv_stride=ks,
           out_stride=os_)
    sh = MxfaBatchShape(n_tok, n_seq, max_q, n_head, n_kv_head, head_dim, block_size, n_blocks, wide, ts, qs, ks, os_,
                        MXFA_BF16 if q.dtype == torch.bfloat16 else MXFA_F32, scale)
    return sh, qp, kp, vp, op, tp, cp, lp


def run_cache_append(qkv, q_out, kcache, vcache, block_table, block_size: int, cu_q, lens, n_head: int, n_kv_head: int,
                     head_dim: int = 64, frequencies=None, interleaved: bool = False, factor: float = 1.0,
                     stream=None):
    """mxfa_run_cache_append: the new tokens of a batch of sequences enter the paged
    cache, with rotary positions, in one launch: of each row of qkv the query
    heads turn into q_out (which may be qkv), the key heads turn into kcache and
    the value heads are copied into vcache, at the row of the token's position.
    This is what run_prefill_batch (or run_prefill_paged) then reads.

    qkv: [n_tok, >= (n_head + 2 n_kv_head) head_dim], q_out: [n_tok, >= n_head
    head_dim], kcache, vcache: [pool rows, >= n_kv_head head_dim] with one row
    stride; block_table: int32 [n_seq, entries]; cu_q: int32 [n_seq + 1], where
    each sequence's rows of qkv begin and the last end; lens: int32 [n_seq],
    the sequences' lengths with their new tokens. frequencies: as for
    run_rotary; None copies without turning. bf16 or fp32."""
    if stream is None:
        rc = _calls().cache_append(qkv, q_out, kcache, vcache, block_table, block_size, cu_q, lens, n_head, n_kv_head,
                                   head_dim, frequencies, interleaved, factor)
        if rc is not NotImplemented:
            return _check("mxfa_run_cache_append", rc)
    sh, qp, kp, vp, op, tp, cp, lp = _batch_args(qkv, n_head + 2 * n_kv_head, kcache, vcache, q_out, block_table,
                                                 block_size, cu_q, lens, 1, n_head, n_kv_head, head_dim, 0.0)
    fp, dim = (None, 0) if frequencies is None else _freqs(frequencies, head_dim, qkv)
    rot = MxfaAppendRotary(dim, int(bool(interleaved)), factor, fp)
    with _on(qkv.device):
        _check("mxfa_run_cache_append",
               load_library().mxfa_run_cache_append(ctypes.byref(sh), ctypes.byref(rot), qp, op, kp, vp, tp, cp, lp,
                                                    _stream(stream)))


def _widest(n_seq):
    """A table width in positions at which a batch's workspace is the largest: 2^17, where
    every form has all its work-groups, or the widest that is taken of so many sequences."""
    return max(min(1 << 17, 64 * ((1 << 31) // max(n_seq, 1) - 2)), 1)


def prefill_batch_workspace_bytes(n_tok: int, n_seq: int, max_q: int, n_head: int, n_kv_head: int, head_dim: int = 64,
                                  bf16: bool = True) -> int:
    """mxfa_prefill_batch_workspace_bytes: what run_prefill_batch needs for such a
    batch, whatever its lengths (0 for one it does not take)."""
    w, entries = n_head * head_dim, _widest(n_seq)
    _c_int(n_tok=n_tok, n_seq=n_seq, max_q=max_q, n_head=n_head, n_kv_head=n_kv_head, head_dim=head_dim, q_stride=w)
    sh = MxfaBatchShape(n_tok, n_seq, max_q, n_head, n_kv_head, head_dim, 1, 1, entries, entries, w,
                        n_kv_head * head_dim, w, MXFA_BF16 if bf16 else MXFA_F32, 0.0)
    return int(load_library().mxfa_prefill_batch_workspace_bytes(ctypes.byref(sh)))


def run_prefill_batch(q, kcache, vcache, out, block_table, block_size: int, cu_q, lens, max_q: int, n_head: int,
                      n_kv_head: int, head_dim: int = 64, scale: float = 0.0, lse=None, workspace=None, stream=None):
    """mxfa_run_prefill_batch: attention of a batch of sequences' new tokens (one
    token, a chunk, or both side by side) over the paged cache: a token attends
    to its sequence's positions up to its own, which the cache holds
    (run_cache_append). Lengths and tables are read on the device.

    q: [n_tok, >= n_head head_dim] (may be the columns of a fused QKV buffer),
    out likewise (may be q, or other columns of its rows; refused where it lies
    over q or a cache otherwise); the caches, block_table, cu_q and lens as for
    run_cache_append; max_q: at least the most new tokens any sequence has
    (rows past it are not computed). lse: None, or float32 [n_tok, n_head] for
    the rows' log-sum-exp. workspace: a contiguous device tensor of
    prefill_batch_workspace_bytes bytes (allocated when None, as memory of
    `stream`); returned. Calls that may overlap need their own. bf16 with
    head_dim 64 or 128, or fp32 with 64."""
    if stream is None:
        rc = _calls().prefill_batch(q, kcache, vcache, out, block_table, block_size, cu_q, lens, max_q, n_head,
                                    n_kv_head, head_dim, scale, lse, workspace)
        if rc is not NotImplemented:
            if isinstance(rc, int):
                _check("mxfa_run_prefill_batch", rc)
            return rc
    return _run_attention("mxfa_run_prefill_batch", (), q, kcache, vcache, out, block_table, block_size, cu_q, lens, max_q,
                          n_head, n_kv_head, head_dim, scale, lse, workspace, stream)


def _run_attention(func, bits, q, kcache, vcache, out, block_table, block_size, cu_q, lens, max_q, n_head, n_kv_head,
                   head_dim, scale, lse, workspace, stream):
    """The attention over either cache; bits: () or (the bits,)."""
    torch = _torch()
    sh, qp, kp, vp, op, tp, cp, lp = _batch_args(q, n_head, kcache, vcache, out, block_table, block_size, cu_q, lens,
                                                 max_q, n_head, n_kv_head, head_dim, scale, *bits)
    ep = None
    if lse is not None:
        _dev(lse, "lse", torch.float32, q)
        if tuple(lse.shape) != (sh.n_tok, n_head) or not lse.is_contiguous():
            raise ValueError(f"lse: expected a contiguous [{sh.n_tok}, {n_head}], got {tuple(lse.shape)}")
        ep = ctypes.c_void_p(lse.data_ptr())
    lib = load_library()
    check, need, run = (getattr(lib, n) for n in (func.replace("run_prefill", "check"),
                                                  func.replace("run_", "") + "_workspace_bytes", func))
    _check("mxfa_check_batch" + func[len("mxfa_run_prefill_batch"):], check(ctypes.byref(sh), *bits))
    with _on(q.device):
        if workspace is None:
            workspace = _scratch(int(need(ctypes.byref(sh), *bits)), q.device, stream)
        elif not _dev(workspace, "workspace", None, q).is_contiguous():
            raise ValueError("workspace: expected a contiguous device tensor")
        _check(func, run(ctypes.byref(sh), *bits, qp, kp, vp, op, ep, tp, cp, lp, ctypes.c_void_p(workspace.data_ptr()),
                         workspace.numel() * workspace.element_size(), _stream(stream)))
    return workspace


# ------------------------------------------------------- a microscaled cache --

def mx_block_bytes(block_size: int, n_kv_head: int, head_dim: int = 64, bits: int = 8) -> int:
    """mxfa_mx_block_bytes: the bytes of a block of a microscaled cache (a multiple of
    16): of each head's row, 32 neighbouring elements share a power of two 2^(E -
    127), one byte E, and are codes of 8 bits (e4m3) or 4 (e2m1) that stand for 2^(E
    - 127) code. A pool is uint8 [blocks, at least this], its row stride a multiple
    of 16; kcache and vcache are two of them. run_pages_copy(pool, 1, pairs) copies
    its blocks."""
    _c_int(block_size=block_size, n_kv_head=n_kv_head, head_dim=head_dim, bits=bits)
    n = int(load_library().mxfa_mx_block_bytes(block_size, n_kv_head, head_dim, bits))
    if n == 0:
        raise ValueError(f"no microscaled blocks of block_size {block_size} (a power of two), {n_kv_head} KV heads, head_dim "
                         f"{head_dim} (a multiple of 32, at most 256), {bits} bits (8 or 4)")
    return n


def run_cache_append_mx(qkv, q_out, kcache, vcache, bits: int, block_table, block_size: int, cu_q, lens, n_head: int,
                        n_kv_head: int, head_dim: int = 64, frequencies=None, interleaved: bool = False,
                        factor: float = 1.0, stream=None):
    """mxfa_run_cache_append_mx: as run_cache_append, into a microscaled cache of `bits`
    (8 or 4) bits a value: K, turned, and V are quantised as they are written, each
    group of 32 elements by its own power of two, to the nearest code. kcache,
    vcache: uint8 [blocks, at least mx_block_bytes]. A group of which an element is
    not finite reads back as NaN. The other arguments are as for run_cache_append;
    head_dim is a multiple of 32, at most 256."""
    if stream is None:
        rc = _calls().cache_append_mx(qkv, q_out, kcache, vcache, block_table, block_size, cu_q, lens, n_head, n_kv_head,
                                      head_dim, frequencies, interleaved, factor, bits)
        if rc is not NotImplemented:
            return _check("mxfa_run_cache_append_mx", rc)
    sh, qp, kp, vp, op, tp, cp, lp = _batch_args(qkv, n_head + 2 * n_kv_head, kcache, vcache, q_out, block_table,
                                                 block_size, cu_q, lens, 1, n_head, n_kv_head, head_dim, 0.0, bits)
    fp, dim = (None, 0) if frequencies is None else _freqs(frequencies, head_dim, qkv)
    rot = MxfaAppendRotaryMx(dim, int(bool(interleaved)), factor, fp)
    with _on(qkv.device):
        _check("mxfa_run_cache_append_mx",
               load_library().mxfa_run_cache_append_mx(ctypes.byref(sh), bits, ctypes.byref(rot), qp, op, kp, vp, tp, cp,
                                                       lp, _stream(stream)))


def run_cache_read_mx(kcache, vcache, bits: int, k_out, v_out, block_table, block_size: int, cu_q, lens, n_kv_head: int,
                      head_dim: int = 64, stream=None):
    """mxfa_run_cache_read_mx: rows of a microscaled cache as bf16 or fp32 again (its
    values are exact in either): row r of k_out and v_out ([rows, >= n_kv_head
    head_dim], one row stride) is what the cache holds at the position of row r of
    run_cache_append_mx for the same cu_q and lens, that is each sequence's last
    cu_q[s + 1] - cu_q[s] positions: what an append wrote, or with the lengths' own
    sums for cu_q the whole sequences. Rows of no position, and those past
    cu_q[-1], stay as they were."""
    torch = _torch()
    if stream is None:
        rc = _calls().cache_read_mx(kcache, vcache, k_out, v_out, block_table, block_size, cu_q, lens, n_kv_head, head_dim,
                                    bits)
        if rc is not NotImplemented:
            return _check("mxfa_run_cache_read_mx", rc)
    sh, op, kp, vp, _, tp, cp, lp = _batch_args(k_out, n_kv_head, kcache, vcache, k_out, block_table, block_size, cu_q,
                                                lens, 1, n_kv_head, n_kv_head, head_dim, 0.0, bits)
    wp, ws = _rows(_dev(v_out, "v_out", k_out.dtype, k_out), "v_out", k_out.dtype, sh.n_tok, n_kv_head * head_dim)
    if v_out.shape[0] != sh.n_tok or (sh.n_tok > 1 and ws != sh.out_stride):
        raise ValueError(f"k_out and v_out must share their rows and row stride ({sh.n_tok}, {sh.out_stride} and "
                         f"{v_out.shape[0]}, {ws})")
    with _on(k_out.device):
        _check("mxfa_run_cache_read_mx",
               load_library().mxfa_run_cache_read_mx(ctypes.byref(sh), bits, kp, vp, op, wp, tp, cp, lp, _stream(stream)))


def prefill_batch_mx_workspace_bytes(n_tok: int, n_seq: int, max_q: int, n_head: int, n_kv_head: int, head_dim: int = 64,
                                     bf16: bool = True, bits: int = 8) -> int:
    """mxfa_prefill_batch_mx_workspace_bytes: what run_prefill_batch_mx needs for such a
    batch, whatever its lengths (0 for one it does not take)."""
    w, entries, block = n_head * head_dim, _widest(n_seq), mx_block_bytes(1, n_kv_head, head_dim, bits)
    _c_int(n_tok=n_tok, n_seq=n_seq, max_q=max_q, n_head=n_head, n_kv_head=n_kv_head, head_dim=head_dim, q_stride=w)
    sh = MxfaBatchShape(n_tok, n_seq, max_q, n_head, n_kv_head, head_dim, 1, 1, entries, entries, w, block, w,
                        MXFA_BF16 if bf16 else MXFA_F32, 0.0)
    return int(load_library().mxfa_prefill_batch_mx_workspace_bytes(ctypes.byref(sh), bits))


def run_prefill_batch_mx(q, kcache, vcache, bits: int, out, block_table, block_size: int, cu_q, lens, max_q: int,
                         n_head: int, n_kv_head: int, head_dim: int = 64, scale: float = 0.0, lse=None, workspace=None,
                         stream=None):
    """mxfa_run_prefill_batch_mx: as run_prefill_batch, over what a microscaled cache of
    `bits` (8 or 4) bits a value holds (run_cache_append_mx): K and V enter the
    products as the values that their codes stand for, without another rounding. The
    workspace is of prefill_batch_mx_workspace_bytes; the other arguments are as
    for run_prefill_batch."""
    if stream is None:
        rc = _calls().prefill_batch_mx(q, kcache, vcache, out, block_table, block_size, cu_q, lens, max_q, n_head,
                                       n_kv_head, head_dim, scale, lse, workspace, bits)
        if rc is not NotImplemented:
            if isinstance(rc, int):
                _check("mxfa_run_prefill_batch_mx", rc)
            return rc
    return _run_attention("mxfa_run_prefill_batch_mx", (bits,), q, kcache, vcache, out, block_table, block_size, cu_q, lens,
                          max_q, n_head, n_kv_head, head_dim, scale, lse, workspace, stream)


# ------------------------------------------------------- the pages of a cache --

def _pages_args(block_table, block_size, lens, refs):
    torch = _torch()
    _dev(lens, "lens", torch.int32)
    tp, wide, ts = _block_table(block_table, lens.numel(), lens)
    _c_int(block_size=block_size, table_stride=ts)
    sh = MxfaPagesShape(lens.numel(), wide, ts, block_size, refs.numel() if isinstance(refs, torch.Tensor) else 0)
    return sh, tp, _ints(lens, "lens", 1, lens), _ints(refs, "refs", 1, lens)


def run_pages_free(block_table, block_size: int, lens, refs, rows, stream=None):
    """mxfa_run_pages_free: the sequences named in rows (int32) end: the use counts
    (refs, int32 per block of the pool) of the blocks they hold go down by one,
    their block_table entries become -1 and their lens 0. Row numbers out of
    range are skipped, a row named twice ends once."""
    if stream is None:
        rc = _calls().pages_free(block_table, block_size, lens, refs, rows)
        if rc is not NotImplemented:
            return _check("mxfa_run_pages_free", rc)
    sh, tp, lp, rp = _pages_args(block_table, block_size, lens, refs)
    n = _ints(rows, "rows", 0, lens)
    with _on(lens.device):
        _check("mxfa_run_pages_free", load_library().mxfa_run_pages_free(ctypes.byref(sh), tp, lp, rp, n, rows.numel(),
                                                                         _stream(stream)))


def run_pages_fork(block_table, block_size: int, lens, refs, parents, children, pairs, status, counts, stream=None):
    """mxfa_run_pages_fork: row children[i] (an empty one) becomes a continuation of
    row parents[i]: it shares the parent's whole blocks, and a last block that is
    not full is given a copy, in the lowest block that nobody uses. The copies
    are written to pairs (int32 [n, 2]: source, destination) and their number to
    counts[0]; run_pages_copy(pool, block_size, pairs, counts) then makes them,
    in each pool of the cache. status[i] (int32 [n]): 0, or 1 where a pair was
    refused (a row out of range, a child that is not empty or that an earlier
    pair names, no block left); counts[1] (int32 [2]): how many were."""
    torch = _torch()
    if stream is None:
        rc = _calls().pages_fork(block_table, block_size, lens, refs, parents, children, pairs, status, counts)
        if rc is not NotImplemented:
            return _check("mxfa_run_pages_fork", rc)
    sh, tp, lp, rp = _pages_args(block_table, block_size, lens, refs)
    n = parents.numel() if isinstance(parents, torch.Tensor) else 0
    pa, ch = _ints(parents, "parents", 0, lens), _ints(children, "children", n, lens)
    if children.numel() != n:
        raise ValueError(f"{n} parents and {children.numel()} children")
    st, ct = _ints(status, "status", n, lens), _ints(counts, "counts", 2, lens)
    pp = _pairs_ptr(pairs, n, lens)
    with _on(lens.device):
        _check("mxfa_run_pages_fork",
               load_library().mxfa_run_pages_fork(ctypes.byref(sh), tp, lp, rp, pa, ch, n, pp, st, ct, _stream(stream)))


def _pairs_ptr(pairs, n, like):
    torch = _torch()
    _dev(pairs, "pairs", torch.int32, like)
    if pairs.dim() != 2 or pairs.shape[1] != 2 or pairs.shape[0] < n or not pairs.is_contiguous():
        raise ValueError(f"pairs: expected a contiguous int32 [at least {n}, 2], got {tuple(pairs.shape)}")
    return ctypes.c_void_p(pairs.data_ptr())


def run_pages_compact(block_table, block_size: int, lens, refs, new_table, new_refs, pairs, counts, stream=None):
    """mxfa_run_pages_compact: the blocks in use move to the pool's low end, in
    their order, as few of them as that takes. Writes the block tables
    (new_table, which may be block_table) and use counts (new_refs, which may not
    be refs) as they are after the moves, the moves to pairs (int32 [at least
    max(1, n_blocks // 2), 2]) and to counts (int32 [2]) their number and that
    of the blocks in use. run_pages_copy(pool, block_size, pairs, counts) then
    makes the moves, in each pool of the cache; the old tables stay valid until
    the blocks that were left are used again."""
    if stream is None:
        rc = _calls().pages_compact(block_table, block_size, lens, refs, new_table, new_refs, pairs, counts)
        if rc is not NotImplemented:
            return _check("mxfa_run_pages_compact", rc)
    sh, tp, lp, rp = _pages_args(block_table, block_size, lens, refs)
    ntp, wide, nts = _block_table(new_table, lens.numel(), lens)
    if wide != sh.max_blocks:
        raise ValueError(f"new_table: {wide} entries to a row, block_table {sh.max_blocks}")
    nr = _ints(new_refs, "new_refs", sh.n_blocks, lens)
    pp, ct = _pairs_ptr(pairs, max(1, sh.n_blocks // 2), lens), _ints(counts, "counts", 2, lens)
    with _on(lens.device):
        _check("mxfa_run_pages_compact",
               load_library().mxfa_run_pages_compact(ctypes.byref(sh), tp, lp, rp, ntp, nts, nr, pp, ct, _stream(stream)))


def run_pages_copy(pools, block_size: int, pairs, count=None, stream=None):
    """mxfa_run_pages_copy: block pairs[j, 0] is copied to block pairs[j, 1], in one
    pool [rows, width] or in several [pools, rows, width] (K and V of every
    layer, say) of contiguous rows, block j being rows j block_size .. (j + 1)
    block_size - 1. count: an int32 device tensor whose first element says how
    many of the pairs count (run_pages_fork's and run_pages_compact's counts);
    None: all. Pairs with a number outside the pool are skipped; no destination
    may be another pair's source or destination. Any dtype; a block is a
    multiple of 16 bytes."""
    if stream is None:
        rc = _calls().pages_copy(pools, block_size, pairs, count)
        if rc is not NotImplemented:
            return _check("mxfa_run_pages_copy", rc)
    _dev(pools, "pools")
    if block_size < 1:
        raise ValueError(f"block_size {block_size}: must be positive")
    if pools.dim() not in (2, 3) or pools.numel() == 0 or not pools[(0,) * (pools.dim() - 2)].is_contiguous() or \
            pools.shape[-2] < block_size:
        raise ValueError(f"pools: expected [rows, width] or [pools, rows, width] of contiguous rows and at least a "
                         f"block of them, got shape {tuple(pools.shape)} strides {pools.stride()}")
    es, many = pools.element_size(), pools.dim() == 3
    pp = _pairs_ptr(pairs, 0, pools)
    cp = None if count is None else _ints(count, "count", 1, pools)
    with _on(pools.device):
        _check("mxfa_run_pages_copy",
               load_library().mxfa_run_pages_copy(ctypes.c_void_p(pools.data_ptr()), pools.shape[0] if many else 1,
                                                  pools.stride(0) * es if many else 0, pools.shape[-2] // block_size,
                                                  block_size * pools.shape[-1] * es, pp, pairs.shape[0], cp,
                                                  _stream(stream)))


# ------------------------------------------------------------ conveniences --

def attention_fwd(q, k, v, causal: bool, scale: float = 0.0, stream=None):
    """Allocates O and LSE and runs the forward; returns (O, LSE)."""
    torch = _torch()
    if stream is None:
        r = _calls().attention_fwd(q, k, v, causal, scale)
        if isinstance(r, tuple):
            return r
        if r is not NotImplemented:
            _check("mxfa_run_flash_lse", r)
    sh = shape_of(q, k, causal, scale)
    o = torch.empty_like(q)
    lse = torch.empty((sh.B, sh.Hq, sh.N), dtype=torch.float32, device=q.device)
    run_flash_lse(q, k, v, o, lse, causal, scale, stream)
    return o, lse


def attention_bwd(q, k, v, o, lse, do, causal: bool, scale: float = 0.0, stream=None):
    """Allocates Delta, dQ, dK, dV (and, for GQA shapes that use one, the dK/dV
    workspace) and runs the backward (run_bwd_ws: Delta folded into the dQ
    pass); returns (dQ, dK, dV)."""
    torch = _torch()
    if stream is None:
        r = _calls().attention_bwd(q, k, v, o, lse, do, causal, scale)
        if isinstance(r, tuple):
            return r
        if r is not NotImplemented:
            _check("mxfa_run_bwd_ws", r)
    sh = shape_of(q, k, causal, scale)
    delta = _scratch(4 * sh.B * sh.Hq * sh.N, q.device, stream).view(torch.float32).view(sh.B, sh.Hq, sh.N)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    nws = bwd_workspace_bytes(q, k, causal)
    ws = _scratch(nws, q.device, stream) if nws else None
    run_bwd_ws(q, k, v, o, do, lse, delta, dq, dk, dv, ws, causal, scale, stream)
    return dq, dk, dv


# ----------------------------------------------------------- roofline probes --

def _time_ms(launch, reps: int) -> float:
    """Mean event time (ms) of `reps` back-to-back launches, after one warm-up."""
    torch = _torch()
    launch()
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize()
    start.record()
    for _ in range(reps):
        launch()
    stop.record()
    torch.cuda.synchronize()
    return start.elapsed_time(stop) / reps


def probe_mfma_tflops(bf16: bool = True, iters: int = 256, reps: int = 5, big: bool = False) -> float:
    """Measured MFMA throughput (TFLOP/s) of the whole device: every wave issues
    independent v_mfma_f32_16x16x32_bf16 (bf16), v_mfma_f32_32x32x16_bf16
    (bf16, big) or v_mfma_f32_16x16x4_f32 (fp32)."""
    torch = _torch()
    lib = load_library()
    sink = torch.empty(lib.mxfa_probe_sink_len(), dtype=torch.float32, device="cuda")
    flops = ctypes.c_double(0.0)
    dt = MXFA_BF16 if bf16 else MXFA_F32
    stream = _stream(None)

    def launch():
        sp = _ptr(sink, "sink", torch.float32)
        if bf16 and big:
            _check("mxfa_probe_mfma32", lib.mxfa_probe_mfma32(iters, sp, ctypes.byref(flops), stream))
        else:
            _check("mxfa_probe_mfma", lib.mxfa_probe_mfma(dt, iters, sp, ctypes.byref(flops), stream))
    ms = _time_ms(launch, reps)
    return flops.value / (ms * 1e-3) / 1e12


# The instruction mixes of mxfa_probe_mix (include/mxfa_probes.h, MXFA_PROBE_MIX_*).
PROBE_MIXES = {"mfma": 0, "dkv": 1, "dkv_valu": 2, "dkv_lds": 3, "dq": 4, "fwd": 5,
               "mfma32": 6, "dkv32": 7, "dq32": 8, "fwd32": 9}


def probe_mix_tflops(mix: str, waves_per_simd: int = 3, iters: int = 64, reps: int = 5) -> float:
    """MFMA throughput (TFLOP/s, whole device) of one of PROBE_MIXES issued with
    no dependencies between its instructions, at waves_per_simd waves per SIMD
    (mxfa_probe_mix): the instruction-issue ceiling of a kernel with that mix."""
    torch = _torch()
    lib = load_library()
    sink = torch.empty(lib.mxfa_probe_sink_len(), dtype=torch.float32, device="cuda")
    flops = ctypes.c_double(0.0)
    stream = _stream(None)
    mid = PROBE_MIXES[mix]

    def launch():
        _check("mxfa_probe_mix", lib.mxfa_probe_mix(mid, waves_per_simd, iters, _ptr(sink, "sink", torch.float32),
                                                    ctypes.byref(flops), stream))
    ms = _time_ms(launch, reps)
    return flops.value / (ms * 1e-3) / 1e12


def probe_wg_times():
    """The per-work-group timeline of the last forward or backward launch
    (mxfa_probe_wg_times; only with TIMELINE_CODE_OBJECT_PATH loaded): a uint64
    numpy array [groups, 8] by linear work-group index. Columns 0-3: 100 MHz
    real-time counter values (start, first stage staged, end of loop, stores
    acknowledged); 4: (kind << 32) | block (kind 0 = dQ and its query block,
    1 = dK/dV and its key block, 2 = forward and its query block); 5: its
    stages; 6: (XCC_ID << 32) | HW_ID, the XCD and the CU (HW_ID bits 8-11),
    shader engine (13-15) it ran on; 7: zero. Zero rows for indices the launch
    did not have (or an earlier launch's values)."""
    import numpy as np
    lib = load_library()
    avail = ctypes.c_size_t(0)
    _check("mxfa_probe_wg_times", lib.mxfa_probe_wg_times(None, 0, ctypes.byref(avail)))
    buf = np.zeros(avail.value // 8, dtype=np.uint64)
    _check("mxfa_probe_wg_times", lib.mxfa_probe_wg_times(buf.ctypes.data_as(ctypes.c_void_p), buf.nbytes,
                                                          ctypes.byref(avail)))
    return buf.reshape(-1, 8)


def probe_dq_atomic(bh: int = 48, n: int = 4096, atomic: bool = True, reps: int = 5) -> dict:
    """Time of the global writes a dQ pass fused into the dK/dV pass would make
    at a causal (bh heads, N = n, d = 64) shape (mxfa_probe_dq_atomic): fp32
    atomic adds, or with atomic=False plain stores of the same bytes. Returns
    {"us", "payload_bytes", "tbps"} (mean of reps launches after one warm-up)."""
    torch = _torch()
    lib = load_library()
    acc = torch.zeros(bh * n * 64, dtype=torch.float32, device="cuda")
    nbytes = ctypes.c_double(0.0)
    stream = _stream(None)

    def launch():
        _check("mxfa_probe_dq_atomic", lib.mxfa_probe_dq_atomic(_ptr(acc, "acc", torch.float32), bh, n,
                                                                  int(atomic), ctypes.byref(nbytes), stream))
    ms = _time_ms(launch, reps)
    return {"us": ms * 1e3, "payload_bytes": nbytes.value, "tbps": nbytes.value / (ms * 1e-3) / 1e12}


def probe_hbm_gbps(mib: int = 1024, reps: int = 5, copy: bool = False) -> float:
    """Measured HBM streaming bandwidth (GB/s): a grid-stride read of `mib` MiB
    (or, with copy=True, a copy of that size, counting read + write bytes)."""
    torch = _torch()
    lib = load_library()
    nbytes = mib * 2**20
    x = torch.ones(nbytes // 4, dtype=torch.float32, device="cuda")
    stream = _stream(None)
    if copy:
        y = torch.empty_like(x)

        def launch():
            _check("mxfa_probe_copy", lib.mxfa_probe_copy(_ptr(x, "x", torch.float32), _ptr(y, "y", torch.float32),
                                                          nbytes, stream))
        moved = 2 * nbytes
    else:
        sink = torch.empty(lib.mxfa_probe_sink_len(), dtype=torch.float32, device="cuda")

        def launch():
            _check("mxfa_probe_read", lib.mxfa_probe_read(_ptr(x, "x", torch.float32), nbytes,
                                                          _ptr(sink, "sink", torch.float32), stream))
        moved = nbytes
    ms = _time_ms(launch, reps)
    return moved / (ms * 1e-3) / 1e9


def init(device: int = 0):
    """mxfa_init: checks that ``device`` is a gfx950, makes it current and
    loads the code object on it."""
    _check("mxfa_init", load_library().mxfa_init(device))


def shutdown():
    """mxfa_shutdown: unloads the code object from every device it was loaded
    on (their work must have completed); the next launch loads it again."""
    _check("mxfa_shutdown", load_library().mxfa_shutdown())


def check_code_object(path: str | None = None) -> int:
    """mxfa_check_code_object: 0 if ``path`` (default: the library's code
    object) is a gfx950 code object, else the MXFA_ERR_CODE_OBJECT status. Host
    only, no device access."""
    return int(load_library().mxfa_check_code_object(path.encode() if path else None))


def set_code_object(path: str | None):
    """mxfa_set_code_object: the code object file later loads read (None: the
    default beside libmxfa.so)."""
    _check("mxfa_set_code_object", load_library().mxfa_set_code_object(path.encode() if path else None))


# The reference's benchmark counts (02-flash-attention/src/main.rs:15-16).
WARMUP = 1
ITERS = 5


def time_median_ms(fn, warmup: int = WARMUP, iters: int = ITERS, stream=None) -> float:
    """Median time of one invocation of `fn` in milliseconds, as
    common/src/lib.rs:22-43 (time_median_ms) measures it: `warmup` calls, a
    synchronisation of the stream, then `iters` calls each bracketed by a pair
    of HIP events on the stream and waited for; the median is the sorted
    times' element iters // 2. `fn` enqueues its work on `stream` (default:
    torch's current stream)."""
    torch = _torch()
    if iters < 1:
        raise ValueError(f"iters must be at least 1 (got {iters})")
    s = stream if stream is not None else torch.cuda.current_stream()
    for _ in range(warmup):
        fn()
    s.synchronize()
    times = []
    for _ in range(iters):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record(s)
        fn()
        end.record(s)
        end.synchronize()
        times.append(start.elapsed_time(end))
    times.sort()
    return times[len(times) // 2]


def fwd_flops(B, Hq, N, d, causal) -> float:
    """Algorithmic forward flops: 4 N^2 d per (batch, query head), halved if causal."""
    return 4.0 * N * N * d * B * Hq * (0.5 if causal else 1.0)


def bwd_flops(B, Hq, N, d, causal) -> float:
    """Algorithmic backward flops: 10 N^2 d per (batch, query head), halved if causal."""
    return 10.0 * N * N * d * B * Hq * (0.5 if causal else 1.0)
