"""ctypes binding of libcortex_b200.so (the C ABI in include/cortex_b200.h).

The shared library is built in-tree by ``cortex-engine_b200/build.py`` and sits
next to this file. There is no fallback: if the library is missing or no CUDA
device is present, every kernel entry point raises.
"""

from __future__ import annotations

import ctypes
import os
import struct
import threading

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libcortex_b200.so")

CK_OK = 0
CK_ERR_INVALID_ARG = -1
CK_ERR_UNSUPPORTED = -2
CK_ERR_CUDA = -3
CK_ERR_INDEX = -4
CK_ERR_TIMEOUT = -5
CK_ERR_WORKSPACE = -6

CK_F32, CK_BF16, CK_I8, CK_I32, CK_I64 = 0, 1, 2, 3, 4
CK_NORM_NONE, CK_NORM_LAYER, CK_NORM_RMS = 0, 1, 2
CK_EPI_STORE, CK_EPI_GELU, CK_EPI_RESID, CK_EPI_BIAS = 0, 1, 2, 3
CK_W_NK, CK_W_KN = 0, 1

_vp = ctypes.c_void_p
_i32 = ctypes.c_int32
_i64 = ctypes.c_int64
_int = ctypes.c_int
_f32 = ctypes.c_float
_sz = ctypes.c_size_t


class AttentionArgs(ctypes.Structure):
    _fields_ = [
        ("dtype", _int),
        ("B", _i32), ("H", _i32), ("Dh", _i32), ("Lq", _i32),
        ("n_keys", _i32),
        ("key_offsets", _vp),
        ("q", _vp), ("q_ld", _i64), ("q_rows", _i64), ("q_rows_per_b", _i64),
        ("q_rows_per_h", _i64), ("q_col_per_h", _i64),
        ("k", _vp), ("k_ld", _i64), ("k_rows", _i64), ("k_rows_per_b", _i64),
        ("k_rows_per_h", _i64), ("k_col_per_h", _i64),
        ("v", _vp), ("v_ld", _i64), ("v_rows", _i64), ("v_rows_per_b", _i64),
        ("v_rows_per_h", _i64), ("v_col_per_h", _i64),
        ("o", _vp), ("o_ld", _i64), ("o_rows_per_b", _i64), ("o_rows_per_h", _i64),
        ("o_col_per_h", _i64),
        ("block_mask", _vp),
        ("n_q_tiles", _i32), ("n_k_tiles", _i32), ("block_l", _i32), ("block_e", _i32),
        ("key_mask", _vp), ("key_mask_ld", _i64),
        ("scale", _f32),
    ]


class LinearWeight(ctypes.Structure):
    _fields_ = [("w", _vp), ("dtype", _int), ("scale", _vp), ("bias", _vp)]


class BlockWeights(ctypes.Structure):
    _fields_ = [
        ("norm_attn_w", _vp), ("norm_attn_b", _vp),
        ("qkv", LinearWeight), ("out", LinearWeight),
        ("norm_mlp_w", _vp), ("norm_mlp_b", _vp),
        ("mlp0", LinearWeight), ("mlp2", LinearWeight),
    ]


class Model(ctypes.Structure):
    _fields_ = [
        ("dtype", _int),
        ("hidden_dim", _i32), ("latent_dim", _i32), ("num_latents", _i32),
        ("num_layers", _i32), ("num_heads", _i32), ("head_dim", _i32),
        ("cross_heads", _i32), ("mlp_hidden", _i32), ("behavior_dim", _i32),
        ("n_vocab", _i64), ("t_vocab", _i64), ("v_vocab", _i64),
        ("neuron_emb", _vp), ("time_emb", _vp), ("value_emb", _vp),
        ("latents", _vp),
        ("norm_q_w", _vp), ("norm_q_b", _vp), ("norm_kv_w", _vp), ("norm_kv_b", _vp),
        ("cross_q", LinearWeight), ("cross_kv", LinearWeight), ("cross_out", LinearWeight),
        ("blocks", ctypes.POINTER(BlockWeights)),
        ("final_norm_w", _vp), ("final_norm_b", _vp),
        ("head_query", _vp),
        ("head_norm_w", _vp), ("head_norm_b", _vp),
        ("head_q", LinearWeight), ("head_kv", LinearWeight), ("head_out", LinearWeight),
    ]


class PagedAttentionArgs(ctypes.Structure):
    _fields_ = [
        ("dtype", _int),
        ("B", _i32), ("H", _i32), ("Hkv", _i32), ("Dh", _i32),
        ("q", _vp), ("q_ld_b", _i64), ("q_ld_h", _i64),
        ("pool", _vp), ("num_pages", _i64), ("page_ld", _i64), ("row_ld", _i64),
        ("page_size", _i32), ("page_table_width", _i32),
        ("page_table", _vp), ("page_table_ld", _i64),
        ("lengths", _vp),
        ("o", _vp), ("o_ld_b", _i64), ("o_ld_h", _i64),
        ("w_in", _vp), ("w_out", _vp), ("w_in_ld", _i64), ("w_out_ld", _i64), ("w_width", _i64),
        ("scale", _f32),
    ]


class EvictArgs(ctypes.Structure):
    _fields_ = [
        ("elem_bytes", _int), ("B", _i32),
        ("pool", _vp), ("num_pages", _i64), ("page_ld", _i64), ("row_ld", _i64),
        ("page_size", _i32), ("width", _i32),
        ("page_table", _vp), ("page_table_ld", _i64), ("page_table_width", _i32),
        ("budget", _i32), ("recent", _i32), ("fill", _i32),
        ("lengths", _vp), ("lengths_out", _vp),
        ("w_in", _vp), ("w_out", _vp), ("pos_in", _vp), ("pos_out", _vp),
        ("w_in_ld", _i64), ("w_out_ld", _i64), ("pos_in_ld", _i64), ("pos_out_ld", _i64),
        ("in_width", _i32), ("out_width", _i32),
    ]


class LoraArgs(ctypes.Structure):
    _fields_ = [
        ("dtype", _int), ("n_adapters", _i32), ("rank", _i32),
        ("M", _i64), ("K", _i64), ("N", _i64),
        ("x", _vp), ("ldx", _i64), ("w", _vp), ("ldw", _i64), ("a", _vp), ("b", _vp),
        ("ids", _vp), ("scaling", _vp), ("bias", _vp), ("y", _vp), ("ldy", _i64),
    ]


# The argument blocks of the serving operators as struct formats (native layout,
# the fields of PagedAttentionArgs, EvictArgs and LoraArgs in order): packing a
# block this way costs a tenth of filling a ctypes.Structure, on calls whose
# kernels take a few microseconds.
PAGED_ATTENTION_ARGS = struct.Struct("@5iP2qP3q2iPqPP2q2P3qf0q")
EVICT_ARGS = struct.Struct("@2iP3q2iPq4i6P4q2i0q")
LORA_ARGS = struct.Struct("@3i3qPqPq2PPPPPq0q")


class TraceRecord(ctypes.Structure):
    _fields_ = [("name", ctypes.c_char * 96), ("stream", _vp), ("ms", _f32)]


_SIGS = {
    "ck_get_last_status": (_int, [ctypes.POINTER(_int)]),
    "ck_last_cuda_error": (_int, []),
    "ck_status_string": (ctypes.c_char_p, [_int]),
    "ck_num_sms": (_int, []),
    "ck_launch_count": (ctypes.c_longlong, []),
    "ck_trace_begin": (_int, [_i32]),
    "ck_trace_end": (_int, [ctypes.POINTER(TraceRecord), _i32, ctypes.POINTER(_i32)]),
    "ck_pack_workspace_bytes": (_sz, [_i64, _i32]),
    "ck_pack_events": (_int, [_vp, _int, _i64, _i64, _i32, _vp, _vp, _vp, _vp, _vp, _sz, _vp]),
    "ck_pack_scatter": (_int, [_vp, _int, _i64, _i32, _i64, _vp, _int, _i64, _vp, _vp, _i32,
                               _vp, _vp, _vp]),
    "ck_tokenize": (_int, [_vp, _vp, _vp, _int, _i32, _i64, _i64, _i64, _i64, _i64, _i64, _vp,
                           _vp, _vp, _int, _i64, _i64, _i64, _i64, _vp, _vp, _vp, _f32, _vp,
                           _i64, _vp]),
    "ck_dequantize_int8": (_int, [_vp, _vp, _i64, _i64, _i64, _vp, _i64, _vp]),
    "ck_tokenize_packed_workspace_bytes": (_sz, []),
    "ck_tokenize_packed": (_int, [_vp, _vp, _vp, _int, _i32, _i64, _i64, _i64, _vp, _vp, _vp, _vp,
                                  _int, _i64, _i32, _vp, _vp, _f32, _vp, _i64, _vp, _vp, _sz,
                                  _vp]),
    "ck_row_norm": (_int, [_vp, _int, _i64, _i32, _i64, _vp, _vp, _f32, _int, _vp, _i64, _vp]),
    "ck_linear": (_int, [_vp, _int, _i64, _i64, _i64, _vp, _int, _int, _i64, _i64, _vp, _int,
                         _vp, _i64, _i64, _vp, _i64, _vp]),
    "ck_norm_linear_workspace_bytes": (_sz, [_int, _i64, _i64]),
    "ck_norm_linear": (_int, [_vp, _int, _i64, _i64, _i64, _vp, _vp, _f32, _int, _vp, _int,
                              _int, _i64, _i64, _vp, _int, _vp, _i64, _i64, _vp, _i64, _vp,
                              _sz, _vp]),
    "ck_norm_linear_static": (_int, [_vp, _int, _i64, _i64, _i64, _vp, _vp, _f32, _int, _vp,
                                     _int, _int, _i64, _i64, _vp, _int, _vp, _i64, _i64, _vp,
                                     _i64, _vp]),
    "ck_attention": (_int, [ctypes.POINTER(AttentionArgs), _vp]),
    "ck_forward_workspace_bytes": (_sz, [ctypes.POINTER(Model), _i64, _i32]),
    "ck_forward": (_int, [ctypes.POINTER(Model), _vp, _vp, _vp, _vp, _int, _i64, _i32, _vp, _vp,
                          _sz, _vp]),
    "ck_batch_stage": (_int, [_vp, _vp, _vp, _vp, _int, _i64, _vp, _i64,
                              ctypes.POINTER(_i32)]),
    "ck_forward_batch": (_int, [ctypes.POINTER(Model), _vp, _i64, _i32, _vp, _vp, _sz, _vp]),
    "ck_runner_create": (_int, [ctypes.POINTER(Model), _i32, ctypes.POINTER(_vp)]),
    "ck_runner_destroy": (None, [_vp]),
    "ck_runner_stage": (_int, [_vp, _vp, _vp, _vp, _vp, _int, _i64, _i32, ctypes.POINTER(_i32)]),
    "ck_runner_launch": (_int, [_vp, _vp, _vp]),
    "ck_runner_launch_batch": (_int, [_vp, _vp, _i64, _i32, _vp, _vp]),
    "ck_runner_invalidate": (_int, [_vp, ctypes.POINTER(Model)]),
    "ck_runner_counters": (_int, [_vp, ctypes.POINTER(ctypes.c_longlong),
                                  ctypes.POINTER(ctypes.c_longlong)]),
    "ck_forward_kv": (_int, [ctypes.POINTER(Model), _vp, _i64, _i32, _vp, _vp, _vp, _sz, _vp]),
    "ck_forward_from_kv": (_int, [ctypes.POINTER(Model), _vp, _i64, _vp, _i32, _vp, _vp, _sz,
                                  _vp]),
    "ck_copy_rows": (_int, [_vp, _i64, _vp, _i64, _i64, _vp, _i32, _vp]),
    "ck_collate_bins_workspace_bytes": (_sz, [_i32, _i32]),
    "ck_collate_bins": (_int, [_vp, _i32, _i32, _i32, _i32, _vp, _i64, _vp, _sz, _vp, _vp]),
    "ck_paged_attention_workspace_bytes": (_sz, [_vp]),
    "ck_evict_workspace_bytes": (_sz, [_vp]),
    "ck_evict_by_weight": (_int, [_vp, _vp, _sz, _vp]),
    "ck_lora_workspace_bytes": (_sz, [_vp]),
    "ck_lora_linear": (_int, [_vp, _vp, _sz, _vp]),
    "ck_paged_attention": (_int, [_vp, _vp, _sz, _vp]),
}

CK_BATCH_HEADER_WORDS = 4


def batch_words(capacity: int) -> int:
    """int32 words of a packed event batch (CK_BATCH_WORDS in cortex_b200.h)."""
    return CK_BATCH_HEADER_WORDS + 4 * capacity

EXPORTED_SYMBOLS = tuple(_SIGS)

_lib = None
_lock = threading.Lock()


def load() -> ctypes.CDLL:
    """Load the shared library (raises if it has not been built)."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise RuntimeError(
                    f"{LIB_PATH} is missing: build it with `python cortex-engine_b200/build.py`")
            lib = ctypes.CDLL(LIB_PATH)
            for name, (res, args) in _SIGS.items():
                fn = getattr(lib, name)
                fn.restype = res
                fn.argtypes = args
            _lib = lib
    return _lib


def memory_range(t: torch.Tensor) -> tuple[int, int]:
    """[first, last) byte address that ``t``'s elements lie in."""
    p = t.data_ptr()
    if t.numel() == 0:
        return p, p
    span = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return p, p + (span + 1) * t.element_size()


def check_output(what: str, name: str, out: torch.Tensor, *inputs: torch.Tensor | None) -> None:
    """An output that a caller provides: its elements must not share memory with
    each other or lie within the span of an input."""
    dims = sorted((s, n) for n, s in zip(out.shape, out.stride()) if n > 1)
    reach = 0
    for s, n in dims:
        if s <= reach:
            raise ValueError(f"{what}: elements of {name} share memory")
        reach += s * (n - 1)
    lo, hi = memory_range(out)
    for t in inputs:
        if t is not None:
            a, b = memory_range(t)
            if a < hi and lo < b:
                raise ValueError(f"{what}: {name} overlaps an input")


class DeviceStatusError(RuntimeError):
    pass


def status_string(code: int) -> str:
    return load().ck_status_string(code).decode()


def check(rc: int, what: str) -> None:
    if rc == CK_OK:
        return
    msg = f"{what}: {status_string(rc)} (code {rc})"
    if rc == CK_ERR_CUDA:
        msg += f", cudaError {load().ck_last_cuda_error()}"
    if rc == CK_ERR_INVALID_ARG:
        raise ValueError(msg)
    if rc == CK_ERR_UNSUPPORTED:
        raise NotImplementedError(msg)
    if rc == CK_ERR_INDEX:
        raise IndexError(msg)
    raise RuntimeError(msg)


def device_status(clear: bool = True) -> tuple[int, list[int]]:
    """Synchronise the current device and read (then clear) its status word."""
    info = (_int * 4)()
    code = load().ck_get_last_status(info)
    return int(code), list(info)


def check_device_status(what: str = "device") -> None:
    code, info = device_status()
    if code == CK_OK:
        return
    msg = f"{what}: {status_string(code)} (code {code}, info {info})"
    if code == CK_ERR_INDEX:
        raise IndexError(msg)
    raise DeviceStatusError(msg)


def dtype_code(dt: torch.dtype) -> int:
    if dt == torch.float32:
        return CK_F32
    if dt == torch.bfloat16:
        return CK_BF16
    if dt == torch.int8:
        return CK_I8
    if dt == torch.int32:
        return CK_I32
    if dt == torch.int64:
        return CK_I64
    raise NotImplementedError(f"dtype {dt} is not supported by the B200 kernels "
                              "(float32, bfloat16, int8 weights, int32/int64 indices)")


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_of(device: torch.device) -> int:
    """The handle of torch's current CUDA stream on ``device``."""
    if _raw_stream is not None:
        idx = device.index
        return _raw_stream(torch.cuda.current_device() if idx is None else idx)
    return torch.cuda.current_stream(device).cuda_stream


_ws_bytes: dict = {}


def launch(what: str, call, query, key: tuple, block: bytes, dev: torch.device, stream: int) -> None:
    """``call(block, workspace, bytes, stream)`` with a workspace on ``dev`` of the
    size that ``query(block)`` gives. The size is remembered per ``key`` (the
    call's sizes) once a call with it has been accepted: a refused argument
    block has no size."""
    n = _ws_bytes.get(key)
    known = n is not None
    if not known:
        n = query(block)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    rc = call(block, ws.data_ptr() if n else 0, n, stream)
    if rc != CK_OK:
        check(rc, what)
    if not known:
        if len(_ws_bytes) > 4096:
            _ws_bytes.clear()
        _ws_bytes[key] = n


_get_device = getattr(torch._C, "_cuda_getDevice", None)


def current_device() -> int:
    """Index of the current CUDA device."""
    return _get_device() if _get_device is not None else torch.cuda.current_device()


def raw_stream(index: int) -> int:
    """The handle of torch's current CUDA stream on device ``index``."""
    if _raw_stream is not None:
        return _raw_stream(index)
    return torch.cuda.current_stream(index).cuda_stream


def require_cuda(*tensors: torch.Tensor, what: str) -> torch.device:
    """All tensors must live on one CUDA device; there is no CPU path."""
    dev = None
    for t in tensors:
        if t is None:
            continue
        if t.device.type != "cuda":
            raise RuntimeError(
                f"{what}: the B200 kernels need CUDA tensors (got {t.device}); "
                "this package has no CPU fallback")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"{what}: tensors are on different devices ({dev}, {t.device})")
    if dev is None:
        raise RuntimeError(f"{what}: no tensor given")
    load()
    return dev
