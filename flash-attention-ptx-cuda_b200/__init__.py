"""Python binding of libfa_b200.so over its C ABI (include/fa_b200.h), via ctypes.

The product is the shared library; this module only marshals pointers so that
tests, the benchmark and Python callers reach the same entry points a C, Go or
Rust binding would.  There is no fallback path: if the library is missing or
the device is not a B200-class GPU, calls raise.

The directory name contains hyphens, so it cannot be imported with a plain
``import`` statement; ``__graft_entry__.load_package()`` loads it under the
module name ``fa_b200``.

Device memory is handled by the caller.  The helpers here accept raw integer
device pointers, or any object with ``data_ptr()`` (torch tensors are used for
allocation and streams only).
"""
from __future__ import annotations

import ctypes
import os
import struct

HERE = os.path.dirname(os.path.abspath(__file__))
# FA_B200_LIB points the binding at another build of the same library (development only).
LIB_PATH = os.environ.get("FA_B200_LIB") or os.path.join(HERE, "libfa_b200.so")

FA_OK = 0
FA_ERR_INVALID_ARGUMENT = -1
FA_ERR_UNSUPPORTED = -2
FA_ERR_MISALIGNED = -3
FA_ERR_WORKSPACE = -4
FA_ERR_CUDA = -5
FA_ERR_DEVICE_TIMEOUT = -6
FA_ERR_NOT_SM100 = -7
FA_ERR_NCCL = -8
FA_DTYPE_F16, FA_DTYPE_BF16, FA_DTYPE_E4M3 = 0, 1, 2
DTYPES = {"f16": FA_DTYPE_F16, "bf16": FA_DTYPE_BF16, "e4m3": FA_DTYPE_E4M3}
FA_CACHE_16BIT, FA_CACHE_E4M3, FA_CACHE_U4 = 0, 1, 2
CACHES = {"f16": FA_CACHE_16BIT, "bf16": FA_CACHE_16BIT, "e4m3": FA_CACHE_E4M3, "u4": FA_CACHE_U4}
ROPE_SCALINGS = {"plain": 0, "linear": 1, "base": 2, "parts": 3, "smooth": 4}

# Every symbol include/fa_b200.h declares; the CPU-only tests check they all resolve.
EXPORTED_SYMBOLS = (
    "fa_prefill", "fa_prefill_host", "fa_decode", "fa_decode_static", "fa_decode_workspace_bytes",
    "fa_decode_default_splits", "fa_decode_gqa", "fa_decode_gqa_default_splits", "fa_backward",
    "fa_backward_workspace_bytes", "fa_combine", "fa_kat",
    "fa_device_status",
    "fa_clear_device_status", "fa_error_string", "fa_last_cuda_error", "fa_version",
    "fa_set_prefill_variant", "fa_combine_packed", "fa_decode_kv_sharded", "fa_decode_kv_sharded_gather_bytes",
    "fa_nccl_unique_id", "fa_nccl_comm_create", "fa_nccl_comm_destroy", "fa_status_word_to_error",
    "fa_rope", "fa_rope_inv_freq", "fa_cache_append", "fa_cache_read_u4", "fa_decode_gqa_u4",
    "fa_decode_gqa_u4_workspace_bytes",
)


class PrefillArgs(ctypes.Structure):
    """Mirror of ``fa_prefill_args`` (include/fa_b200.h)."""
    _fields_ = [
        ("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
        ("o", ctypes.c_void_p), ("lse", ctypes.c_void_p),
        ("batch_size", ctypes.c_int), ("num_heads", ctypes.c_int), ("seq_len", ctypes.c_int),
        ("d_head", ctypes.c_int), ("scale", ctypes.c_float), ("causal", ctypes.c_int),
        ("dtype", ctypes.c_int),
        ("q_scale", ctypes.c_void_p), ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p),
        ("stream", ctypes.c_void_p),
    ]


class DecodeArgs(ctypes.Structure):
    """Mirror of ``fa_decode_args`` (include/fa_b200.h)."""
    _fields_ = [
        ("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
        ("o", ctypes.c_void_p), ("lse", ctypes.c_void_p), ("o_f32", ctypes.c_void_p),
        ("batch_size", ctypes.c_int), ("num_heads", ctypes.c_int), ("seq_len_kv", ctypes.c_int),
        ("d_head", ctypes.c_int), ("scale", ctypes.c_float), ("dtype", ctypes.c_int),
        ("num_splits", ctypes.c_int),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
        ("stream", ctypes.c_void_p),
    ]


class DecodeGqaArgs(ctypes.Structure):
    """Mirror of ``fa_decode_gqa_args`` (include/fa_b200.h)."""
    _fields_ = [
        ("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
        ("o", ctypes.c_void_p), ("lse", ctypes.c_void_p),
        ("batch_size", ctypes.c_int), ("num_q_heads", ctypes.c_int), ("num_kv_heads", ctypes.c_int),
        ("seq_len_kv", ctypes.c_int), ("d_head", ctypes.c_int), ("scale", ctypes.c_float),
        ("dtype", ctypes.c_int), ("num_splits", ctypes.c_int),
        ("kv_batch_stride", ctypes.c_longlong), ("kv_head_stride", ctypes.c_longlong),
        ("kv_row_stride", ctypes.c_longlong),
        ("block_table", ctypes.c_void_p), ("block_table_stride", ctypes.c_int), ("page_size", ctypes.c_int),
        ("num_pages", ctypes.c_int), ("kv_page_stride", ctypes.c_longlong), ("seq_lens", ctypes.c_void_p),
        ("q_scale", ctypes.c_void_p), ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p),
        ("num_q_tokens", ctypes.c_int),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
        ("stream", ctypes.c_void_p),
    ]


class BackwardArgs(ctypes.Structure):
    """Mirror of ``fa_backward_args`` (include/fa_b200.h)."""
    _fields_ = [
        ("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("o", ctypes.c_void_p),
        ("d_o", ctypes.c_void_p), ("lse", ctypes.c_void_p),
        ("dq", ctypes.c_void_p), ("dk", ctypes.c_void_p), ("dv", ctypes.c_void_p),
        ("batch_size", ctypes.c_int), ("num_heads", ctypes.c_int), ("seq_len", ctypes.c_int),
        ("d_head", ctypes.c_int), ("scale", ctypes.c_float), ("causal", ctypes.c_int), ("dtype", ctypes.c_int),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t), ("stream", ctypes.c_void_p),
    ]


class Rotary(ctypes.Structure):
    """Mirror of ``fa_rotary`` (include/fa_b200.h)."""
    _fields_ = [("inv_freq", ctypes.c_void_p), ("rotary_dim", ctypes.c_int), ("interleaved", ctypes.c_int),
                ("amplitude", ctypes.c_float)]


class Strides(ctypes.Structure):
    """Mirror of ``fa_strides`` (include/fa_b200.h)."""
    _fields_ = [("batch", ctypes.c_longlong), ("head", ctypes.c_longlong), ("row", ctypes.c_longlong)]


class RopeArgs(ctypes.Structure):
    """Mirror of ``fa_rope_args`` (include/fa_b200.h)."""
    _fields_ = [
        ("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("q_out", ctypes.c_void_p), ("k_out", ctypes.c_void_p),
        ("q_strides", Strides), ("k_strides", Strides), ("q_out_strides", Strides), ("k_out_strides", Strides),
        ("batch_size", ctypes.c_int), ("num_q_heads", ctypes.c_int), ("num_kv_heads", ctypes.c_int),
        ("seq_len", ctypes.c_int), ("d_head", ctypes.c_int), ("dtype", ctypes.c_int),
        ("positions", ctypes.c_void_p), ("positions_stride", ctypes.c_int), ("position_offset", ctypes.c_int),
        ("inverse", ctypes.c_int), ("rotary", Rotary), ("stream", ctypes.c_void_p),
    ]


class RopeScaling(ctypes.Structure):
    """Mirror of ``fa_rope_scaling`` (include/fa_b200.h)."""
    _fields_ = [("kind", ctypes.c_int), ("base", ctypes.c_double), ("factor", ctypes.c_double),
                ("original_length", ctypes.c_double), ("slow", ctypes.c_double), ("fast", ctypes.c_double)]


class CacheLayout(ctypes.Structure):
    """Mirror of ``fa_cache_layout`` (include/fa_b200.h)."""
    _fields_ = [
        ("block_stride", ctypes.c_longlong), ("head_stride", ctypes.c_longlong), ("row_stride", ctypes.c_longlong),
        ("param_block_stride", ctypes.c_longlong), ("param_head_stride", ctypes.c_longlong),
        ("param_row_stride", ctypes.c_longlong),
        ("block_table", ctypes.c_void_p), ("block_table_stride", ctypes.c_int), ("page_size", ctypes.c_int),
        ("num_pages", ctypes.c_int), ("seq_lens", ctypes.c_void_p),
    ]


class CacheAppendArgs(ctypes.Structure):
    """Mirror of ``fa_cache_append_args`` (include/fa_b200.h)."""
    _fields_ = [
        ("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("q_out", ctypes.c_void_p),
        ("k_cache", ctypes.c_void_p), ("v_cache", ctypes.c_void_p), ("k_params", ctypes.c_void_p),
        ("v_params", ctypes.c_void_p),
        ("q_token_stride", ctypes.c_longlong), ("k_token_stride", ctypes.c_longlong), ("v_token_stride", ctypes.c_longlong),
        ("batch_size", ctypes.c_int), ("num_tokens", ctypes.c_int), ("num_q_heads", ctypes.c_int),
        ("num_kv_heads", ctypes.c_int), ("seq_len_kv", ctypes.c_int), ("d_head", ctypes.c_int),
        ("dtype", ctypes.c_int), ("cache", ctypes.c_int), ("layout", CacheLayout),
        ("num_new", ctypes.c_void_p), ("positions", ctypes.c_void_p), ("rotary", Rotary),
        ("q_scale", ctypes.c_void_p), ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p),
        ("stream", ctypes.c_void_p),
    ]


class CacheReadArgs(ctypes.Structure):
    """Mirror of ``fa_cache_read_args`` (include/fa_b200.h)."""
    _fields_ = [
        ("k_cache", ctypes.c_void_p), ("k_params", ctypes.c_void_p), ("v_cache", ctypes.c_void_p),
        ("v_params", ctypes.c_void_p), ("k_out", ctypes.c_void_p), ("v_out", ctypes.c_void_p),
        ("batch_size", ctypes.c_int), ("num_kv_heads", ctypes.c_int), ("seq_len_kv", ctypes.c_int),
        ("d_head", ctypes.c_int), ("num_rows", ctypes.c_int), ("dtype", ctypes.c_int), ("layout", CacheLayout),
        ("first_rows", ctypes.c_void_p), ("stream", ctypes.c_void_p),
    ]


class DecodeGqaU4Args(ctypes.Structure):
    """Mirror of ``fa_decode_gqa_u4_args`` (include/fa_b200.h)."""
    _fields_ = [
        ("q", ctypes.c_void_p), ("k_cache", ctypes.c_void_p), ("k_params", ctypes.c_void_p),
        ("v_cache", ctypes.c_void_p), ("v_params", ctypes.c_void_p), ("o", ctypes.c_void_p), ("lse", ctypes.c_void_p),
        ("batch_size", ctypes.c_int), ("num_q_heads", ctypes.c_int), ("num_kv_heads", ctypes.c_int),
        ("num_q_tokens", ctypes.c_int), ("seq_len_kv", ctypes.c_int), ("d_head", ctypes.c_int), ("scale", ctypes.c_float),
        ("dtype", ctypes.c_int), ("layout", CacheLayout),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t), ("stream", ctypes.c_void_p),
    ]


def _packer(cls):
    """``struct.Struct(...).pack`` with the memory layout of a ctypes structure, nested ones flattened.  An argument block
    packed this way takes a serving step's call a third of the time that building the ctypes object takes (40 fields:
    1.5 us against 5)."""
    codes = {ctypes.c_void_p: "Q", ctypes.c_int: "i", ctypes.c_longlong: "q", ctypes.c_size_t: "Q", ctypes.c_float: "f",
             ctypes.c_double: "d"}
    fmt, at = ["="], 0

    def walk(c, base):
        nonlocal at
        for name, t in c._fields_:
            off = base + getattr(c, name).offset
            if issubclass(t, ctypes.Structure):
                walk(t, off)
            else:
                fmt.append(f"{off - at}x{codes[t]}" if off > at else codes[t])
                at = off + ctypes.sizeof(t)

    walk(cls, 0)
    fmt.append(f"{ctypes.sizeof(cls) - at}x")
    return struct.Struct("".join(fmt)).pack


_pack_rope, _pack_append, _pack_read, _pack_decode_u4 = map(_packer, (RopeArgs, CacheAppendArgs, CacheReadArgs, DecodeGqaU4Args))


class FaError(RuntimeError):
    def __init__(self, code: int, what: str):
        super().__init__(f"{what}: {error_string(code)} ({code})"
                         + (f" [{last_cuda_error()}]" if code == FA_ERR_CUDA else ""))
        self.code = code


_lib = None


def lib() -> ctypes.CDLL:
    """Loads libfa_b200.so (no fallback: a missing library is an error)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise FileNotFoundError(
                f"{LIB_PATH} not built; run `python flash-attention-ptx-cuda_b200/build.py`")
        l = ctypes.CDLL(LIB_PATH)
        l.fa_prefill.restype = ctypes.c_int
        l.fa_prefill.argtypes = [ctypes.POINTER(PrefillArgs)]
        l.fa_prefill_host.restype = ctypes.c_int
        l.fa_prefill_host.argtypes = [ctypes.POINTER(PrefillArgs)]
        l.fa_decode.restype = ctypes.c_int
        l.fa_decode.argtypes = [ctypes.POINTER(DecodeArgs)]
        l.fa_decode_static.restype = ctypes.c_int
        l.fa_decode_static.argtypes = [ctypes.POINTER(DecodeArgs)]
        l.fa_decode_workspace_bytes.restype = ctypes.c_size_t
        l.fa_decode_workspace_bytes.argtypes = [ctypes.c_int] * 4
        l.fa_decode_default_splits.restype = ctypes.c_int
        l.fa_decode_default_splits.argtypes = [ctypes.c_int] * 3
        l.fa_decode_gqa.restype = ctypes.c_int
        l.fa_decode_gqa.argtypes = [ctypes.POINTER(DecodeGqaArgs)]
        l.fa_decode_gqa_default_splits.restype = ctypes.c_int
        l.fa_decode_gqa_default_splits.argtypes = [ctypes.c_int] * 3
        l.fa_backward.restype = ctypes.c_int
        l.fa_backward.argtypes = [ctypes.POINTER(BackwardArgs)]
        l.fa_backward_workspace_bytes.restype = ctypes.c_size_t
        l.fa_backward_workspace_bytes.argtypes = [ctypes.c_int] * 3
        l.fa_combine.restype = ctypes.c_int
        l.fa_combine.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_int,
                                 ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int,
                                 ctypes.c_void_p]
        l.fa_kat.restype = ctypes.c_int
        l.fa_kat.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p,
                             ctypes.c_void_p, ctypes.c_float, ctypes.c_void_p, ctypes.c_void_p]
        l.fa_device_status.restype = ctypes.c_int
        l.fa_device_status.argtypes = [ctypes.POINTER(ctypes.c_int)]
        l.fa_clear_device_status.restype = ctypes.c_int
        l.fa_error_string.restype = ctypes.c_char_p
        l.fa_error_string.argtypes = [ctypes.c_int]
        l.fa_last_cuda_error.restype = ctypes.c_char_p
        l.fa_version.restype = ctypes.c_int
        l.fa_combine_packed.restype = ctypes.c_int
        l.fa_combine_packed.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_void_p,
                                        ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p]
        l.fa_decode_kv_sharded.restype = ctypes.c_int
        l.fa_decode_kv_sharded.argtypes = [ctypes.POINTER(DecodeArgs), ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t]
        l.fa_decode_kv_sharded_gather_bytes.restype = ctypes.c_size_t
        l.fa_decode_kv_sharded_gather_bytes.argtypes = [ctypes.c_int] * 4
        l.fa_nccl_unique_id.restype = ctypes.c_int
        l.fa_nccl_unique_id.argtypes = [ctypes.c_void_p, ctypes.c_size_t]
        l.fa_nccl_comm_create.restype = ctypes.c_int
        l.fa_nccl_comm_create.argtypes = [ctypes.POINTER(ctypes.c_void_p), ctypes.c_int, ctypes.c_void_p, ctypes.c_size_t,
                                          ctypes.c_int]
        l.fa_nccl_comm_destroy.restype = ctypes.c_int
        l.fa_nccl_comm_destroy.argtypes = [ctypes.c_void_p]
        l.fa_status_word_to_error.restype = ctypes.c_int
        l.fa_status_word_to_error.argtypes = [ctypes.c_int]
        l.fa_set_prefill_variant.restype = ctypes.c_int
        l.fa_set_prefill_variant.argtypes = [ctypes.c_int]
        for name in ("fa_rope", "fa_cache_append", "fa_cache_read_u4", "fa_decode_gqa_u4"):
            getattr(l, name).restype = ctypes.c_int
            getattr(l, name).argtypes = [ctypes.c_void_p]              # a packed block, or byref() of the mirror
        l.fa_rope_inv_freq.restype = ctypes.c_int
        l.fa_rope_inv_freq.argtypes = [ctypes.POINTER(RopeScaling), ctypes.c_int, ctypes.POINTER(ctypes.c_double),
                                       ctypes.POINTER(ctypes.c_float)]
        l.fa_decode_gqa_u4_workspace_bytes.restype = ctypes.c_size_t
        l.fa_decode_gqa_u4_workspace_bytes.argtypes = [ctypes.c_int] * 6
        _lib = l
    return _lib


def error_string(code: int) -> str:
    return lib().fa_error_string(code).decode()


def last_cuda_error() -> str:
    return lib().fa_last_cuda_error().decode()


def _ptr(x) -> int | None:
    if x is None:
        return None
    if isinstance(x, int):
        return x
    return x.data_ptr()


def _stream_handle(stream) -> int | None:
    if stream is None:
        return None
    if isinstance(stream, int):
        return stream or None
    return stream.cuda_stream or None


def prefill_raw(q, k, v, o, lse, batch_size, num_heads, seq_len, d_head, scale, causal,
                dtype="f16", q_scale=None, k_scale=None, v_scale=None, stream=None,
                host=False) -> int:
    """Calls fa_prefill (or fa_prefill_host) and returns its status code unchanged."""
    a = PrefillArgs(_ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(lse), batch_size, num_heads, seq_len,
                    d_head, scale, int(bool(causal)), DTYPES[dtype] if isinstance(dtype, str) else dtype,
                    _ptr(q_scale), _ptr(k_scale), _ptr(v_scale), _stream_handle(stream))
    fn = lib().fa_prefill_host if host else lib().fa_prefill
    return fn(ctypes.byref(a))


def prefill(q, k, v, o, lse, batch_size, num_heads, seq_len, d_head, scale, causal, **kw) -> None:
    """fa_prefill on device buffers; raises FaError on a non-zero status."""
    rc = prefill_raw(q, k, v, o, lse, batch_size, num_heads, seq_len, d_head, scale, causal, **kw)
    if rc != FA_OK:
        raise FaError(rc, "fa_prefill")


PREFILL_VARIANTS = {"auto": 0, "one_tile": 1, "tile_pair": 2, "cta_pair": 3}


def set_prefill_variant(variant: str) -> None:
    """fa_set_prefill_variant: which 16-bit prefill kernel runs ("auto" picks by problem size)."""
    rc = lib().fa_set_prefill_variant(PREFILL_VARIANTS[variant])
    if rc != FA_OK:
        raise FaError(rc, "fa_set_prefill_variant")


def decode_workspace_bytes(batch_size, num_heads, d_head, num_splits) -> int:
    return lib().fa_decode_workspace_bytes(batch_size, num_heads, d_head, num_splits)


def decode_default_splits(batch_size, num_heads, seq_len_kv) -> int:
    return lib().fa_decode_default_splits(batch_size, num_heads, seq_len_kv)


def decode_raw(q, k, v, o, lse, o_f32, batch_size, num_heads, seq_len_kv, d_head, scale,
               dtype="f16", num_splits=0, workspace=None, workspace_bytes=0, stream=None) -> int:
    a = DecodeArgs(_ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(lse), _ptr(o_f32), batch_size, num_heads,
                   seq_len_kv, d_head, scale, DTYPES[dtype] if isinstance(dtype, str) else dtype,
                   num_splits, _ptr(workspace), workspace_bytes, _stream_handle(stream))
    return lib().fa_decode(ctypes.byref(a))


DECODE_STATIC_SCRATCH_BYTES = 8 * 1024 * 1024 + 512 * 1024


def decode_static_raw(q, k, v, o, lse, o_f32, batch_size, num_heads, seq_len_kv, d_head, scale,
                      dtype="f16", num_splits=0, stream=None) -> int:
    """fa_decode_static: decode with the library's built-in scratch array instead of a
    caller workspace (for callers that may not allocate).  Returns the status code."""
    a = DecodeArgs(_ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(lse), _ptr(o_f32), batch_size, num_heads,
                   seq_len_kv, d_head, scale, DTYPES[dtype] if isinstance(dtype, str) else dtype,
                   num_splits, None, 0, _stream_handle(stream))
    return lib().fa_decode_static(ctypes.byref(a))


def decode(*args, **kw) -> None:
    rc = decode_raw(*args, **kw)
    if rc != FA_OK:
        raise FaError(rc, "fa_decode")


def decode_gqa_default_splits(batch_size, num_kv_heads, seq_len_kv) -> int:
    return lib().fa_decode_gqa_default_splits(batch_size, num_kv_heads, seq_len_kv)


def decode_gqa_raw(q, k, v, o, lse, batch_size, num_q_heads, num_kv_heads, seq_len_kv, d_head, scale,
                   dtype="f16", num_splits=0, kv_strides=(0, 0, 0), workspace=None, workspace_bytes=0,
                   stream=None, block_table=None, block_table_stride=0, page_size=0, num_pages=0,
                   kv_page_stride=0, seq_lens=None, q_scale=None, k_scale=None, v_scale=None,
                   num_q_tokens=0) -> int:
    """fa_decode_gqa; ``kv_strides`` = (batch, head, row) strides of the cache in elements
    ((0, 0, 0) = dense [B, Hkv, Skv, D]); ``block_table`` (int32, device) selects the paged
    layout; ``seq_lens`` (int32, device) gives per-sequence lengths.  Returns the status code."""
    a = DecodeGqaArgs(_ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(lse), batch_size, num_q_heads, num_kv_heads,
                      seq_len_kv, d_head, scale, DTYPES[dtype] if isinstance(dtype, str) else dtype,
                      num_splits, kv_strides[0], kv_strides[1], kv_strides[2], _ptr(block_table),
                      block_table_stride, page_size, num_pages, kv_page_stride, _ptr(seq_lens),
                      _ptr(q_scale), _ptr(k_scale), _ptr(v_scale), num_q_tokens,
                      _ptr(workspace), workspace_bytes, _stream_handle(stream))
    return lib().fa_decode_gqa(ctypes.byref(a))


def decode_gqa(*args, **kw) -> None:
    rc = decode_gqa_raw(*args, **kw)
    if rc != FA_OK:
        raise FaError(rc, "fa_decode_gqa")


def backward_workspace_bytes(batch_size, num_heads, seq_len) -> int:
    return lib().fa_backward_workspace_bytes(batch_size, num_heads, seq_len)


def backward_raw(q, k, v, o, d_o, lse, dq, dk, dv, batch_size, num_heads, seq_len, d_head, scale, causal,
                 dtype="f16", workspace=None, workspace_bytes=0, stream=None) -> int:
    """fa_backward on device buffers; returns the status code."""
    a = BackwardArgs(_ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(d_o), _ptr(lse), _ptr(dq), _ptr(dk), _ptr(dv),
                     batch_size, num_heads, seq_len, d_head, scale, int(bool(causal)),
                     DTYPES[dtype] if isinstance(dtype, str) else dtype, _ptr(workspace), workspace_bytes,
                     _stream_handle(stream))
    return lib().fa_backward(ctypes.byref(a))


def backward(*args, **kw) -> None:
    rc = backward_raw(*args, **kw)
    if rc != FA_OK:
        raise FaError(rc, "fa_backward")


def _adr(x) -> int:
    """Address of a tensor, or the address given; 0 for None."""
    if x is None:
        return 0
    return x if x.__class__ is int else x.data_ptr()


def _host_doubles(x, rotary_dim) -> int:
    """Address of the rotary_dim / 2 doubles in host memory that the library reads during the call: a tensor's or a ctypes
    array's, which are checked, or the address given."""
    if x is None:
        return 0
    if x.__class__ is int:
        return x
    try:
        ok = x.is_cpu and x.element_size() == 8 and x.is_floating_point() and x.is_contiguous()
        n, at = x.numel(), x.data_ptr()
    except AttributeError:
        ok = isinstance(x, ctypes.Array) and x._type_ is ctypes.c_double
        n, at = (len(x), ctypes.addressof(x)) if ok else (0, 0)
    if not ok:
        raise TypeError("fa_b200: frequencies are contiguous doubles in host memory (a tensor, a ctypes array or an address)")
    if 2 * n < rotary_dim:
        raise ValueError("fa_b200: fewer frequencies than rotary_dim / 2")
    return at


def rope_inv_freq(rotary_dim, base=10000.0, scaling="plain", factor=1.0, original_length=0.0, slow=0.0, fast=0.0):
    """fa_rope_inv_freq: (ctypes array of rotary_dim / 2 doubles, amplitude).  ``scaling``: "plain", "linear", "base",
    "parts" or "smooth"."""
    sc = RopeScaling(ROPE_SCALINGS[scaling], base, factor, original_length, slow, fast)
    out = (ctypes.c_double * max(1, rotary_dim // 2))()
    amp = ctypes.c_float(1.0)
    rc = lib().fa_rope_inv_freq(ctypes.byref(sc), rotary_dim, out, ctypes.byref(amp))
    if rc != FA_OK:
        raise FaError(rc, "fa_rope_inv_freq")
    return out, amp.value


def rope_raw(q, k, q_out, k_out, batch_size, num_q_heads, num_kv_heads, seq_len, d_head, inv_freq, rotary_dim,
             interleaved=False, amplitude=1.0, dtype="f16", positions=None, positions_stride=0, position_offset=0,
             inverse=False, q_strides=(0, 0, 0), k_strides=(0, 0, 0), q_out_strides=(0, 0, 0), k_out_strides=(0, 0, 0),
             stream=None) -> int:
    """fa_rope; ``inv_freq``: doubles in host memory (a CPU tensor, a ctypes array or an address); strides are (batch, head,
    row) in elements ((0, 0, 0) = dense [B, H, S, D]).  Returns the status code."""
    return (_lib or lib()).fa_rope(_pack_rope(
        _adr(q), _adr(k), _adr(q_out), _adr(k_out), *q_strides, *k_strides, *q_out_strides, *k_out_strides, batch_size,
        num_q_heads, num_kv_heads, seq_len, d_head, DTYPES.get(dtype, dtype), _adr(positions), positions_stride,
        position_offset, inverse, _host_doubles(inv_freq, rotary_dim), rotary_dim, interleaved, amplitude, _stream_handle(stream) or 0))


def rope(*args, **kw) -> None:
    rc = rope_raw(*args, **kw)
    if rc != FA_OK:
        raise FaError(rc, "fa_rope")


def cache_append_raw(k, v, k_cache, v_cache, batch_size, num_tokens, num_kv_heads, seq_len_kv, d_head, dtype="f16",
                     cache_dtype=None, kv_strides=(0, 0, 0), q=None, q_out=None, num_q_heads=0,
                     token_strides=(0, 0, 0), k_params=None, v_params=None, param_strides=(0, 0, 0), block_table=None,
                     block_table_stride=0, page_size=0, num_pages=0, seq_lens=None, num_new=None, positions=None,
                     inv_freq=None, rotary_dim=0, interleaved=False, amplitude=1.0, q_scale=None, k_scale=None,
                     v_scale=None, stream=None) -> int:
    """fa_cache_append; ``cache_dtype`` is that of q, k and v (also if None), "e4m3" or "u4"; ``kv_strides`` and ``param_strides`` are
    (block, head, row) strides of the cache, a block being a page or a whole sequence; ``token_strides`` those between
    the tokens of q, k, v.  Returns the status code."""
    if cache_dtype is None:
        cache_dtype = FA_CACHE_16BIT
    elif cache_dtype in ("f16", "bf16") and DTYPES[cache_dtype] != DTYPES.get(dtype, dtype):
        return FA_ERR_UNSUPPORTED
    return (_lib or lib()).fa_cache_append(_pack_append(
        _adr(q), _adr(k), _adr(v), _adr(q_out), _adr(k_cache), _adr(v_cache), _adr(k_params), _adr(v_params),
        *token_strides, batch_size, num_tokens, num_q_heads, num_kv_heads, seq_len_kv, d_head, DTYPES.get(dtype, dtype),
        CACHES.get(cache_dtype, cache_dtype), *kv_strides, *param_strides, _adr(block_table), block_table_stride, page_size,
        num_pages, _adr(seq_lens), _adr(num_new), _adr(positions), _host_doubles(inv_freq, rotary_dim), rotary_dim, interleaved, amplitude,
        _adr(q_scale), _adr(k_scale), _adr(v_scale), _stream_handle(stream) or 0))


def cache_append(*args, **kw) -> None:
    rc = cache_append_raw(*args, **kw)
    if rc != FA_OK:
        raise FaError(rc, "fa_cache_append")


def cache_read_u4_raw(k_cache, k_params, v_cache, v_params, k_out, v_out, batch_size, num_kv_heads, seq_len_kv, d_head,
                      num_rows, dtype="f16", first_rows=None, kv_strides=(0, 0, 0), param_strides=(0, 0, 0),
                      block_table=None, block_table_stride=0, page_size=0, num_pages=0, seq_lens=None, stream=None) -> int:
    """fa_cache_read_u4; the cache is described as for cache_append.  Returns the status code."""
    return (_lib or lib()).fa_cache_read_u4(_pack_read(
        _adr(k_cache), _adr(k_params), _adr(v_cache), _adr(v_params), _adr(k_out), _adr(v_out), batch_size, num_kv_heads,
        seq_len_kv, d_head, num_rows, DTYPES.get(dtype, dtype), *kv_strides, *param_strides, _adr(block_table),
        block_table_stride, page_size, num_pages, _adr(seq_lens), _adr(first_rows), _stream_handle(stream) or 0))


def cache_read_u4(*args, **kw) -> None:
    rc = cache_read_u4_raw(*args, **kw)
    if rc != FA_OK:
        raise FaError(rc, "fa_cache_read_u4")


def decode_gqa_u4_workspace_bytes(batch_size, num_q_heads, num_kv_heads, num_q_tokens, seq_len_kv, d_head) -> int:
    return lib().fa_decode_gqa_u4_workspace_bytes(batch_size, num_q_heads, num_kv_heads, num_q_tokens, seq_len_kv, d_head)


def decode_gqa_u4_raw(q, k_cache, k_params, v_cache, v_params, o, lse, batch_size, num_q_heads, num_kv_heads, seq_len_kv,
                      d_head, scale, dtype="f16", num_q_tokens=0, kv_strides=(0, 0, 0), param_strides=(0, 0, 0),
                      block_table=None, block_table_stride=0, page_size=0, num_pages=0, seq_lens=None, workspace=None,
                      workspace_bytes=0, stream=None) -> int:
    """fa_decode_gqa_u4; the cache is described as for cache_append.  Returns the status code."""
    return (_lib or lib()).fa_decode_gqa_u4(_pack_decode_u4(
        _adr(q), _adr(k_cache), _adr(k_params), _adr(v_cache), _adr(v_params), _adr(o), _adr(lse), batch_size, num_q_heads,
        num_kv_heads, num_q_tokens, seq_len_kv, d_head, scale, DTYPES.get(dtype, dtype), *kv_strides, *param_strides,
        _adr(block_table), block_table_stride, page_size, num_pages, _adr(seq_lens), _adr(workspace), workspace_bytes,
        _stream_handle(stream) or 0))


def decode_gqa_u4(*args, **kw) -> None:
    rc = decode_gqa_u4_raw(*args, **kw)
    if rc != FA_OK:
        raise FaError(rc, "fa_decode_gqa_u4")


def combine(o_parts, lse_parts, n_parts, rows, d_head, o, lse, dtype="f16", stream=None) -> None:
    rc = lib().fa_combine(_ptr(o_parts), _ptr(lse_parts), n_parts, rows, d_head, _ptr(o), _ptr(lse),
                          DTYPES[dtype] if isinstance(dtype, str) else dtype, _stream_handle(stream))
    if rc != FA_OK:
        raise FaError(rc, "fa_combine")


def combine_packed(packed_parts, n_parts, rows, d_head, o, lse, dtype="f16", stream=None) -> None:
    """fa_combine_packed: LSE merge of [n_parts, rows, d_head + 1] fp32 partials (O then LSE per row)."""
    rc = lib().fa_combine_packed(_ptr(packed_parts), n_parts, rows, d_head, _ptr(o), _ptr(lse),
                                 DTYPES[dtype] if isinstance(dtype, str) else dtype, _stream_handle(stream))
    if rc != FA_OK:
        raise FaError(rc, "fa_combine_packed")


NCCL_UNIQUE_ID_BYTES = 128


def nccl_unique_id() -> bytes:
    """fa_nccl_unique_id: a fresh NCCL id (rank 0 creates it, every rank passes it to nccl_comm_create)."""
    buf = ctypes.create_string_buffer(NCCL_UNIQUE_ID_BYTES)
    rc = lib().fa_nccl_unique_id(buf, NCCL_UNIQUE_ID_BYTES)
    if rc != FA_OK:
        raise FaError(rc, "fa_nccl_unique_id")
    return buf.raw


def nccl_comm_create(n_ranks: int, unique_id: bytes, rank: int) -> int:
    """fa_nccl_comm_create: an ncclComm_t (as an integer handle) for the current device."""
    comm = ctypes.c_void_p()
    buf = ctypes.create_string_buffer(unique_id, NCCL_UNIQUE_ID_BYTES)
    rc = lib().fa_nccl_comm_create(ctypes.byref(comm), n_ranks, buf, NCCL_UNIQUE_ID_BYTES, rank)
    if rc != FA_OK:
        raise FaError(rc, "fa_nccl_comm_create")
    return comm.value


def nccl_comm_destroy(comm: int) -> None:
    rc = lib().fa_nccl_comm_destroy(comm)
    if rc != FA_OK:
        raise FaError(rc, "fa_nccl_comm_destroy")


def decode_kv_sharded_gather_bytes(batch_size, num_heads, d_head, n_ranks) -> int:
    return lib().fa_decode_kv_sharded_gather_bytes(batch_size, num_heads, d_head, n_ranks)


def decode_kv_sharded_raw(q, k, v, o, lse, batch_size, num_heads, local_kv, d_head, scale, comm, gather,
                          gather_bytes, dtype="f16", num_splits=0, workspace=None, workspace_bytes=0,
                          stream=None) -> int:
    """fa_decode_kv_sharded on this rank's key slice; returns the status code."""
    a = DecodeArgs(_ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(lse), None, batch_size, num_heads, local_kv,
                   d_head, scale, DTYPES[dtype] if isinstance(dtype, str) else dtype, num_splits,
                   _ptr(workspace), workspace_bytes, _stream_handle(stream))
    return lib().fa_decode_kv_sharded(ctypes.byref(a), comm, _ptr(gather), gather_bytes)


def kat(dtype: str, d_head: int, q, k, v, p_scale: float):
    """Tensor-core known-answer test.  q,k,v: numpy uint16 arrays [128,d_head] holding
    fp16/bf16 bit patterns.  Returns (S [128,128], O [128,d_head]) float32."""
    import numpy as np
    s = np.zeros((128, 128), np.float32)
    o = np.zeros((128, d_head), np.float32)
    rc = lib().fa_kat(DTYPES[dtype], d_head, q.ctypes.data, k.ctypes.data, v.ctypes.data,
                      p_scale, s.ctypes.data, o.ctypes.data)
    if rc != FA_OK:
        raise FaError(rc, "fa_kat")
    return s, o


def device_status() -> int:
    """Status word of the current device (0 = clean).  Synchronises."""
    w = ctypes.c_int(0)
    rc = lib().fa_device_status(ctypes.byref(w))
    if rc not in (FA_OK, FA_ERR_DEVICE_TIMEOUT):
        raise FaError(rc, "fa_device_status")
    return w.value


def clear_device_status() -> None:
    rc = lib().fa_clear_device_status()
    if rc != FA_OK:
        raise FaError(rc, "fa_clear_device_status")
