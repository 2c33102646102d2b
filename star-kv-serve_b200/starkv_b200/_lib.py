"""ctypes binding of the C ABI in ``include/starkv_b200.h``.

This module is the only place Python touches the native library. There is no
fallback: if the library is missing or fails to load, every operator raises.
The struct layouts below mirror the header field for field; ``check_abi()``
compares their sizes with the library's own ``starkv_abi_sizeof``.
"""
from __future__ import annotations

import ctypes as C
import os
import struct

import torch

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_lib", "libstarkv_b200.so")

F16, BF16, F32, U8, I32, I64 = 0, 1, 2, 3, 4, 5
_DTYPES = {torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32, torch.uint8: U8,
           torch.int32: I32, torch.int64: I64}

STATUS = {
    0: "ok", 22: "EINVAL", 100: "EALIGN", 101: "EDTYPE", 102: "EWORKSPACE", 103: "ECUDA",
    104: "ENODEV", 105: "EBOUNDS", 106: "ETIMEOUT",
}

p, i32, i64, f32 = C.c_void_p, C.c_int32, C.c_int64, C.c_float


class DecodeArgs(C.Structure):
    _fields_ = [
        ("query", p), ("q_stride", i64 * 3), ("q_dtype", i32),
        ("kv_cache", p), ("cache_stride", i64 * 3), ("cache_dtype", i32),
        ("num_blocks", i32), ("block_size", i32),
        ("block_table", p), ("bt_stride", i64 * 2), ("max_blocks", i32),
        ("seq_lens", p),
        ("n", i32), ("num_heads", i32), ("num_kv_heads", i32), ("head_dim", i32),
        ("max_seq_len", i32),
        ("k_up", p), ("k_up_stride", i64 * 2), ("k_up_dtype", i32),
        ("k_ranks", p), ("k_head_offsets", p),
        ("k_width", i32),
        ("v_up_by_q", p), ("v_up_stride", i64 * 3), ("v_up_dtype", i32),
        ("v_rank", i32),
        ("cos_sin_cache", p), ("cs_stride", i64 * 2), ("cs_dtype", i32), ("cs_rows", i32),
        ("scale", f32),
        ("out", p), ("out_stride", i64 * 3), ("out_dtype", i32),
        ("row_nbytes", i32), ("ks_off", i32), ("vs_off", i32), ("vq_off", i32),
        ("v_nout", i32), ("v_nbo", i32), ("v_bytes", i32),
        ("head_of_lane", p),
        ("tile_head", p), ("tile_nout", p), ("tile_last", p),
    ]


class PackArgs(C.Structure):
    _fields_ = [
        ("k_codes", p), ("k_stride0", i64), ("k_dtype", i32),
        ("v_codes", p), ("v_stride0", i64), ("v_dtype", i32),
        ("cache", p), ("cache_stride", i64 * 2),
        ("num_blocks", i32), ("block_size", i32),
        ("slot_mapping", p), ("slot_dtype", i32),
        ("n", i32), ("num_kv_heads", i32), ("k_width", i32), ("v_rank", i32),
        ("k_ranks", p), ("k_offsets", p), ("k_nouts", p),
        ("ks_off", i32), ("vs_off", i32), ("vq_off", i32), ("v_nout", i32), ("v_nbo", i32), ("v_bytes", i32),
        ("status", p),
    ]


class CacheWriteArgs(C.Structure):
    _fields_ = [
        ("key", p), ("key_stride0", i64), ("key_dtype", i32),
        ("value", p), ("value_stride0", i64), ("value_dtype", i32),
        ("cache", p), ("cache_stride", i64 * 3), ("cache_dtype", i32),
        ("num_blocks", i32), ("block_size", i32),
        ("slot_mapping", p), ("slot_dtype", i32),
        ("n", i32), ("k_width", i32), ("v_rank", i32),
        ("status", p),
    ]


class PagedAttnArgs(C.Structure):
    _fields_ = [
        ("query", p), ("q_stride", i64 * 2), ("k_cache", p), ("k_stride", i64 * 3), ("v_cache", p),
        ("v_stride", i64 * 3), ("block_table", p), ("bt_stride", i64 * 2), ("seq_lens", p),
        ("pages", p), ("pages_stride", i64 * 2), ("out", p), ("out_stride", i64 * 2),
        ("m_out", p), ("l_out", p), ("status", p),
        ("dtype", i32), ("n", i32), ("num_heads", i32), ("num_kv_heads", i32), ("head_dim", i32),
        ("num_blocks", i32), ("block_size", i32), ("max_blocks", i32), ("max_seq_len", i32), ("top", i32),
        ("scale", f32),
    ]


class PageBoundsArgs(C.Structure):
    _fields_ = [
        ("k_cache", p), ("k_stride", i64 * 3), ("bounds", p), ("bounds_stride", i64 * 2),
        ("block_table", p), ("bt_stride", i64 * 2), ("seq_lens", p), ("new_lens", p), ("status", p),
        ("dtype", i32), ("n", i32), ("num_kv_heads", i32), ("head_dim", i32),
        ("num_blocks", i32), ("block_size", i32), ("max_blocks", i32), ("max_seq_len", i32), ("max_new", i32),
    ]


class SelectPagesArgs(C.Structure):
    _fields_ = [
        ("query", p), ("q_stride", i64 * 2), ("bounds", p), ("bounds_stride", i64 * 2),
        ("block_table", p), ("bt_stride", i64 * 2), ("seq_lens", p), ("pages", p), ("pages_stride", i64 * 2),
        ("status", p),
        ("dtype", i32), ("n", i32), ("num_heads", i32), ("num_kv_heads", i32), ("head_dim", i32),
        ("num_blocks", i32), ("block_size", i32), ("max_blocks", i32), ("max_seq_len", i32),
        ("top", i32), ("sinks", i32), ("recent", i32),
    ]


class NormRopeArgs(C.Structure):
    _fields_ = [
        ("query", p), ("q_stride", i64 * 2), ("key", p), ("k_stride", i64 * 2), ("value", p), ("v_stride", i64 * 2),
        ("q_out", p), ("qo_stride", i64 * 2), ("k_out", p), ("ko_stride", i64 * 2),
        ("q_weight", p), ("k_weight", p), ("positions", p), ("cos_sin", p), ("cs_stride0", i64),
        ("k_cache", p), ("kc_stride", i64 * 3), ("v_cache", p), ("vc_stride", i64 * 3),
        ("slot_mapping", p), ("status", p),
        ("dtype", i32), ("w_dtype", i32), ("pos_dtype", i32), ("cs_dtype", i32), ("slot_dtype", i32),
        ("n", i32), ("num_heads", i32), ("num_kv_heads", i32), ("head_dim", i32), ("rot", i32), ("cs_rows", i32),
        ("num_blocks", i32), ("block_size", i32), ("eps", f32),
    ]


def _packed(cls):
    """``pack(*values)`` -> the bytes of an argument struct, array members flattened. The
    operators of the full-rank paged cache are short enough on the GPU for the filling of
    a ctypes structure (about 15 us) to show; one struct.pack takes 2."""
    fmt = ""
    for _, t in cls._fields_:
        n, t = (t._length_, t._type_) if issubclass(t, C.Array) else (1, t)
        fmt += f"{n}{ {p: 'Q', i64: 'q', i32: 'i', f32: 'f'}[t] }"
    pad = C.sizeof(cls) - struct.calcsize("@" + fmt)
    return struct.Struct(f"@{fmt}{pad}x").pack


pack_paged_attn, pack_page_bounds = _packed(PagedAttnArgs), _packed(PageBoundsArgs)
pack_select_pages, pack_norm_rope = _packed(SelectPagesArgs), _packed(NormRopeArgs)

EXPORTS = {
    "starkv_decode_workspace_bytes": (C.c_size_t, [i32, i32, i32, i32, i32, i32]),
    "starkv_paged_decode_bf16": (C.c_int, [C.POINTER(DecodeArgs), p, C.c_size_t, p]),
    "starkv_paged_decode_q32": (C.c_int, [C.POINTER(DecodeArgs), p, C.c_size_t, p]),
    "starkv_paged_decode_bf16_noalloc": (C.c_int, [C.POINTER(DecodeArgs), p]),
    "starkv_noalloc_read_status": (C.c_int, [C.POINTER(i32), i32, p]),
    "starkv_paged_decode_bf16_partial": (C.c_int, [C.POINTER(DecodeArgs), i32, i32, p, p, p, C.c_size_t, p]),
    "starkv_paged_decode_q32_partial": (C.c_int, [C.POINTER(DecodeArgs), i32, i32, p, p, p, C.c_size_t, p]),
    "starkv_cp_combine": (C.c_int, [p, i32, i32, i32, p, C.POINTER(i64), i32, p]),
    "starkv_selftest_wait_timeout": (C.c_int, [p, p]),
    "starkv_fold_q": (C.c_int, [p, C.POINTER(i64), i32, p, C.POINTER(i64), i32, p, i32, i32, i32, f32, p, p, p]),
    "starkv_pack_kv_q32": (C.c_int, [C.POINTER(PackArgs), p]),
    "starkv_kv_down_cache_write": (C.c_int, [p, i64, p, i64, i32, i32, i32, i32, p, C.POINTER(i64), i32, i32, p, i32,
                                             p, p]),
    "starkv_prefill_attention": (C.c_int, [p, C.POINTER(i64), p, C.POINTER(i64), p, C.POINTER(i64), i32, i32, i32, i32,
                                           i32, p, i32, i32, f32, p, C.POINTER(i64), p, p]),
    "starkv_paged_attention_workspace_bytes": (C.c_size_t, [i32, i32, i32, i32]),
    "starkv_paged_attention": (C.c_int, [C.c_char_p, p, C.c_size_t, p]),
    "starkv_page_bounds": (C.c_int, [C.c_char_p, p]),
    "starkv_select_pages_workspace_bytes": (C.c_size_t, [i32, i32, i32, i32, i32]),
    "starkv_select_pages": (C.c_int, [C.c_char_p, p, C.c_size_t, p]),
    "starkv_selftest_select_timeout": (C.c_int, [C.c_char_p, p, C.c_size_t, p]),
    "starkv_sparse_paged_attention": (C.c_int, [C.c_char_p, p, i64, i64, i32, i32, p, C.c_size_t, p]),
    "starkv_norm_rope": (C.c_int, [C.c_char_p, p]),
    "starkv_cache_write_bf16": (C.c_int, [C.POINTER(CacheWriteArgs), p]),
    "starkv_read_status": (C.c_int, [p, C.POINTER(i32), i32, p]),
    "starkv_status_offset": (C.c_size_t, []),
    "starkv_abi_sizeof": (C.c_size_t, [i32]),
    "starkv_profile_begin": (C.c_int, [i32]),
    "starkv_profile_end": (C.c_int, [C.POINTER(f32), C.POINTER(i32)]),
    "starkv_version": (C.c_char_p, []),
    "starkv_strerror": (C.c_char_p, [C.c_int]),
}

_lib = None


def lib() -> C.CDLL:
    """Load the native library once; raise if it is not built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"starkv_b200 native library not built: {LIB_PATH} "
                               "(run python star-kv-serve_b200/build.py)")
        h = C.CDLL(LIB_PATH)
        for name, (res, args) in EXPORTS.items():
            fn = getattr(h, name)
            fn.restype = res
            fn.argtypes = args
        _lib = h
    return _lib


def check_abi() -> None:
    L = lib()
    for which, cls in enumerate((DecodeArgs, PackArgs, CacheWriteArgs, PagedAttnArgs, PageBoundsArgs,
                                 SelectPagesArgs, NormRopeArgs)):
        got = L.starkv_abi_sizeof(which)
        if got != C.sizeof(cls):
            raise RuntimeError(f"ABI mismatch for {cls.__name__}: library {got} B, binding {C.sizeof(cls)} B")


def check(status: int, what: str) -> None:
    if status != 0:
        msg = lib().starkv_strerror(status).decode()
        if status in (22, 101):
            raise ValueError(f"{what}: {msg} ({STATUS.get(status, status)})")
        raise RuntimeError(f"{what}: {msg} ({STATUS.get(status, status)})")


def dtype_code(t: torch.Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise ValueError(f"unsupported dtype {t.dtype}") from None


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def addr(t: torch.Tensor | None) -> int:
    """Address for the pack_* functions, which take 0 for a null pointer."""
    return 0 if t is None else t.data_ptr()


def refuse_status(what: str, status: torch.Tensor | None) -> None:
    """The error for a status tensor that does not hold one aligned int32."""
    if status is not None and (status.nbytes < 4 or status.data_ptr() & 3):
        raise ValueError(f"{what}: status must hold an int32")


def stream_ptr(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def same_device(what: str, first: torch.Tensor, *rest) -> int:
    """Index of the CUDA device that all tensors (None: left out) are on; ValueError otherwise."""
    idx = first.get_device()
    for t in rest:
        if t is not None and t.get_device() != idx:
            idx = -1
            break
    if idx < 0:
        raise ValueError(f"{what}: all tensors must be on one CUDA device")
    return idx


def launch(what: str, idx: int, fn, *args) -> None:
    """``fn(*args, stream)`` on the current stream of device `idx`, whichever device is current."""
    if idx == torch._C._cuda_getDevice():
        st = fn(*args, torch._C._cuda_getCurrentRawStream(idx))
    else:
        with torch.cuda.device(idx):
            st = fn(*args, torch._C._cuda_getCurrentRawStream(idx))
    if st:
        check(st, what)


def i64s(values):
    arr = (i64 * len(values))(*[int(v) for v in values])
    return arr
