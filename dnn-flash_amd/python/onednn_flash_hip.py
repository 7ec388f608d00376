"""Python binding of the MI355X attention forward library over its C ABI
(include/onednn_flash_hip.h), loaded with ctypes from
dnn-flash_amd/lib/libonednn_flash_hip.so.

Device memory and streams come from PyTorch tensors (torch is plumbing here:
the computation is the library's HIP kernels). There is no fallback: if the
shared library is missing, loading raises.

Python-side counterpart of the reference's TensorFlow wrapper
(python/onednn_flash_tf/ops.py:63-115): `onednn_flash_attention(q, k, v, ...)`
with the same keyword names and validation, on device tensors.
"""

from __future__ import annotations

import contextlib
import ctypes
import math
import operator
import struct
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parents[1]
LIB_PATH = PKG_DIR / "lib" / "libonednn_flash_hip.so"

OFH_SUCCESS = 0
OFH_ERROR_INVALID_ARGUMENT = 1
OFH_ERROR_UNSUPPORTED = 2
OFH_ERROR_HIP = 3
OFH_ERROR_WORKSPACE_TOO_SMALL = 4
OFH_ERROR_OUT_OF_PAGES = 5

DTYPE_F32, DTYPE_BF16, DTYPE_F16 = 0, 1, 2
BIAS_NONE, BIAS_ALIBI, BIAS_DENSE = 0, 1, 2
ALGO_AUTO, ALGO_FLASH_MFMA, ALGO_ROWWISE = 0, 1, 2
QK_AUTO, QK_EXACT, QK_MFMA = 0, 1, 2

# Every function the C header declares; tests check the library exports each.
EXPORTED_SYMBOLS = (
    "ofh_attention_params_init",
    "ofh_attention_workspace_bytes",
    "ofh_attention_fwd",
    "ofh_attention_fwd_noalloc",
    "ofh_attention_fwd_host",
    "ofh_attention_launch_info",
    "ofh_attention_useful_flops",
    "ofh_qk_score_params_init",
    "ofh_qk_score_tile",
    "ofh_window_params_init",
    "ofh_window_attention_workspace_bytes",
    "ofh_window_attention_fwd",
    "ofh_paged_params_init",
    "ofh_paged_attention_workspace_bytes",
    "ofh_paged_attention_fwd",
    "ofh_cache_write_params_init",
    "ofh_cache_write",
    "ofh_prefix_groups_init",
    "ofh_shared_prefix_workspace_bytes",
    "ofh_shared_prefix_attention_fwd",
    "ofh_selected_attention_workspace_bytes",
    "ofh_selected_attention_fwd",
    "ofh_page_bounds_params_init",
    "ofh_page_bounds",
    "ofh_select_params_init",
    "ofh_select_pages_workspace_bytes",
    "ofh_select_pages",
    "ofh_rotary_params_init",
    "ofh_rotary_fwd",
    "ofh_cache_append_params_init",
    "ofh_cache_append",
    "ofh_cache_copy_pages",
    "ofh_page_pool_create",
    "ofh_page_pool_destroy",
    "ofh_page_pool_add",
    "ofh_page_pool_extend",
    "ofh_page_pool_fork",
    "ofh_page_pool_truncate",
    "ofh_page_pool_free",
    "ofh_page_pool_compact",
    "ofh_page_pool_table",
    "ofh_page_pool_length",
    "ofh_page_pool_info",
    "ofh_last_error",
    "ofh_abi_version",
)


class AttentionParams(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("batch", ctypes.c_size_t),
        ("heads", ctypes.c_size_t),
        ("query_tokens", ctypes.c_size_t),
        ("key_tokens", ctypes.c_size_t),
        ("head_dim", ctypes.c_size_t),
        ("value_dim", ctypes.c_size_t),
        ("dtype", ctypes.c_int32),
        ("out_dtype", ctypes.c_int32),
        ("q_strides", ctypes.c_int64 * 3),
        ("k_strides", ctypes.c_int64 * 3),
        ("v_strides", ctypes.c_int64 * 3),
        ("o_strides", ctypes.c_int64 * 3),
        ("scale", ctypes.c_float),
        ("causal", ctypes.c_int32),
        ("mask_allowed", ctypes.c_void_p),
        ("mask_query_block_size", ctypes.c_size_t),
        ("mask_key_block_size", ctypes.c_size_t),
        ("mask_query_blocks", ctypes.c_size_t),
        ("mask_key_blocks", ctypes.c_size_t),
        ("bias_kind", ctypes.c_int32),
        ("alibi_slopes", ctypes.c_void_p),
        ("bias", ctypes.c_void_p),
        ("bias_strides", ctypes.c_int64 * 3),
        ("softcap", ctypes.c_float),
        ("algorithm", ctypes.c_int32),
        ("max_key_splits", ctypes.c_int32),
    ]


def _flat_fields(fields):
    """The fields with their arrays taken apart: the same layout, for one positional
    construction instead of an assignment per field and array element."""
    flat = []
    for name, t in fields:
        if isinstance(t, type) and issubclass(t, ctypes.Array):
            flat += [(f"{name}{i}", t._type_) for i in range(t._length_)]
        else:
            flat.append((name, t))
    return flat


class _FlatAttentionParams(ctypes.Structure):
    _fields_ = _flat_fields(AttentionParams._fields_)


assert ctypes.sizeof(_FlatAttentionParams) == ctypes.sizeof(AttentionParams)


class LaunchInfo(ctypes.Structure):
    _fields_ = [
        ("algorithm", ctypes.c_int32),
        ("block_m", ctypes.c_int32),
        ("block_n", ctypes.c_int32),
        ("threads", ctypes.c_int32),
        ("workgroups", ctypes.c_int64),
        ("uses_tile_list", ctypes.c_int32),
        ("key_splits", ctypes.c_int32),
        ("kernel_name", ctypes.c_char * 96),
        ("merge_in_launch", ctypes.c_int32),
    ]


class QkScoreParams(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("batch", ctypes.c_int64),
        ("m", ctypes.c_int64),
        ("n", ctypes.c_int64),
        ("k", ctypes.c_int64),
        ("a_stride_m", ctypes.c_int64),
        ("a_stride_k", ctypes.c_int64),
        ("a_stride_batch", ctypes.c_int64),
        ("b_stride_k", ctypes.c_int64),
        ("b_stride_n", ctypes.c_int64),
        ("b_stride_batch", ctypes.c_int64),
        ("c_stride_m", ctypes.c_int64),
        ("c_stride_n", ctypes.c_int64),
        ("c_stride_batch", ctypes.c_int64),
        ("dtype", ctypes.c_int32),
        ("has_scale", ctypes.c_int32),
        ("scale", ctypes.c_float),
        ("bias", ctypes.c_void_p),
        ("bias_stride_m", ctypes.c_int64),
        ("bias_stride_n", ctypes.c_int64),
        ("bias_stride_batch", ctypes.c_int64),
        ("softcap", ctypes.c_float),
        ("algorithm", ctypes.c_int32),
    ]


class WindowParams(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("batch", ctypes.c_size_t),
        ("heads", ctypes.c_size_t),
        ("kv_heads", ctypes.c_size_t),
        ("query_tokens", ctypes.c_size_t),
        ("key_tokens", ctypes.c_size_t),
        ("head_dim", ctypes.c_size_t),
        ("value_dim", ctypes.c_size_t),
        ("dtype", ctypes.c_int32),
        ("out_dtype", ctypes.c_int32),
        ("q_strides", ctypes.c_int64 * 3),
        ("k_strides", ctypes.c_int64 * 3),
        ("v_strides", ctypes.c_int64 * 3),
        ("o_strides", ctypes.c_int64 * 3),
        ("scale", ctypes.c_float),
        ("softcap", ctypes.c_float),
        ("alibi_slopes", ctypes.c_void_p),
        ("window", ctypes.c_size_t),
        ("sink_tokens", ctypes.c_size_t),
        ("query_offset", ctypes.c_size_t),
        ("lengths", ctypes.c_void_p),
        ("max_key_splits", ctypes.c_int32),
    ]


# WindowParams as one pack of its fields: a quarter of a Structure's construction
_pack_window = struct.Struct("@I7Q2i12q2f5Qi0Q")
assert _pack_window.size == ctypes.sizeof(WindowParams)


class PagedParams(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("batch", ctypes.c_size_t),
        ("heads", ctypes.c_size_t),
        ("kv_heads", ctypes.c_size_t),
        ("query_tokens", ctypes.c_size_t),
        ("head_dim", ctypes.c_size_t),
        ("value_dim", ctypes.c_size_t),
        ("num_pages", ctypes.c_size_t),
        ("page_size", ctypes.c_size_t),
        ("max_pages", ctypes.c_size_t),
        ("table_stride", ctypes.c_int64),
        ("dtype", ctypes.c_int32),
        ("out_dtype", ctypes.c_int32),
        ("q_strides", ctypes.c_int64 * 3),
        ("o_strides", ctypes.c_int64 * 3),
        ("k_strides", ctypes.c_int64 * 3),
        ("v_strides", ctypes.c_int64 * 3),
        ("page_table", ctypes.c_void_p),
        ("lengths", ctypes.c_void_p),
        ("scale", ctypes.c_float),
        ("softcap", ctypes.c_float),
        ("alibi_slopes", ctypes.c_void_p),
        ("window", ctypes.c_size_t),
        ("sink_tokens", ctypes.c_size_t),
        ("max_key_splits", ctypes.c_int32),
    ]


class CacheWriteParams(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("batch", ctypes.c_size_t),
        ("kv_heads", ctypes.c_size_t),
        ("tokens", ctypes.c_size_t),
        ("head_dim", ctypes.c_size_t),
        ("value_dim", ctypes.c_size_t),
        ("num_pages", ctypes.c_size_t),
        ("page_size", ctypes.c_size_t),
        ("max_pages", ctypes.c_size_t),
        ("table_stride", ctypes.c_int64),
        ("dtype", ctypes.c_int32),
        ("k_strides", ctypes.c_int64 * 3),
        ("v_strides", ctypes.c_int64 * 3),
        ("k_page_strides", ctypes.c_int64 * 3),
        ("v_page_strides", ctypes.c_int64 * 3),
        ("page_table", ctypes.c_void_p),
        ("lengths", ctypes.c_void_p),
        ("counts", ctypes.c_void_p),
    ]


class PrefixGroupsParams(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("groups", ctypes.c_size_t),
        ("starts", ctypes.c_void_p),
        ("shared_tokens", ctypes.c_void_p),
        ("least_shared", ctypes.c_size_t),
        ("most_shared", ctypes.c_size_t),
        ("most_sequences", ctypes.c_size_t),
        ("sharing_groups", ctypes.c_size_t),
        ("sharing_sequences", ctypes.c_size_t),
    ]


class PageBoundsParams(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("batch", ctypes.c_size_t),
        ("kv_heads", ctypes.c_size_t),
        ("tokens", ctypes.c_size_t),
        ("head_dim", ctypes.c_size_t),
        ("num_pages", ctypes.c_size_t),
        ("page_size", ctypes.c_size_t),
        ("max_pages", ctypes.c_size_t),
        ("table_stride", ctypes.c_int64),
        ("dtype", ctypes.c_int32),
        ("k_page_strides", ctypes.c_int64 * 3),
        ("bounds_strides", ctypes.c_int64 * 3),
        ("page_table", ctypes.c_void_p),
        ("lengths", ctypes.c_void_p),
        ("counts", ctypes.c_void_p),
    ]


class SelectParams(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("batch", ctypes.c_size_t),
        ("heads", ctypes.c_size_t),
        ("kv_heads", ctypes.c_size_t),
        ("query_tokens", ctypes.c_size_t),
        ("head_dim", ctypes.c_size_t),
        ("num_pages", ctypes.c_size_t),
        ("page_size", ctypes.c_size_t),
        ("max_pages", ctypes.c_size_t),
        ("table_stride", ctypes.c_int64),
        ("dtype", ctypes.c_int32),
        ("negative", ctypes.c_int32),
        ("q_strides", ctypes.c_int64 * 3),
        ("bounds_strides", ctypes.c_int64 * 3),
        ("page_table", ctypes.c_void_p),
        ("lengths", ctypes.c_void_p),
        ("pages", ctypes.c_size_t),
        ("first_pages", ctypes.c_size_t),
        ("recent_pages", ctypes.c_size_t),
    ]


class RotaryFields(ctypes.Structure):
    _fields_ = [
        ("frequencies", ctypes.c_void_p),
        ("rotary_dim", ctypes.c_size_t),
        ("interleaved", ctypes.c_int32),
        ("magnitude", ctypes.c_float),
    ]


class RotaryParams(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("batch", ctypes.c_size_t),
        ("heads", ctypes.c_size_t),
        ("tokens", ctypes.c_size_t),
        ("head_dim", ctypes.c_size_t),
        ("dtype", ctypes.c_int32),
        ("transpose", ctypes.c_int32),
        ("x_strides", ctypes.c_int64 * 3),
        ("o_strides", ctypes.c_int64 * 3),
        ("rotary", RotaryFields),
        ("positions", ctypes.c_void_p),
        ("position_stride", ctypes.c_int64),
        ("lengths", ctypes.c_void_p),
        ("offset", ctypes.c_int64),
    ]


class CacheAppendParams(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("cache", CacheWriteParams),
        ("rotary", RotaryFields),
        ("heads", ctypes.c_size_t),
        ("q_strides", ctypes.c_int64 * 3),
        ("o_strides", ctypes.c_int64 * 3),
    ]


class OfhError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(f"[ofh status {code}] {message}")
        self.code = code


_lib = None


def lib() -> ctypes.CDLL:
    """Loads the shared library (raises if it was not built)."""
    global _lib
    if _lib is None:
        # torch links its own copy of the HIP runtime under another file name;
        # loaded after this library it would start a second runtime in the
        # process, and this library's would then see no device. Importing
        # torch first makes the library bind the runtime torch already loaded.
        try:
            import torch  # noqa: F401, PLC0415
        except ImportError:
            pass
        if not LIB_PATH.exists():
            raise FileNotFoundError(
                f"{LIB_PATH} is missing: build it with `make -C dnn-flash_amd` "
                "(or __graft_entry__.build())")
        L = ctypes.CDLL(str(LIB_PATH))
        P = ctypes.POINTER(AttentionParams)
        L.ofh_attention_params_init.argtypes = [P]
        L.ofh_attention_params_init.restype = None
        L.ofh_attention_workspace_bytes.argtypes = [P, ctypes.POINTER(ctypes.c_size_t)]
        L.ofh_attention_fwd.argtypes = [P] + [ctypes.c_void_p] * 5 + [ctypes.c_size_t, ctypes.c_void_p]
        L.ofh_attention_fwd_noalloc.argtypes = [P] + [ctypes.c_void_p] * 5
        L.ofh_attention_fwd_host.argtypes = [P] + [ctypes.c_void_p] * 4
        L.ofh_attention_launch_info.argtypes = [P, ctypes.POINTER(LaunchInfo)]
        L.ofh_attention_useful_flops.argtypes = [P, ctypes.POINTER(ctypes.c_double)]
        QP = ctypes.POINTER(QkScoreParams)
        L.ofh_qk_score_params_init.argtypes = [QP]
        L.ofh_qk_score_params_init.restype = None
        L.ofh_qk_score_tile.argtypes = [QP] + [ctypes.c_void_p] * 4
        L.ofh_qk_score_tile.restype = ctypes.c_int
        vp, sz, i64 = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int64
        i32s, i64s, szs = ctypes.POINTER(ctypes.c_int32), ctypes.POINTER(i64), ctypes.POINTER(sz)
        for fn, result, args in (
                ("ofh_window_params_init", None, [vp]),
                ("ofh_window_attention_workspace_bytes", ctypes.c_int, [vp, szs]),
                ("ofh_window_attention_fwd", ctypes.c_int, [vp] * 6 + [sz, vp]),
                ("ofh_paged_params_init", None, [vp]),
                ("ofh_paged_attention_workspace_bytes", ctypes.c_int, [vp, szs]),
                ("ofh_paged_attention_fwd", ctypes.c_int, [vp] * 6 + [sz, vp]),
                ("ofh_cache_write_params_init", None, [vp]),
                ("ofh_cache_write", ctypes.c_int, [vp] * 6),
                ("ofh_prefix_groups_init", None, [vp]),
                ("ofh_shared_prefix_workspace_bytes", ctypes.c_int, [vp, vp, szs]),
                ("ofh_shared_prefix_attention_fwd", ctypes.c_int, [vp] * 7 + [sz, vp]),
                ("ofh_selected_attention_workspace_bytes", ctypes.c_int, [vp, sz, szs]),
                ("ofh_selected_attention_fwd", ctypes.c_int, [vp, vp, sz] + [vp] * 5 + [sz, vp]),
                ("ofh_page_bounds_params_init", None, [vp]),
                ("ofh_page_bounds", ctypes.c_int, [vp] * 4),
                ("ofh_select_params_init", None, [vp]),
                ("ofh_select_pages_workspace_bytes", ctypes.c_int, [vp, szs]),
                ("ofh_select_pages", ctypes.c_int, [vp] * 5 + [sz, vp]),
                ("ofh_rotary_params_init", None, [vp]),
                ("ofh_rotary_fwd", ctypes.c_int, [vp] * 4),
                ("ofh_cache_append_params_init", None, [vp]),
                ("ofh_cache_append", ctypes.c_int, [vp] * 8),
                ("ofh_cache_copy_pages", ctypes.c_int, [vp, sz, sz, sz, sz, vp, vp, sz, vp]),
                ("ofh_page_pool_create", ctypes.c_int, [sz, sz, ctypes.POINTER(vp)]),
                ("ofh_page_pool_destroy", ctypes.c_int, [vp]),
                ("ofh_page_pool_add", ctypes.c_int, [vp, i64s]),
                ("ofh_page_pool_extend", ctypes.c_int, [vp, i64s, szs, sz, i32s, i32s, szs]),
                ("ofh_page_pool_fork", ctypes.c_int, [vp, i64, i64s]),
                ("ofh_page_pool_truncate", ctypes.c_int, [vp, i64, sz]),
                ("ofh_page_pool_free", ctypes.c_int, [vp, i64]),
                ("ofh_page_pool_compact", ctypes.c_int, [vp, i32s, i32s, sz, szs]),
                ("ofh_page_pool_table", ctypes.c_int, [vp, i64s, sz, i32s, sz, i32s]),
                ("ofh_page_pool_length", ctypes.c_int, [vp, i64, szs]),
                ("ofh_page_pool_info", ctypes.c_int, [vp, szs, szs])):
            getattr(L, fn).restype = result
            getattr(L, fn).argtypes = args
        L.ofh_last_error.restype = ctypes.c_char_p
        L.ofh_last_error.argtypes = []
        L.ofh_abi_version.restype = ctypes.c_int
        for fn in ("ofh_attention_workspace_bytes", "ofh_attention_fwd", "ofh_attention_fwd_noalloc",
                   "ofh_attention_fwd_host",
                   "ofh_attention_launch_info", "ofh_attention_useful_flops"):
            getattr(L, fn).restype = ctypes.c_int
        # attention_fwd's own handle of the entry (its parameters are built flat)
        fwd = L["ofh_attention_fwd"]
        fwd.argtypes = [ctypes.c_void_p] * 6 + [ctypes.c_size_t, ctypes.c_void_p]
        fwd.restype = ctypes.c_int
        L.fwd_flat = fwd
        _lib = L
    return _lib


def check(rc: int) -> None:
    if rc != OFH_SUCCESS:
        raise OfhError(rc, lib().ofh_last_error().decode())


def make_params(batch, heads, query_tokens, key_tokens, head_dim, value_dim=None, *,
                dtype=DTYPE_F32, out_dtype=None, scale=1.0, causal=False, mask_allowed=None,
                mask_query_block_size=0, mask_key_block_size=0, mask_query_blocks=0,
                mask_key_blocks=0, bias_kind=BIAS_NONE, alibi_slopes=None, bias=None,
                bias_strides=(0, 0, 0), softcap=0.0, algorithm=ALGO_AUTO,
                strides=None, max_key_splits=0) -> AttentionParams:
    """Builds an ofh_attention_params. Pointer arguments are integers (device or
    host addresses, as the entry point expects)."""
    p = AttentionParams()
    lib().ofh_attention_params_init(ctypes.byref(p))
    p.batch, p.heads = batch, heads
    p.query_tokens, p.key_tokens = query_tokens, key_tokens
    p.head_dim = head_dim
    p.value_dim = head_dim if value_dim is None else value_dim
    p.dtype = dtype
    p.out_dtype = dtype if out_dtype is None else out_dtype
    p.scale = scale
    p.causal = int(bool(causal))
    if mask_allowed is not None:
        p.mask_allowed = mask_allowed
        p.mask_query_block_size = mask_query_block_size
        p.mask_key_block_size = mask_key_block_size
        p.mask_query_blocks = mask_query_blocks
        p.mask_key_blocks = mask_key_blocks
    p.bias_kind = bias_kind
    if alibi_slopes is not None:
        p.alibi_slopes = alibi_slopes
    if bias is not None:
        p.bias = bias
    for i in range(3):
        p.bias_strides[i] = bias_strides[i]
    if strides is not None:
        for name, s in zip(("q_strides", "k_strides", "v_strides", "o_strides"), strides):
            arr = getattr(p, name)
            for i in range(3):
                arr[i] = s[i]
    p.softcap = softcap
    p.algorithm = algorithm
    p.max_key_splits = max_key_splits
    return p


def launch_info(p: AttentionParams) -> LaunchInfo:
    info = LaunchInfo()
    check(lib().ofh_attention_launch_info(ctypes.byref(p), ctypes.byref(info)))
    return info


def useful_flops(p: AttentionParams) -> float:
    f = ctypes.c_double()
    check(lib().ofh_attention_useful_flops(ctypes.byref(p), ctypes.byref(f)))
    return f.value


def workspace_bytes(p: AttentionParams) -> int:
    n = ctypes.c_size_t()
    check(lib().ofh_attention_workspace_bytes(ctypes.byref(p), ctypes.byref(n)))
    return n.value


# ---------------------------------------------------------------------------
# torch-facing helpers (device tensors)

_torch_module = None
_DTYPE_CODES: dict = {}


def _torch():
    global _torch_module
    if _torch_module is None:
        import torch  # noqa: PLC0415
        _DTYPE_CODES.update({torch.float32: DTYPE_F32, torch.bfloat16: DTYPE_BF16, torch.float16: DTYPE_F16})
        _torch_module = torch
    return _torch_module


def dtype_code(t) -> int:
    _torch()
    return _DTYPE_CODES[t]


def _raw_stream(torch, device) -> int:
    """The current stream's handle on a GPU device (the caller has checked that it
    is one: another device's lookup would be the current GPU's)."""
    index = device.index
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if index is None else index)


def _plain_inputs_fit(torch, q, k, v) -> bool:
    """What _check_attention_inputs asks of q, k and v, in one pass: true only where
    it would find nothing to report about them."""
    tensor = torch.Tensor
    if not (isinstance(q, tensor) and isinstance(k, tensor) and isinstance(v, tensor)):
        return False
    qs, ks, vs, dt, dev = q.shape, k.shape, v.shape, q.dtype, q.device
    if not (len(qs) == 4 and len(ks) == 4 and len(vs) == 4 and dt in _DTYPE_CODES and k.dtype == dt and v.dtype == dt):
        return False
    a, b, c = q.stride(), k.stride(), v.stride()
    return (a[3] == 1 and b[3] == 1 and c[3] == 1 and min(a) >= 0 and min(b) >= 0 and min(c) >= 0
            and ks[0] == qs[0] and ks[1] == qs[1] and vs[0] == qs[0] and vs[1] == qs[1]
            and ks[3] == qs[3] and vs[2] == ks[2] and dev.type == "cuda" and k.device == dev and v.device == dev)


def _check_attention_inputs(q, k, v, mask, mask_block_size, alibi_slopes, bias, out, out_dtype,
                            workspace):
    """Raises ValueError for any argument the kernels would read or write out of
    bounds: shapes, dtypes, devices and layouts are checked before a pointer
    reaches the C ABI (the checks of the TensorFlow op, onednn_flash_attention_op.cc)."""
    torch = _torch()
    floats = (torch.float32, torch.bfloat16, torch.float16)
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or t.dim() != 4:
            raise ValueError(f"{name} must be a rank-4 [B,H,T,D] tensor")
        if t.dtype not in floats:
            raise ValueError(f"{name} must be float32, bfloat16 or float16")
        if t.stride(-1) != 1 or min(t.stride()) < 0:
            raise ValueError(f"{name}: last axis must be contiguous and strides non-negative")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must share one dtype")
    B, H, M, D = q.shape
    if tuple(k.shape[:2]) != (B, H) or tuple(v.shape[:2]) != (B, H):
        raise ValueError("q, k and v must have the same batch and head dimensions")
    if k.shape[3] != D:
        raise ValueError("q/k head dimensions must match")
    if v.shape[2] != k.shape[2]:
        raise ValueError("k/v key-token dimensions must match")
    N, Dv = k.shape[2], v.shape[3]
    dev = q.device
    tensors = [("k", k), ("v", v)]
    if mask is not None:
        if not isinstance(mask, torch.Tensor) or mask.dtype != torch.uint8 or mask.dim() != 2:
            raise ValueError("mask must be a 2-D uint8 tensor [query_blocks, key_blocks]")
        if not mask.is_contiguous():
            raise ValueError("mask must be contiguous")
        if len(mask_block_size) != 2 or min(int(x) for x in mask_block_size) <= 0:
            raise ValueError("mask_block_size must be two positive integers")
        tensors.append(("mask", mask))
    if alibi_slopes is not None and bias is not None:
        raise ValueError("pass either alibi_slopes or bias, not both")
    if alibi_slopes is not None:
        if alibi_slopes.dtype != torch.float32 or alibi_slopes.dim() != 1 or alibi_slopes.shape[0] != H:
            raise ValueError("alibi_slopes must be a float32 tensor of length H")
        if not alibi_slopes.is_contiguous():
            raise ValueError("alibi_slopes must be contiguous")
        tensors.append(("alibi_slopes", alibi_slopes))
    if bias is not None:
        if bias.dtype != torch.float32:
            raise ValueError("bias must be float32")
        if bias.dim() == 2:
            if tuple(bias.shape) != (M, N) or not bias.is_contiguous():
                raise ValueError("a shared bias must be a contiguous [M, N] tensor")
        elif bias.dim() == 4:
            if tuple(bias.shape) != (B, H, M, N) or bias.stride(-1) != 1 or min(bias.stride()) < 0:
                raise ValueError("a per-head bias must be [B, H, M, N] with a contiguous last axis")
        else:
            raise ValueError("bias must be [M, N] or [B, H, M, N]")
        tensors.append(("bias", bias))
    if out is not None:
        if tuple(out.shape) != (B, H, M, Dv):
            raise ValueError(f"out must have shape {(B, H, M, Dv)}")
        if out.dtype not in (q.dtype, torch.float32):
            raise ValueError("out must have the dtype of q or float32")
        if out_dtype is not None and out.dtype != out_dtype:
            raise ValueError("out and out_dtype disagree")
        if out.stride(-1) != 1 or min(out.stride()) < 0:
            raise ValueError("out: last axis must be contiguous and strides non-negative")
        tensors.append(("out", out))
    elif out_dtype is not None and out_dtype not in (q.dtype, torch.float32):
        raise ValueError("out_dtype must be the dtype of q or float32")
    if workspace is not None:
        if workspace.dtype != torch.uint8 or not workspace.is_contiguous():
            raise ValueError("workspace must be a contiguous uint8 tensor")
        tensors.append(("workspace", workspace))
    if dev.type != "cuda":
        raise ValueError("q must be a GPU tensor")
    for name, t in tensors:
        if t.device != dev:
            raise ValueError(f"{name} must be on {dev}")


def attention_fwd(q, k, v, *, scale: float | None = None, causal: bool = False, mask=None,
                  mask_block_size: tuple[int, int] = (1, 1), alibi_slopes=None, bias=None,
                  softcap: float = 0.0, out=None, out_dtype=None, algorithm: int = ALGO_AUTO,
                  workspace=None, stream=None, max_key_splits: int = 0):
    """q: [B,H,M,D], k: [B,H,N,D], v: [B,H,N,Dv] device tensors (f32/bf16/f16, last
    axis contiguous). mask: uint8 device tensor [qblocks, kblocks]. alibi_slopes:
    f32 device [H]. bias: f32 device [M,N] (shared) or [B,H,M,N]. Returns out.
    Raises ValueError before any launch when the arguments do not fit together."""
    torch = _torch()
    # (with q, k and v alone there is nothing else to check)
    alone = (mask is None and alibi_slopes is None and bias is None and out is None and out_dtype is None
             and workspace is None)
    if not (alone and _plain_inputs_fit(torch, q, k, v)):
        _check_attention_inputs(q, k, v, mask, mask_block_size, alibi_slopes, bias, out, out_dtype,
                                workspace)
    B, H, M, D = q.shape
    N, Dv = k.shape[2], v.shape[3]
    if out is None:
        out = torch.empty((B, H, M, Dv), device=q.device,
                          dtype=q.dtype if out_dtype is None else out_dtype)
    mask_args = (None, 0, 0, 0, 0)
    if mask is not None:
        mask_args = (mask.data_ptr(), int(mask_block_size[0]), int(mask_block_size[1]), mask.shape[0], mask.shape[1])
    bias_kind, slopes_ptr, bias_ptr, bias_strides = BIAS_NONE, None, None, (0, 0, 0)
    if alibi_slopes is not None:
        bias_kind, slopes_ptr = BIAS_ALIBI, alibi_slopes.data_ptr()
    elif bias is not None:
        bias_kind, bias_ptr = BIAS_DENSE, bias.data_ptr()
        if bias.dim() == 4:
            bias_strides = bias.stride()[:3]
    p = _FlatAttentionParams(
        ctypes.sizeof(AttentionParams), B, H, M, N, D, Dv, _DTYPE_CODES[q.dtype], _DTYPE_CODES[out.dtype],
        *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *out.stride()[:3],
        (1.0 / math.sqrt(D)) if scale is None else scale, int(bool(causal)), *mask_args, bias_kind, slopes_ptr,
        bias_ptr, *bias_strides, softcap, algorithm, max_key_splits)
    if stream is None:
        stream = _raw_stream(torch, q.device)
    ws_ptr, ws_bytes = (0, 0) if workspace is None else (workspace.data_ptr(), workspace.numel() * workspace.element_size())
    rc = lib().fwd_flat(ctypes.addressof(p), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), ws_ptr or None,
                        ws_bytes, stream)
    if rc != OFH_SUCCESS:
        check(rc)
    return out


def qk_score_tile(q, k, *, scale: float | None = None, bias=None, softcap: float = 0.0,
                  out=None, algorithm: int = QK_AUTO, stream=None):
    """Scores S = (Q K^T) * scale + bias for a batch of tiles on the device
    (qk_score_tile_inplace, src/onednn_flash/qk_score_tile.cpp:353-418).
    q: [T, M, D], k: [T, N, D] device tensors (f32/bf16/f16, any strides);
    bias: f32 [T, M, N], [M, N] (shared by every tile) or None; scale None
    means no scale post-op. Returns out, f32 [T, M, N]."""
    torch = _torch()
    T, M, D = q.shape
    N = k.shape[1]
    if k.shape[0] != T or k.shape[2] != D or k.dtype != q.dtype:
        raise ValueError("k must be [T, N, D] with the dtype of q")
    if q.device.type != "cuda":
        raise ValueError(f"Expected a cuda device, but got: {q.device}")
    if out is None:
        out = torch.empty((T, M, N), device=q.device, dtype=torch.float32)
    p = QkScoreParams()
    lib().ofh_qk_score_params_init(ctypes.byref(p))
    p.batch, p.m, p.n, p.k = T, M, N, D
    p.a_stride_batch, p.a_stride_m, p.a_stride_k = q.stride()
    p.b_stride_batch, p.b_stride_n, p.b_stride_k = k.stride()
    p.c_stride_batch, p.c_stride_m, p.c_stride_n = out.stride()
    p.dtype = dtype_code(q.dtype)
    if scale is not None:
        p.has_scale, p.scale = 1, scale
    if bias is not None:
        if bias.dtype != torch.float32:
            raise ValueError("bias must be float32")
        p.bias = bias.data_ptr()
        if bias.dim() == 2:
            p.bias_stride_batch, (p.bias_stride_m, p.bias_stride_n) = 0, bias.stride()
        else:
            p.bias_stride_batch, p.bias_stride_m, p.bias_stride_n = bias.stride()
    p.softcap = softcap
    p.algorithm = algorithm
    if stream is None:
        stream = _raw_stream(torch, q.device)
    check(lib().ofh_qk_score_tile(ctypes.byref(p), q.data_ptr(), k.data_ptr(), out.data_ptr(),
                                  stream))
    return out


# ---------------------------------------------------------------------------
# Serving: windowed attention of prompts, attention over a paged key-value
# cache, writing and copying of its pages. onednn_flash_cache.PagedCache keeps
# such a cache.

def _launch(torch, device, stream, entry, *args):
    """entry(*args, stream handle) with `device` current: the library launches on
    the current device."""
    index = device.index
    if stream is None:
        stream = torch._C._cuda_getCurrentRawStream(index)
    if index == torch._C._cuda_getDevice():
        rc = entry(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = entry(*args, stream)
    return rc


def _check_rows(torch, name, t, dims, dtype, device):
    """t is a tensor of `dims` dimensions with contiguous rows (None: any dtype or device)."""
    if not isinstance(t, torch.Tensor) or t.dim() != dims:
        raise ValueError(f"{name} must be a rank-{dims} tensor")
    if t.dtype not in _DTYPE_CODES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}")
    if 0 in t.shape:
        raise ValueError(f"{name} must not be empty")
    if (t.shape[-1] > 1 and t.stride(-1) != 1) or min(t.stride()) < 0:
        raise ValueError(f"{name}: last axis must be contiguous and strides non-negative")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be a GPU tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name} must be on {device}")


def _axis_strides(name, t):
    """The strides of t's first three axes as the C ABI takes them: those of axes of
    one element, which torch leaves open, as a row's length, and never all zero
    (which would mean a contiguous tensor)."""
    s0, s1, s2, row = t.shape
    a, b, c, _ = t.stride()
    if s0 == 1:
        a = row
    if s1 == 1:
        b = row
    if s2 == 1:
        c = row
    if a == 0 and b == 0 and c == 0:
        raise ValueError(f"{name} must not be one row broadcast over every axis")
    return a, b, c


def _is_rows(torch, t, dtype, device):
    """What _check_rows asks of a 4-axis tensor, in one pass: true only where it
    would find nothing to report."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != device:
        return False
    shape, stride = t.shape, t.stride()
    return len(shape) == 4 and 0 not in shape and min(stride) >= 0 and (stride[3] == 1 or shape[3] == 1)


def _check_written(name, t):
    """No two elements of t may share memory: it is written."""
    for size, stride in zip(t.shape, t.stride()):
        if size > 1 and stride == 0:
            raise ValueError(f"{name} must not be a broadcast tensor")


def _check_ints(torch, name, t, shape, device):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be an int32 tensor of shape {shape}")
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        raise ValueError(f"{name}: last axis must be contiguous")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")


def _check_slopes(torch, slopes, heads, device):
    if not isinstance(slopes, torch.Tensor) or slopes.dtype != torch.float32 or tuple(slopes.shape) != (heads,) \
            or not slopes.is_contiguous():
        raise ValueError("alibi_slopes must be a contiguous float32 tensor of length H")
    if slopes.device != device:
        raise ValueError(f"alibi_slopes must be on {device}")


def _check_counts(**values):
    for name, x in values.items():
        if type(x) is not int or x < 0 or x >= 1 << (31 if name == "max_key_splits" else 63):
            raise ValueError(f"{name} must be a non-negative integer")


def _check_out(torch, out, shape, dtype, device):
    _check_rows(torch, "out", out, 4, None, device)
    if tuple(out.shape) != shape:
        raise ValueError(f"out must have shape {shape}")
    if out.dtype not in (dtype, torch.float32):
        raise ValueError("out must have the dtype of q or float32")
    _check_written("out", out)


def _given_workspace(torch, workspace, out):
    """Address and bytes of a caller's workspace. An empty one has no address, which
    would mean the library's scratch: out's stands for it, with no bytes."""
    if not isinstance(workspace, torch.Tensor) or workspace.dtype != torch.uint8 or not workspace.is_contiguous() \
            or workspace.device != out.device:
        raise ValueError(f"workspace must be a contiguous uint8 tensor on {out.device}")
    return workspace.data_ptr() or out.data_ptr(), workspace.numel()


def _new_workspace(torch, need, device, stream):
    """Scratch of one call on `stream` (a handle or a torch stream; None: the current
    one). It is freed when the call returns, so it belongs to the stream that uses it."""
    with _on_stream(torch, device, stream):
        return torch.empty(need, dtype=torch.uint8, device=device)


def _on_stream(torch, device, stream):
    """Context in which tensors are allocated on `stream` (as _new_workspace takes it)."""
    if stream is None or device.type != "cuda":
        return contextlib.nullcontext()
    if not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.ExternalStream(stream, device=device)
    return torch.cuda.stream(stream)


class _Kept:
    """Device tensors of the library's own that kernels read, on whichever stream an
    object is called. When nothing holds them their memory goes to the next tensor of
    the stream that they were made on, so a call on another torch stream tells the
    allocator, which then waits for it. (Not for a stream given by its handle or as an
    ExternalStream, which may be gone by then and is nothing to wait for: such a call's
    object is kept until it has run.)"""

    def __init__(self, torch, *tensors):
        self._torch, self.tensors, self._index = torch, tensors, tensors[0].device.index
        self._told = set()
        if self._index is not None:  # (None: on the CPU)
            self._current = torch._C._cuda_getCurrentRawStream
            self._told.add(self._current(self._index))

    def used(self, stream) -> None:
        """A call on `stream` (as _launch takes it) reads the tensors."""
        if self._index is None:
            return
        if stream is None:
            if self._current(self._index) in self._told:
                return
            stream = self._torch.cuda.current_stream(self._index)
        elif not isinstance(stream, self._torch.cuda.Stream) or isinstance(stream, self._torch.cuda.ExternalStream):
            return
        if stream.cuda_stream not in self._told:
            for t in self.tensors:
                t.record_stream(stream)
            self._told.add(stream.cuda_stream)


def _workspace_need(query, p, *more) -> int:
    need = ctypes.c_size_t()
    rc = query(p if isinstance(p, bytes) else ctypes.addressof(p), *more, ctypes.byref(need))
    if rc != OFH_SUCCESS:
        check(rc)
    return need.value


def window_attention(q, k, v, *, window: int = 0, sink_tokens: int = 0, scale: float | None = None,
                     query_offset: int = 0, lengths=None, alibi_slopes=None, softcap: float = 0.0, out=None,
                     out_dtype=None, workspace=None, stream=None, max_key_splits: int = 0):
    """Causal attention of prompts with a sliding window and first tokens that
    stay visible. q: [B,H,M,D], k: [B,Hkv,N,D], v: [B,Hkv,N,Dv] device tensors,
    H a multiple of Hkv (query head h reads key-value head h / (H / Hkv)).

    Query row i is at position p = query_offset + i and sees key j iff j <= p
    and p - j < window (any, with window 0) or j < sink_tokens. lengths: int32
    device [B], the tokens of each sequence of a padded batch: keys from there
    on are not seen, query rows at those positions are written as 0. scale
    defaults to 1 / sqrt(D); alibi_slopes: f32 device [H]. Rows that see nothing
    are 0. Returns out, [B,H,M,Dv].

    The workspace (partial rows of calls with few query rows) is taken from
    torch's allocator unless given."""
    torch = _torch()
    if not (isinstance(q, torch.Tensor) and q.dtype in _DTYPE_CODES and q.device.type == "cuda"
            and _is_rows(torch, q, q.dtype, q.device) and _is_rows(torch, k, q.dtype, q.device)
            and _is_rows(torch, v, q.dtype, q.device)):
        _check_rows(torch, "q", q, 4, None, None)
        _check_rows(torch, "k", k, 4, q.dtype, q.device)
        _check_rows(torch, "v", v, 4, q.dtype, q.device)
    dev, dtype = q.device, q.dtype
    B, H, M, D = q.shape
    _, Hkv, N, _ = k.shape
    Dv = v.shape[3]
    if k.shape != (B, Hkv, N, D) or v.shape != (B, Hkv, N, Dv) or H % Hkv != 0:
        raise ValueError("k must be [B, Hkv, N, D] and v [B, Hkv, N, Dv] with H a multiple of Hkv")
    if not (type(window) is int is type(sink_tokens) is type(query_offset) is type(max_key_splits)
            and 0 <= window < 1 << 63 and 0 <= sink_tokens < 1 << 63 and 0 <= query_offset < 1 << 63
            and 0 <= max_key_splits < 1 << 31):
        _check_counts(window=window, sink_tokens=sink_tokens, query_offset=query_offset, max_key_splits=max_key_splits)
    if lengths is not None:
        _check_ints(torch, "lengths", lengths, (B,), dev)
    if alibi_slopes is not None:
        _check_slopes(torch, alibi_slopes, H, dev)
    if out is None:
        if out_dtype not in (None, dtype, torch.float32):
            raise ValueError("out_dtype must be the dtype of q or float32")
        out = torch.empty((B, H, M, Dv), dtype=dtype if out_dtype is None else out_dtype, device=dev)
        o_strides = (0, 0, 0)  # contiguous
    else:
        _check_out(torch, out, (B, H, M, Dv), dtype, dev)
        if out_dtype is not None and out.dtype != out_dtype:
            raise ValueError("out and out_dtype disagree")
        o_strides = _axis_strides("out", out)
    p = _pack_window.pack(
        _pack_window.size, B, H, Hkv, M, N, D, Dv, _DTYPE_CODES[dtype], _DTYPE_CODES[out.dtype],
        *_axis_strides("q", q), *_axis_strides("k", k), *_axis_strides("v", v), *o_strides,
        (1.0 / math.sqrt(D)) if scale is None else scale, softcap,
        0 if alibi_slopes is None else alibi_slopes.data_ptr(), window, sink_tokens, query_offset,
        0 if lengths is None else lengths.data_ptr(), max_key_splits)
    L = lib()
    args = (p, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr())
    if workspace is not None:
        rc = _launch(torch, dev, stream, L.ofh_window_attention_fwd, *args, *_given_workspace(torch, workspace, out))
    else:
        # most calls need none: first with an empty one, which a call that does refuses
        rc = _launch(torch, dev, stream, L.ofh_window_attention_fwd, *args, out.data_ptr(), 0)
        if rc == OFH_ERROR_WORKSPACE_TOO_SMALL:
            need = _workspace_need(L.ofh_window_attention_workspace_bytes, p)
            workspace = _new_workspace(torch, need, dev, stream)
            rc = _launch(torch, dev, stream, L.ofh_window_attention_fwd, *args, workspace.data_ptr(), need)
    if rc != OFH_SUCCESS:
        check(rc)
    return out


def _check_pool(torch, k_pages, v_pages, page_table, lengths, batch=None):
    """The tensors of a paged cache: k_pages [P,Hkv,S,D], v_pages [P,Hkv,S,Dv],
    page_table [B,max_pages] and lengths [B]. Returns the batch."""
    _check_rows(torch, "k_pages", k_pages, 4, None, None)
    dev = k_pages.device
    _check_rows(torch, "v_pages", v_pages, 4, k_pages.dtype, dev)
    if v_pages.shape[:3] != k_pages.shape[:3]:
        raise ValueError("k_pages must be [P, Hkv, S, D] and v_pages [P, Hkv, S, Dv]")
    if not isinstance(page_table, torch.Tensor) or page_table.dim() != 2 or 0 in page_table.shape:
        raise ValueError("page_table must be an int32 tensor [B, max_pages]")
    _check_ints(torch, "page_table", page_table, tuple(page_table.shape), dev)
    if page_table.shape[0] > 1 and page_table.stride(0) == 0:  # (a stride of 0 means contiguous rows)
        raise ValueError("page_table must not be a broadcast tensor")
    _check_ints(torch, "lengths", lengths, (page_table.shape[0],), dev)


class PagedAttention:
    """Attention of new tokens over a paged key-value cache, for a program that
    keeps the cache's tensors and calls it step after step: their checks are made
    once, here, and each call reads what they hold then.

    k_pages: [P,Hkv,S,D], v_pages: [P,Hkv,S,Dv] (S a power of two, 16 or more);
    page_table: int32 [B,max_pages], key j of sequence b being row j % S of page
    page_table[b, j // S]; lengths: int32 [B], the tokens of each sequence with
    the query_tokens new ones, whose keys are in the cache by then (cache_write).
    Token t of a sequence is at position lengths[b] - query_tokens + t and sees
    what window_attention lets it see. Entries of keys that no token sees are
    not read; the keys of an entry outside the pool are not seen."""

    def __init__(self, k_pages, v_pages, page_table, lengths, *, heads: int, query_tokens: int = 1, window: int = 0,
                 sink_tokens: int = 0, scale: float | None = None, alibi_slopes=None, softcap: float = 0.0,
                 out_dtype=None, max_key_splits: int = 0):
        torch = _torch()
        _check_pool(torch, k_pages, v_pages, page_table, lengths)
        _check_counts(heads=heads, query_tokens=query_tokens, window=window, sink_tokens=sink_tokens,
                      max_key_splits=max_key_splits)
        P, Hkv, S, D = k_pages.shape
        B, max_pages = page_table.shape
        Dv = v_pages.shape[3]
        if heads == 0 or heads % Hkv != 0 or query_tokens == 0:
            raise ValueError("heads must be a positive multiple of the cache's heads, query_tokens positive")
        if alibi_slopes is not None:
            _check_slopes(torch, alibi_slopes, heads, k_pages.device)
        if out_dtype not in (None, k_pages.dtype, torch.float32):
            raise ValueError("out_dtype must be the dtype of the cache or float32")
        self._torch = torch
        self._held = (k_pages, v_pages, page_table, lengths, alibi_slopes)
        self._device, self._dtype = k_pages.device, k_pages.dtype
        self._out_dtype = k_pages.dtype if out_dtype is None else out_dtype
        self._q_shape, self._out_shape = (B, heads, query_tokens, D), (B, heads, query_tokens, Dv)
        p = PagedParams()
        L = lib()
        L.ofh_paged_params_init(ctypes.addressof(p))
        p.batch, p.heads, p.kv_heads, p.query_tokens, p.head_dim, p.value_dim = B, heads, Hkv, query_tokens, D, Dv
        p.num_pages, p.page_size, p.max_pages, p.table_stride = P, S, max_pages, page_table.stride(0) if B > 1 else 0
        p.dtype = _DTYPE_CODES[self._dtype]
        p.k_strides[:], p.v_strides[:] = _axis_strides("k_pages", k_pages), _axis_strides("v_pages", v_pages)
        p.page_table, p.lengths = page_table.data_ptr(), lengths.data_ptr()
        p.scale = (1.0 / math.sqrt(D)) if scale is None else scale
        p.softcap = softcap
        if alibi_slopes is not None:
            p.alibi_slopes = alibi_slopes.data_ptr()
        p.window, p.sink_tokens, p.max_key_splits = window, sink_tokens, max_key_splits
        p.out_dtype = _DTYPE_CODES[self._out_dtype]
        self._params = bytes(p)
        self._ptrs = (k_pages.data_ptr(), v_pages.data_ptr())
        self._plan(L, p)

    def _plan(self, L, p: PagedParams) -> None:
        """The entry, its arguments behind the parameters, and the scratch it needs."""
        self._fwd, self._more = L.ofh_paged_attention_fwd, ()
        self._need = _workspace_need(L.ofh_paged_attention_workspace_bytes, p)

    @property
    def workspace_bytes(self) -> int:
        return self._need

    def __call__(self, q, *, out=None, workspace=None, stream=None):
        """q: [B,H,T,D] in the cache's dtype. Returns out, [B,H,T,Dv]."""
        self._check_query(q)
        return self._attend(q, self._more, out, workspace, stream)

    def _check_query(self, q) -> None:
        torch, dev = self._torch, self._device
        if not (_is_rows(torch, q, self._dtype, dev) and q.shape == self._q_shape):
            raise ValueError(f"q must be a {self._dtype} tensor of shape {self._q_shape} on {dev}, its last axis "
                             "contiguous and strides non-negative")

    def _attend(self, q, more, out, workspace, stream):
        torch, dev = self._torch, self._device
        p = PagedParams.from_buffer_copy(self._params)  # (its own: calls may run on several threads)
        if not q.is_contiguous():
            p.q_strides[:] = _axis_strides("q", q)
        if out is None:
            out = torch.empty(self._out_shape, dtype=self._out_dtype, device=dev)
        else:
            _check_out(torch, out, self._out_shape, self._dtype, dev)
            p.out_dtype = _DTYPE_CODES[out.dtype]
            p.o_strides[:] = _axis_strides("out", out)
        ws, ws_bytes = None, 0
        if workspace is not None:
            ws, ws_bytes = _given_workspace(torch, workspace, out)
        elif self._need:
            workspace = _new_workspace(torch, self._need, dev, stream)
            ws, ws_bytes = workspace.data_ptr(), self._need
        rc = _launch(torch, dev, stream, self._fwd, ctypes.addressof(p), *more, q.data_ptr(), *self._ptrs, out.data_ptr(),
                     ws, ws_bytes)
        if rc != OFH_SUCCESS:
            check(rc)
        return out


def paged_attention(q, k_pages, v_pages, page_table, lengths, *, window: int = 0, sink_tokens: int = 0,
                    scale: float | None = None, alibi_slopes=None, softcap: float = 0.0, out=None, out_dtype=None,
                    workspace=None, stream=None, max_key_splits: int = 0):
    """One call of PagedAttention: q [B,H,T,D], the T new tokens of each sequence."""
    if q.dim() != 4:
        raise ValueError("q must be a rank-4 tensor")
    if out is not None and out_dtype is not None and out.dtype != out_dtype:
        raise ValueError("out and out_dtype disagree")
    return PagedAttention(k_pages, v_pages, page_table, lengths, heads=q.shape[1], query_tokens=q.shape[2],
                          window=window, sink_tokens=sink_tokens, scale=scale, alibi_slopes=alibi_slopes,
                          softcap=softcap, out_dtype=out_dtype, max_key_splits=max_key_splits)(
                              q, out=out, workspace=workspace, stream=stream)


class PrefixGroups:
    """Which sequences of a batch share prefixes: (sequences, shared tokens) of each
    group, in the batch's order. The sequences of a group have their first shared
    tokens, whole pages of the cache, in the same pages (0: they share nothing).
    Kept on `device` for the calls that take it."""

    def __init__(self, groups, *, page_size: int, device="cuda"):
        torch = _torch()
        groups = [tuple(g) for g in groups]
        for g in groups:
            if len(g) != 2 or any(type(x) is not int for x in g) or g[0] <= 0 or not 0 <= g[1] < 1 << 31:
                raise ValueError("groups must be pairs of a positive number of sequences and a number of shared tokens")
            if g[1] % page_size:
                raise ValueError("shared tokens must be whole pages")
        if not groups:
            raise ValueError("groups must not be empty")
        self.groups = groups
        self.batch = sum(n for n, _ in groups)
        starts, shared = [0], []
        for n, tokens in groups:
            starts.append(starts[-1] + n)
            shared += [tokens] * n
        self._kept = _Kept(torch, *(torch.tensor(x, dtype=torch.int32, device=device) for x in (starts, shared)))
        p = PrefixGroupsParams()
        lib().ofh_prefix_groups_init(ctypes.addressof(p))
        p.groups, p.starts, p.shared_tokens = len(groups), *(t.data_ptr() for t in self._kept.tensors)
        p.least_shared, p.most_shared = min(shared), max(shared)
        sharing = [n for n, tokens in groups if tokens > 0]
        p.most_sequences, p.sharing_groups, p.sharing_sequences = max(sharing, default=0), len(sharing), sum(sharing)
        self._params = p


class SharedPrefixAttention(PagedAttention):
    """PagedAttention of a batch whose sequences share prefixes: the keys that a
    group of sequences has in common are read once for all of it. The result is
    PagedAttention's, up to rounding. groups: a PrefixGroups, or its list of
    (sequences, shared tokens)."""

    def __init__(self, k_pages, v_pages, page_table, lengths, *, groups, heads: int, query_tokens: int = 1, **options):
        self._groups_given = groups
        super().__init__(k_pages, v_pages, page_table, lengths, heads=heads, query_tokens=query_tokens, **options)

    def _plan(self, L, p: PagedParams) -> None:
        groups = self._groups_given
        if not isinstance(groups, PrefixGroups):
            groups = PrefixGroups(groups, page_size=p.page_size, device=self._device)
        if groups.batch != p.batch:
            raise ValueError(f"groups must have the batch's {p.batch} sequences together")
        if groups._kept.tensors[0].device != self._device:
            raise ValueError(f"groups must be on {self._device}")
        if any(tokens % p.page_size or tokens > p.max_pages * p.page_size for _, tokens in groups.groups):
            raise ValueError("shared tokens must be whole pages of the table's rows")
        self._groups = groups
        self._fwd, self._more = L.ofh_shared_prefix_attention_fwd, (ctypes.addressof(groups._params),)
        self._need = _workspace_need(L.ofh_shared_prefix_workspace_bytes, p, *self._more)

    def _attend(self, q, more, out, workspace, stream):
        self._groups._kept.used(stream)
        return super()._attend(q, more, out, workspace, stream)


def shared_prefix_attention(q, k_pages, v_pages, page_table, lengths, *, groups, out=None, out_dtype=None, workspace=None,
                            stream=None, **options):
    """One call of SharedPrefixAttention: q [B,H,T,D], the T new tokens of each sequence."""
    if q.dim() != 4:
        raise ValueError("q must be a rank-4 tensor")
    if out is not None and out_dtype is not None and out.dtype != out_dtype:
        raise ValueError("out and out_dtype disagree")
    # (the groups of a list are freed when the call returns, as its scratch is)
    with _on_stream(_torch(), q.device, stream):
        attend = SharedPrefixAttention(k_pages, v_pages, page_table, lengths, groups=groups, heads=q.shape[1],
                                       query_tokens=q.shape[2], out_dtype=out_dtype, **options)
    return attend(q, out=out, workspace=workspace, stream=stream)


def _check_bounds(torch, k_pages, k_bounds):
    _check_rows(torch, "k_bounds", k_bounds, 4, k_pages.dtype, k_pages.device)
    P, Hkv, _, D = k_pages.shape
    if k_bounds.shape != (P, Hkv, 2, D):
        raise ValueError("k_bounds must be [P, Hkv, 2, D]")


class PageBounds:
    """Keeps what SelectedAttention scores pages by: k_bounds [P,Hkv,2,D], the
    smallest and the largest value of every column of a page's keys (NaN where one
    is). Each call renews those of the pages that hold the last counts[b] tokens of
    each sequence (`tokens` without counts, which are at most that): what a
    cache_write of these tokens is followed by. The page's own tokens count, up to
    lengths[b]; sequences that share a page agree on them."""

    def __init__(self, k_pages, k_bounds, page_table, lengths, *, tokens: int, counts=None):
        torch = _torch()
        _check_pool(torch, k_pages, k_pages, page_table, lengths)
        _check_bounds(torch, k_pages, k_bounds)
        _check_written("k_bounds", k_bounds)
        if type(tokens) is not int or not 0 < tokens < 1 << 63:
            raise ValueError("tokens must be a positive integer")
        P, Hkv, S, D = k_pages.shape
        B, max_pages = page_table.shape
        if counts is not None:
            _check_ints(torch, "counts", counts, (B,), k_pages.device)
        self._torch, self._device = torch, k_pages.device
        self._held = (k_pages, k_bounds, page_table, lengths, counts)
        p = PageBoundsParams()
        L = lib()
        L.ofh_page_bounds_params_init(ctypes.addressof(p))
        p.batch, p.kv_heads, p.tokens, p.head_dim = B, Hkv, tokens, D
        p.num_pages, p.page_size, p.max_pages, p.table_stride = P, S, max_pages, page_table.stride(0) if B > 1 else 0
        p.dtype = _DTYPE_CODES[k_pages.dtype]
        p.k_page_strides[:], p.bounds_strides[:] = _axis_strides("k_pages", k_pages), _axis_strides("k_bounds", k_bounds)
        p.page_table, p.lengths = page_table.data_ptr(), lengths.data_ptr()
        if counts is not None:
            p.counts = counts.data_ptr()
        self._params = p  # (read by calls, never changed)
        self._args = (ctypes.addressof(p), k_pages.data_ptr(), k_bounds.data_ptr())
        self._update = L.ofh_page_bounds

    def __call__(self, *, stream=None) -> None:
        rc = _launch(self._torch, self._device, stream, self._update, *self._args)
        if rc != OFH_SUCCESS:
            check(rc)


def page_bounds(k_pages, k_bounds, page_table, lengths, *, tokens: int | None = None, counts=None, stream=None) -> None:
    """One call of PageBounds; without `tokens` it renews every page of the sequences."""
    if tokens is None:
        tokens = 1 << 30  # (the most that a sequence has)
    PageBounds(k_pages, k_bounds, page_table, lengths, tokens=tokens, counts=counts)(stream=stream)


class SelectedAttention(PagedAttention):
    """Sparse attention of new tokens over a paged cache: each token attends, for
    each key-value head, to `pages` of its sequence's pages: the first
    `first_pages`, the last `recent_pages` of those with keys up to the token's
    position, and between them those of the highest score (all when there are at
    most `pages`). The score bounds q.k over a page from its k_bounds (PageBounds):
    the largest, over the query heads of the key-value head, of
    sum_d q_d (q_d > 0 ? hi_d : lo_d); ties go to the lower page. Scores leave
    ALiBi and the soft-cap out. Otherwise as PagedAttention, without a window."""

    def __init__(self, k_pages, v_pages, k_bounds, page_table, lengths, *, heads: int, pages: int, first_pages: int = 1,
                 recent_pages: int = 2, query_tokens: int = 1, scale: float | None = None, alibi_slopes=None,
                 softcap: float = 0.0, out_dtype=None, max_key_splits: int = 0):
        torch = _torch()
        _check_pool(torch, k_pages, v_pages, page_table, lengths)
        _check_bounds(torch, k_pages, k_bounds)
        _check_counts(pages=pages, first_pages=first_pages, recent_pages=recent_pages)
        if pages == 0 or first_pages + recent_pages > pages:
            raise ValueError("pages must be positive and hold first_pages and recent_pages together")
        self._pages, self._select_pages = pages, (first_pages, recent_pages)
        self._bounds = k_bounds
        super().__init__(k_pages, v_pages, page_table, lengths, heads=heads, query_tokens=query_tokens, scale=scale,
                         alibi_slopes=alibi_slopes, softcap=softcap, out_dtype=out_dtype, max_key_splits=max_key_splits)

    def _plan(self, L, p: PagedParams) -> None:
        s = SelectParams()
        L.ofh_select_params_init(ctypes.addressof(s))
        for name in ("batch", "heads", "kv_heads", "query_tokens", "head_dim", "num_pages", "page_size", "max_pages",
                     "table_stride", "dtype", "page_table", "lengths"):
            setattr(s, name, getattr(p, name))
        s.bounds_strides[:] = _axis_strides("k_bounds", self._bounds)
        s.negative = int(p.scale < 0)
        s.pages, (s.first_pages, s.recent_pages) = self._pages, self._select_pages
        self._select_params = bytes(s)
        self._select = L.ofh_select_pages
        self._select_need = _workspace_need(L.ofh_select_pages_workspace_bytes, s)
        self._selected_shape = (p.batch, p.kv_heads, p.query_tokens, self._pages)
        self._fwd, self._more = L.ofh_selected_attention_fwd, ()
        self._need = _workspace_need(L.ofh_selected_attention_workspace_bytes, p, self._pages)

    @property
    def select_workspace_bytes(self) -> int:
        return self._select_need

    def _check_selected(self, selected) -> None:
        _check_ints(self._torch, "selected", selected, self._selected_shape, self._device)
        if not selected.is_contiguous():
            raise ValueError("selected must be contiguous")

    def _run_select(self, q, address, workspace, stream) -> None:
        torch, dev = self._torch, self._device
        s = SelectParams.from_buffer_copy(self._select_params)
        if not q.is_contiguous():
            s.q_strides[:] = _axis_strides("q", q)
        ws, ws_bytes = None, 0
        if workspace is not None:
            ws, ws_bytes = _given_workspace(torch, workspace, q)
        elif self._select_need:
            workspace = _new_workspace(torch, self._select_need, dev, stream)
            ws, ws_bytes = workspace.data_ptr(), self._select_need
        rc = _launch(torch, dev, stream, self._select, ctypes.addressof(s), q.data_ptr(), self._bounds.data_ptr(), address,
                     ws, ws_bytes)
        if rc != OFH_SUCCESS:
            check(rc)

    def select(self, q, *, out=None, workspace=None, stream=None):
        """The pages that the tokens of q [B,H,T,D] attend to: int32
        [B,Hkv,T,pages], places in the sequence's row of the page table, ascending,
        then -1. workspace: of select_workspace_bytes."""
        self._check_query(q)
        if out is None:
            out = self._torch.empty(self._selected_shape, dtype=self._torch.int32, device=self._device)
        else:
            self._check_selected(out)
        self._run_select(q, out.data_ptr(), workspace, stream)
        return out

    def __call__(self, q, *, selected=None, out=None, workspace=None, stream=None):
        """q: [B,H,T,D] in the cache's dtype. selected: of select() for these or other
        queries (several layers or steps may share one), or of the program's own
        making; without it the call selects. Returns out, [B,H,T,Dv]. workspace: of
        workspace_bytes, for the attention."""
        self._check_query(q)
        if selected is None:
            held = _new_workspace(self._torch, 4 * math.prod(self._selected_shape), self._device, stream)
            address = held.data_ptr()
            self._run_select(q, address, None, stream)
        else:
            self._check_selected(selected)
            address = selected.data_ptr()
        return self._attend(q, (address, self._pages), out, workspace, stream)


class CacheWriter:
    """Writes new keys and values into the pages of a cache, for a program that
    keeps the cache's tensors (as PagedAttention). Token t < counts[b] of
    sequence b (every token without counts) goes to position lengths[b] -
    counts[b] + t; tokens without a place in the table or the pool are not
    written. Sequences that share a page must not write the same place of it
    (PagedCache.extend gives each its own)."""

    def __init__(self, k_pages, v_pages, page_table, lengths, *, counts=None):
        torch = _torch()
        _check_pool(torch, k_pages, v_pages, page_table, lengths)
        _check_written("k_pages", k_pages)
        _check_written("v_pages", v_pages)
        P, Hkv, S, D = k_pages.shape
        B, max_pages = page_table.shape
        if counts is not None:
            _check_ints(torch, "counts", counts, (B,), k_pages.device)
        self._torch = torch
        self._held = (k_pages, v_pages, page_table, lengths, counts)
        self._device, self._dtype = k_pages.device, k_pages.dtype
        self._row = (B, Hkv, D, v_pages.shape[3])
        p = CacheWriteParams()
        L = lib()
        L.ofh_cache_write_params_init(ctypes.addressof(p))
        p.batch, p.kv_heads, p.head_dim, p.value_dim = B, Hkv, D, v_pages.shape[3]
        p.num_pages, p.page_size, p.max_pages, p.table_stride = P, S, max_pages, page_table.stride(0) if B > 1 else 0
        p.dtype = _DTYPE_CODES[self._dtype]
        p.k_page_strides[:] = _axis_strides("k_pages", k_pages)
        p.v_page_strides[:] = _axis_strides("v_pages", v_pages)
        p.page_table, p.lengths = page_table.data_ptr(), lengths.data_ptr()
        if counts is not None:
            p.counts = counts.data_ptr()
        self._params = bytes(p)
        self._write = L.ofh_cache_write
        self._ptrs = (k_pages.data_ptr(), v_pages.data_ptr())

    def _check_new(self, k, v) -> int:
        """Checks the new rows; returns how many there are per sequence."""
        torch, dev = self._torch, self._device
        B, Hkv, D, Dv = self._row
        if not (_is_rows(torch, k, self._dtype, dev) and _is_rows(torch, v, self._dtype, dev)):
            _check_rows(torch, "k", k, 4, self._dtype, dev)
            _check_rows(torch, "v", v, 4, self._dtype, dev)
        T = k.shape[2]
        if k.shape != (B, Hkv, T, D) or v.shape != (B, Hkv, T, Dv):
            raise ValueError(f"k must be {(B, Hkv, 'T', D)} and v {(B, Hkv, 'T', Dv)}")
        return T

    def __call__(self, k, v, *, stream=None) -> None:
        """k: [B,Hkv,T,D], v: [B,Hkv,T,Dv], the (padded) new rows."""
        torch, dev = self._torch, self._device
        T = self._check_new(k, v)
        p = CacheWriteParams.from_buffer_copy(self._params)
        p.tokens = T
        if not k.is_contiguous():
            p.k_strides[:] = _axis_strides("k", k)
        if not v.is_contiguous():
            p.v_strides[:] = _axis_strides("v", v)
        rc = _launch(torch, dev, stream, self._write, ctypes.addressof(p), k.data_ptr(), v.data_ptr(), *self._ptrs)
        if rc != OFH_SUCCESS:
            check(rc)


def cache_write(k, v, k_pages, v_pages, page_table, lengths, *, counts=None, stream=None) -> None:
    """One call of CacheWriter."""
    CacheWriter(k_pages, v_pages, page_table, lengths, counts=counts)(k, v, stream=stream)


def rotary_frequencies(rotary_dim: int, *, base: float = 10000.0, scaling: dict | None = None) -> list[float]:
    """Radians per position of the rotary_dim / 2 pairs: f_i = base ** (-2 i / rotary_dim).
    `scaling` stretches them by a factor for contexts longer than trained on:

    {"type": "linear", "factor": s}: f_i / s.
    {"type": "base", "factor": s}: base * s ** (rotary_dim / (rotary_dim - 2)) for base,
        which leaves the fastest pair and divides the slowest by s.
    {"type": "parts", "factor": s, "original_tokens": n, "low": l, "high": h}: by the
        turns r_i = n f_i / (2 pi) of a pair over the original length: f_i from h turns
        on, f_i / s up to l, in between f_i g + f_i / s (1 - g), g = (r_i - l) / (h - l)
        (l = 1 and h = 32 unless given)."""
    if type(rotary_dim) is not int or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be a positive even integer")
    if not (base > 0 and math.isfinite(base)):
        raise ValueError("base must be positive")
    keys = {"linear": {"factor"}, "base": {"factor"}, "parts": {"factor", "original_tokens", "low", "high"}}
    options = dict(scaling or {})
    kind = options.pop("type", None)
    if scaling is not None:
        if kind not in keys:
            raise ValueError("scaling must have a type: 'linear', 'base' or 'parts'")
        if set(options) - keys[kind]:
            raise ValueError(f"scaling of type {kind!r} takes {sorted(keys[kind])}")
        if not (options.get("factor", 0) > 0 and math.isfinite(options["factor"])):
            raise ValueError("scaling needs a positive factor")
    factor = options.get("factor", 1.0)
    if kind == "base":
        if rotary_dim == 2:
            raise ValueError("scaling of the base needs two pairs at least")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if kind == "linear":
        return [x / factor for x in f]
    if kind == "parts":
        n, low, high = options.get("original_tokens", 0), options.get("low", 1.0), options.get("high", 32.0)
        if not (n > 0 and 0 <= low < high):
            raise ValueError("scaling by parts needs positive original_tokens and 0 <= low < high")
        keep = [min(1.0, max(0.0, (n * x / (2.0 * math.pi) - low) / (high - low))) for x in f]
        return [x * g + x / factor * (1.0 - g) for x, g in zip(f, keep)]
    return f


class Rotary:
    """Rotary positions of rows of head_dim columns, of which the first rotary_dim
    (all, unless given) are turned in pairs: columns i and i + rotary_dim / 2, or
    with `interleaved` 2 i and 2 i + 1. Pair i at position p turns by the angle
    p * frequencies[i] and is scaled by `magnitude`. Frequencies: numbers in
    radians per position, or those of rotary_frequencies(rotary_dim, base=,
    scaling=). They are kept on `device`."""

    def __init__(self, head_dim: int, *, rotary_dim: int | None = None, base: float = 10000.0, scaling: dict | None = None,
                 frequencies=None, interleaved: bool = False, magnitude: float = 1.0, device="cuda"):
        torch = _torch()
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if type(head_dim) is not int or type(rotary_dim) is not int or not 2 <= rotary_dim <= head_dim or rotary_dim % 2:
            raise ValueError("rotary_dim must be even, from 2 to head_dim")
        if not math.isfinite(magnitude):
            raise ValueError("magnitude must be finite")
        if frequencies is None:
            frequencies = rotary_frequencies(rotary_dim, base=base, scaling=scaling)
        elif scaling is not None:
            raise ValueError("pass either frequencies or scaling, not both")
        frequencies = torch.as_tensor(frequencies, dtype=torch.float64)
        if tuple(frequencies.shape) != (rotary_dim // 2,):
            raise ValueError("frequencies must be rotary_dim / 2 numbers")
        on_host = frequencies.device.type == "cpu"
        if on_host and not bool(torch.isfinite(frequencies).all()):
            raise ValueError("frequencies must be finite")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("device must be a GPU")
        self._shape, self._interleaved, self._magnitude = (head_dim, rotary_dim), bool(interleaved), float(magnitude)
        # (its own copy: a program may go on with its tensor)
        self._frequencies = frequencies.detach().to(device, copy=True).contiguous()
        # (a copy from a device has ended when what was copied is looked at: calls may run on any stream)
        if not on_host and not bool(torch.isfinite(self._frequencies).all()):
            raise ValueError("frequencies must be finite")
        self._kept = _Kept(torch, self._frequencies)
        self._torch, self._device = torch, self._frequencies.device
        p = RotaryParams()
        self._lib = lib()
        self._lib.ofh_rotary_params_init(ctypes.addressof(p))
        p.head_dim = head_dim
        self._fields(p.rotary)
        self._params = bytes(p)
        self._held = None  # (layout of the last call, its parameters): calls are laid out alike

    # (not to be assigned: calls, also of a CacheAppender, go by what they were when it was made)
    head_dim = property(lambda self: self._shape[0])
    rotary_dim = property(lambda self: self._shape[1])
    interleaved = property(lambda self: self._interleaved)
    magnitude = property(lambda self: self._magnitude)
    frequencies = property(lambda self: self._frequencies, doc="float64 on the device: the tensor that calls read")

    def _fields(self, r: RotaryFields) -> None:
        r.frequencies, r.rotary_dim = self._frequencies.data_ptr(), self.rotary_dim
        r.interleaved, r.magnitude = int(self.interleaved), self.magnitude

    def __call__(self, x, *, offset: int = 0, positions=None, lengths=None, transpose: bool = False, out=None,
                 stream=None):
        """x: [B,H,T,D] (f32/bf16/f16, last axis contiguous). Token t of a sequence
        is at position offset + t; or positions[t] or positions[b, t] (int32
        device [T] or [B,T]); or lengths[b] - T + t (int32 device [B]: the last
        T of lengths[b] tokens). `transpose` turns back: the gradient of x from
        that of the result. out: x itself, or a tensor like it elsewhere. Returns out."""
        torch, dev = self._torch, self._device
        layout = (x.shape, x.stride(), x.dtype, x.device) if isinstance(x, torch.Tensor) else None
        held = self._held
        if held is None or layout != held[0]:
            held = self._held = (layout, self._lay_out(x))
        B, H, T, D = x.shape
        p = RotaryParams.from_buffer_copy(held[1])
        if offset != 0 or type(offset) is not int:
            if type(offset) is not int or not -(1 << 31) <= offset < 1 << 31:
                raise ValueError("offset must be an integer within 32 bits")
            p.offset = offset
        if transpose:
            p.transpose = 1
        if (positions is not None) + (lengths is not None) + (offset != 0) > 1:
            raise ValueError("pass one of offset, positions and lengths")
        if positions is not None:
            _check_ints(torch, "positions", positions, (T,) if isinstance(positions, torch.Tensor) and positions.dim() == 1
                        else (B, T), dev)
            p.positions = positions.data_ptr()
            p.position_stride = positions.stride(0) if positions.dim() == 2 and B > 1 else 0
        elif lengths is not None:
            _check_ints(torch, "lengths", lengths, (B,), dev)
            p.lengths = lengths.data_ptr()
        if out is None:
            out = torch.empty((B, H, T, D), dtype=x.dtype, device=dev)
        else:
            _check_rows(torch, "out", out, 4, x.dtype, dev)
            if out.shape != x.shape:
                raise ValueError(f"out must have shape {tuple(x.shape)}")
            _check_written("out", out)
            if not out.is_contiguous():
                p.o_strides[:] = _axis_strides("out", out)
            if out.data_ptr() == x.data_ptr():
                # (axes of one element have any stride)
                if _axis_strides("out", out) != _axis_strides("x", x):
                    raise ValueError("x turned in place must keep its strides")
                p.o_strides[:] = p.x_strides[:]
        self._kept.used(stream)
        rc = _launch(torch, dev, stream, self._lib.ofh_rotary_fwd, ctypes.addressof(p), x.data_ptr(), out.data_ptr())
        if rc != OFH_SUCCESS:
            check(rc)
        return out

    def _lay_out(self, x) -> bytes:
        """Checks x and its layout; the parameters of a call with a contiguous result."""
        torch, dev = self._torch, self._device
        if not (isinstance(x, torch.Tensor) and x.dtype in _DTYPE_CODES and _is_rows(torch, x, x.dtype, dev)):
            _check_rows(torch, "x", x, 4, None, dev)
        if x.shape[3] != self.head_dim:
            raise ValueError(f"x must have rows of {self.head_dim} columns")
        p = RotaryParams.from_buffer_copy(self._params)
        p.batch, p.heads, p.tokens, p.dtype = *x.shape[:3], _DTYPE_CODES[x.dtype]
        if not x.is_contiguous():
            p.x_strides[:] = _axis_strides("x", x)
        return bytes(p)


class CacheAppender:
    """CacheWriter with the rotation on the way: K rows are turned by their
    positions into the pages, V rows copied, and the queries of the same tokens
    turned too. One launch for what follows a layer's projections in a decode
    step. Position and place of token t < counts[b] of sequence b are
    CacheWriter's, lengths[b] - counts[b] + t."""

    def __init__(self, k_pages, v_pages, page_table, lengths, rotary: Rotary, *, counts=None):
        writer = CacheWriter(k_pages, v_pages, page_table, lengths, counts=counts)
        if not isinstance(rotary, Rotary) or rotary.head_dim != k_pages.shape[3] or rotary._device != k_pages.device:
            raise ValueError("rotary must be a Rotary of the cache's head_dim on its device")
        self._writer, self._rotary = writer, rotary
        p = CacheAppendParams()
        L = lib()
        L.ofh_cache_append_params_init(ctypes.addressof(p))
        p.cache = CacheWriteParams.from_buffer_copy(writer._params)
        rotary._fields(p.rotary)
        self._params = bytes(p)
        self._append = L.ofh_cache_append
        self._held = None  # (layout of the last call, its parameters): steps are laid out alike

    def __call__(self, k, v, q=None, *, q_out=None, stream=None):
        """k: [B,Hkv,T,D], v: [B,Hkv,T,Dv], the (padded) new rows; q: [B,H,T,D].
        Returns the turned q (q_out: q itself, or a tensor like it), whose rows at
        t >= counts[b] are 0; None without q."""
        w = self._writer
        torch, dev = w._torch, w._device
        tensor = torch.Tensor
        layout = None
        if isinstance(k, tensor) and isinstance(v, tensor) and (q is None or isinstance(q, tensor)):
            layout = (k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype, v.device)
            if q is not None:
                layout += (q.shape, q.stride(), q.dtype, q.device)
        held = self._held
        if held is not None and layout == held[0]:
            p = held[1]
        else:
            p = self._lay_out(k, v, q)
            self._held = (layout, p)
        q_ptr = out_ptr = None
        if q is not None:
            q_ptr = q.data_ptr()
            if q_out is None:
                q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
            else:
                p = self._lay_out_result(p, q, q_out)
            out_ptr = q_out.data_ptr()
        elif q_out is not None:
            raise ValueError("q_out needs q")
        self._rotary._kept.used(stream)
        rc = _launch(torch, dev, stream, self._append, p, k.data_ptr(), v.data_ptr(), q_ptr, *w._ptrs, out_ptr)
        if rc != OFH_SUCCESS:
            check(rc)
        return q_out

    def _lay_out(self, k, v, q) -> bytes:
        """Checks the rows and their layout; the parameters of a call with a contiguous q_out."""
        w = self._writer
        T = w._check_new(k, v)
        B, _, D, _ = w._row
        p = CacheAppendParams.from_buffer_copy(self._params)
        p.cache.tokens = T
        if not k.is_contiguous():
            p.cache.k_strides[:] = _axis_strides("k", k)
        if not v.is_contiguous():
            p.cache.v_strides[:] = _axis_strides("v", v)
        if q is not None:
            if not _is_rows(w._torch, q, w._dtype, w._device):
                _check_rows(w._torch, "q", q, 4, w._dtype, w._device)
            if q.shape != (B, q.shape[1], T, D):
                raise ValueError(f"q must be {(B, 'H', T, D)}")
            p.heads = q.shape[1]
            if not q.is_contiguous():
                p.q_strides[:] = _axis_strides("q", q)
        return bytes(p)

    def _lay_out_result(self, params: bytes, q, q_out) -> bytes:
        w = self._writer
        _check_rows(w._torch, "q_out", q_out, 4, w._dtype, w._device)
        if q_out.shape != q.shape:
            raise ValueError(f"q_out must have shape {tuple(q.shape)}")
        _check_written("q_out", q_out)
        p = CacheAppendParams.from_buffer_copy(params)
        if not q_out.is_contiguous():
            p.o_strides[:] = _axis_strides("q_out", q_out)
        if q_out.data_ptr() == q.data_ptr():
            # (axes of one element have any stride)
            if _axis_strides("q_out", q_out) != _axis_strides("q", q):
                raise ValueError("q turned in place must keep its strides")
            p.o_strides[:] = p.q_strides[:]
        return bytes(p)


def cache_append(k, v, k_pages, v_pages, page_table, lengths, rotary: Rotary, *, q=None, q_out=None, counts=None,
                 stream=None):
    """One call of CacheAppender."""
    return CacheAppender(k_pages, v_pages, page_table, lengths, rotary, counts=counts)(k, v, q, q_out=q_out, stream=stream)


def _page_numbers(torch, name, x, pages):
    """x, a row of integers on the host, as contiguous int32."""
    if not isinstance(x, torch.Tensor):
        try:
            x = list(x)
            if set(map(type, x)) - {int}:  # integers of other kinds, but no truth values
                if any("bool" in str(getattr(i, "dtype", type(i))) for i in x):
                    raise TypeError
                x = [operator.index(i) for i in x]
        except TypeError:
            raise ValueError(f"{name} must be a row of integers on the host") from None
        try:
            x = torch.tensor(x, dtype=torch.int64)
        except (OverflowError, RuntimeError, ValueError):  # past 64 bits
            raise ValueError(f"{name}: copied pages must be within the pool") from None
    if x.dim() != 1 or x.device.type != "cpu" or x.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be a row of integers on the host")
    if x.dtype == torch.int64:
        if x.numel() and (int(x.min()) < 0 or int(x.max()) >= pages):
            raise ValueError(f"{name}: copied pages must be within the pool")
        x = x.to(torch.int32)
    return x if x.is_contiguous() else x.contiguous()


def copy_pages(pools, src, dst, *, stream=None) -> None:
    """Copies pages src[i] -> dst[i] of every pool. pools: device tensors
    [P, ...] of one shape and dtype whose pages are contiguous; src, dst: page
    numbers on the host (int32 CPU tensors, or sequences of integers), read
    before the call returns. Raises for pages outside the pools, a page twice in
    dst, or a page in both src and dst."""
    torch = _torch()
    pools = list(pools)
    if not pools or not all(isinstance(t, torch.Tensor) for t in pools):
        raise ValueError("pools must be tensors [P, ...]")
    first = pools[0]
    shape, strides, dtype, dev = first.shape, first.stride(), first.dtype, first.device
    if len(shape) < 2 or 0 in shape or dev.type != "cuda":
        raise ValueError("pools must be GPU tensors [P, ...]")
    for t in pools:
        if t.shape != shape or t.dtype != dtype or t.device != dev or t.stride() != strides:
            raise ValueError("pools must share shape, dtype, strides and device")
    page = 1
    for size, stride in zip(reversed(shape[1:]), reversed(strides[1:])):
        if size > 1 and stride != page:
            raise ValueError("pools: pages must be contiguous")
        page *= size
    between = strides[0] if shape[0] > 1 else page
    if between < page:
        raise ValueError("pools: pages must not overlap")

    src, dst = _page_numbers(torch, "src", src, shape[0]), _page_numbers(torch, "dst", dst, shape[0])
    count, size = src.numel(), first.element_size()
    if count != dst.numel():
        raise ValueError("src and dst must have the same length")
    addresses = (ctypes.c_void_p * len(pools))(*[t.data_ptr() for t in pools])
    rc = _launch(torch, dev, stream, lib().ofh_cache_copy_pages, addresses, len(pools), shape[0], page * size,
                 between * size, src.data_ptr(), dst.data_ptr(), count)
    if rc != OFH_SUCCESS:
        check(rc)


# Tile heuristic and layout choice of the reference wrapper
# (python/onednn_flash_tf/ops.py:13-47). On the GPU the kernel's own tiles are
# used; these values are accepted, validated and otherwise advisory.
def select_tile_sizes(query_tokens: int, key_tokens: int | None = None) -> tuple[int, int]:
    if query_tokens <= 0:
        raise ValueError("query_tokens must be positive")
    key_tokens = query_tokens if key_tokens is None else key_tokens
    if key_tokens <= 0:
        raise ValueError("key_tokens must be positive")
    if query_tokens <= 64 and key_tokens <= 64:
        return min(64, query_tokens), min(64, key_tokens)
    return min(32, query_tokens), min(64, key_tokens)


def select_qk_tile_layout(query_tokens: int, key_tokens: int | None = None) -> str:
    if query_tokens <= 0:
        raise ValueError("query_tokens must be positive")
    key_tokens = query_tokens if key_tokens is None else key_tokens
    if key_tokens <= 0:
        raise ValueError("key_tokens must be positive")
    return "strided_k"


def onednn_flash_attention(q, k, v, *, causal: bool = True, query_block_size: int | None = None,
                           key_block_size: int | None = None, use_onednn: bool = True,
                           tile_kernel: str = "onednn", qk_tile_layout: str | None = None,
                           op_path=None):
    """Same keywords and checks as the reference wrapper (ops.py:63-115); scale
    is 1/sqrt(D) as in the op (onednn_flash_attention_op.cc:91). Runs the HIP
    kernels on device tensors."""
    del use_onednn, op_path
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("q and k must be rank 4 [B,H,T,D] tensors")
    if query_block_size is None or key_block_size is None:
        hq, hk = select_tile_sizes(int(q.shape[2]), int(k.shape[2]))
        query_block_size = hq if query_block_size is None else query_block_size
        key_block_size = hk if key_block_size is None else key_block_size
    if qk_tile_layout is None:
        qk_tile_layout = select_qk_tile_layout(int(q.shape[2]), int(k.shape[2]))
    if qk_tile_layout not in {"strided_k", "copied_transposed", "brgemm_transformed_k"}:
        raise ValueError("qk_tile_layout must be 'strided_k', 'copied_transposed', or 'brgemm_transformed_k'")
    if tile_kernel not in {"onednn", "onednn_brgemm"}:
        raise ValueError("tile_kernel must be 'onednn' or 'onednn_brgemm'")
    if tile_kernel == "onednn_brgemm" and qk_tile_layout == "strided_k":
        raise ValueError("tile_kernel='onednn_brgemm' does not support qk_tile_layout='strided_k'; use 'copied_transposed' or 'brgemm_transformed_k'")
    if query_block_size <= 0 or key_block_size <= 0:
        raise ValueError("block sizes must be positive")
    return attention_fwd(q, k, v, scale=1.0 / math.sqrt(q.shape[3]), causal=causal)
