"""ctypes binding of latent attention and of attention for trees of drafts
(include/fa2_latent.h).

They live in ``libfa2.so`` next to the attention (``_fa2``), which loads it;
there is no fallback.
"""

from __future__ import annotations

import ctypes
import threading

from . import _fa2
from ._ops import OpsError, _fields

# Every symbol include/fa2_latent.h declares.
EXPORTS = ("fa2_latent_append", "fa2_latent_decode_workspace_size", "fa2_latent_decode",
           "fa2_latent_prefill_workspace_size", "fa2_latent_prefill",
           "fa2_tree_decode_workspace_size", "fa2_tree_decode", "fa2_latent_params_size")

MASK_TREE = 3
TREE_MAX = 64
LATENT_DIMS = (256, 512)
ROPE_DIM = 64

_I32, _I64, _PTR = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p
_END = ((ctypes.c_float, "softmax_scale"), (_I32, "reserved0"), (_PTR, "workspace"),
        (ctypes.c_size_t, "workspace_bytes"))


class LatentAppendParams(ctypes.Structure):
    """Mirror of ``struct fa2_latent_append_params``."""

    _fields_ = _fields(
        (_I32, "dtype weight_dtype interleaved"), (ctypes.c_float, "eps"),
        (_I64, "batch num_rows latent_dim rope_dim page_size num_pages table_width table_stride "
               "positions rope_stride x_ts"),
        (_PTR, "x rows_out cache weight rope indptr start_pos block_table"))


class LatentDecodeParams(ctypes.Structure):
    """Mirror of ``struct fa2_latent_decode_params``."""

    _fields_ = _fields(
        (_I32, "dtype mask"),
        (_I64, "batch q_heads q_len latent_dim rope_dim page_size num_pages table_width "
               "table_stride q_sb q_sh q_ss o_sb o_sh o_ss tree_sb tree_sr"),
        (_PTR, "q o cache kv_lens block_table tree"), *_END)


class TreeDecodeParams(ctypes.Structure):
    """Mirror of ``struct fa2_tree_decode_params``."""

    _fields_ = _fields(
        (_I32, "layout dtype"),
        (_I64, "batch q_heads kv_heads head_dim q_len kv_len q_sb q_sh q_ss k_sb k_sh k_ss v_sb "
               "v_sh v_ss o_sb o_sh o_ss page_size table_width k_table_stride v_table_stride "
               "tree_sb tree_sr"),
        (_PTR, "q k v o kv_indptr k_block_table v_block_table tree"), *_END)


class LatentPrefillParams(ctypes.Structure):
    """Mirror of ``struct fa2_latent_prefill_params``."""

    _fields_ = _fields(
        (_I32, "layout dtype mask reserved0"),
        (_I64, "batch heads head_dim rope_dim q_len kv_len q_sb q_sh q_ss k_sb k_sh k_ss v_sb "
               "v_sh v_ss o_sb o_sh o_ss kr_sb kr_ss"),
        (_PTR, "q k kr v o q_indptr kv_indptr"), (ctypes.c_float, "softmax_scale"),
        (_I32, "reserved1"), *_END[2:])


_PARAMS = (LatentAppendParams, LatentDecodeParams, TreeDecodeParams, LatentPrefillParams)
_lib = None
_lock = threading.Lock()


def lib():
    """libfa2.so with these entry points' signatures set."""
    global _lib
    if _lib is None:
        with _lock:
            if _lib is None:
                L = _fa2.lib()
                L.fa2_latent_params_size.argtypes = [ctypes.c_int]
                L.fa2_latent_params_size.restype = ctypes.c_size_t
                for i, p in enumerate(_PARAMS):
                    if L.fa2_latent_params_size(i) != ctypes.sizeof(p):
                        raise RuntimeError("libfa2.so: parameter struct layout mismatch with the "
                                           f"binding ({p.__name__})")
                for name, p in (("fa2_latent_append", LatentAppendParams),
                                ("fa2_latent_decode", LatentDecodeParams),
                                ("fa2_tree_decode", TreeDecodeParams),
                                ("fa2_latent_prefill", LatentPrefillParams)):
                    fn = getattr(L, name)
                    fn.argtypes = [ctypes.POINTER(p), ctypes.c_void_p]
                    fn.restype = ctypes.c_int
                    if name != "fa2_latent_append":
                        fn = getattr(L, name + "_workspace_size")
                        fn.argtypes = [ctypes.POINTER(p), ctypes.POINTER(ctypes.c_size_t)]
                        fn.restype = ctypes.c_int
                _lib = L
    return _lib


def check(name: str, rc: int) -> None:
    if rc != 0:
        raise OpsError(name, rc)


def call(name: str, entry: str, p, stream: int) -> None:
    """Enqueue ``entry`` on the HIP stream ``stream``."""
    check(name, getattr(lib(), entry)(ctypes.byref(p), ctypes.c_void_p(stream)))


def workspace_size(name: str, entry: str, p) -> int:
    n = ctypes.c_size_t(0)
    check(name, getattr(lib(), entry + "_workspace_size")(ctypes.byref(p), ctypes.byref(n)))
    return n.value
