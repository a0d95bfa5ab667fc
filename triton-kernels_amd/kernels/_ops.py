"""ctypes binding of the operators around the attention (include/fa2_ops.h):
query/key norms with rotation and the paged cache held in 4 bits.

They live in ``libfa2.so`` next to the attention (``_fa2``), which loads it;
there is no fallback.
"""

from __future__ import annotations

import ctypes
import threading

from . import _fa2

# Every symbol include/fa2_ops.h declares.
EXPORTS = ("fa2_norm_rope", "fa2_fp4_append", "fa2_fp4_gather", "fa2_fp4_decode_workspace_size",
           "fa2_fp4_decode", "fa2_ops_params_size")


def _fields(*groups):
    return [(n, t) for t, names in groups for n in names.split()]


_I32, _I64, _PTR = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p


class NormRopeParams(ctypes.Structure):
    """Mirror of ``struct fa2_norm_rope_params``."""

    _fields_ = _fields(
        (_I32, "dtype weight_dtype interleaved"), (ctypes.c_float, "eps"),
        (_I64, "tokens q_heads kv_heads head_dim rotary_dim positions rope_stride q_rows k_rows "
               "q_sb q_sh q_ss k_sb k_sh k_ss qo_sb qo_sh qo_ss ko_sb ko_sh ko_ss"),
        (_PTR, "q k q_out k_out q_weight k_weight rope position"), (_I32, "position_64 reserved0"))


class Fp4RowsParams(ctypes.Structure):
    """Mirror of ``struct fa2_fp4_rows_params``."""

    _fields_ = _fields(
        (_I32, "dtype reserved0"),
        (_I64, "batch kv_heads head_dim num_rows page_size num_pages table_width k_table_stride "
               "v_table_stride k_ts k_hs v_ts v_hs"),
        (_PTR, "k v k_codes k_scales v_codes v_scales indptr start_pos k_block_table "
               "v_block_table"))


class Fp4DecodeParams(ctypes.Structure):
    """Mirror of ``struct fa2_fp4_decode_params``."""

    _fields_ = _fields(
        (_I32, "dtype mask"),
        (_I64, "batch q_heads kv_heads head_dim q_len page_size num_pages table_width "
               "k_table_stride v_table_stride q_sb q_sh q_ss o_sb o_sh o_ss"),
        (_PTR, "q o k_codes k_scales v_codes v_scales kv_lens k_block_table v_block_table"),
        (ctypes.c_float, "softmax_scale"), (_I32, "reserved0"), (_PTR, "workspace"),
        (ctypes.c_size_t, "workspace_bytes"))


_PARAMS = (NormRopeParams, Fp4RowsParams, Fp4DecodeParams)
_lib = None
_lock = threading.Lock()


def lib():
    """libfa2.so with these entry points' signatures set."""
    global _lib
    if _lib is None:
        with _lock:
            if _lib is None:
                L = _fa2.lib()
                L.fa2_ops_params_size.argtypes = [ctypes.c_int]
                L.fa2_ops_params_size.restype = ctypes.c_size_t
                for i, p in enumerate(_PARAMS):
                    if L.fa2_ops_params_size(i) != ctypes.sizeof(p):
                        raise RuntimeError("libfa2.so: parameter struct layout mismatch with the "
                                           f"binding ({p.__name__})")
                for name, p in (("fa2_norm_rope", NormRopeParams),
                                ("fa2_fp4_append", Fp4RowsParams),
                                ("fa2_fp4_gather", Fp4RowsParams),
                                ("fa2_fp4_decode", Fp4DecodeParams)):
                    fn = getattr(L, name)
                    fn.argtypes = [ctypes.POINTER(p), ctypes.c_void_p]
                    fn.restype = ctypes.c_int
                L.fa2_fp4_decode_workspace_size.argtypes = [ctypes.POINTER(Fp4DecodeParams),
                                                            ctypes.POINTER(ctypes.c_size_t)]
                L.fa2_fp4_decode_workspace_size.restype = ctypes.c_int
                _lib = L
    return _lib


class OpsError(_fa2.Fa2Error):
    """A status of one of these entry points, named after the operator."""

    def __init__(self, name: str, code: int):
        msg = lib().fa2_strerror(code).decode()
        RuntimeError.__init__(self, f"{name}: {msg} (fa2 status {code})")
        self.code = code


def check(name: str, rc: int) -> None:
    if rc != 0:
        raise OpsError(name, rc)


def call(name: str, entry: str, p, stream: int) -> None:
    """Enqueue ``entry`` on the HIP stream ``stream``."""
    check(name, getattr(lib(), entry)(ctypes.byref(p), ctypes.c_void_p(stream)))


def decode_workspace_size(name: str, p: Fp4DecodeParams) -> int:
    n = ctypes.c_size_t(0)
    check(name, lib().fa2_fp4_decode_workspace_size(ctypes.byref(p), ctypes.byref(n)))
    return n.value
