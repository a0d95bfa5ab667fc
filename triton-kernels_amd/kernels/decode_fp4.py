"""Decode and speculative decode attention over a cache held in 4 bits, on
MI355X: ``decode_attention`` and ``speculative_decode_attention`` (their paged
layout, masks and results) with ``fp4_cache.Fp4Cache`` K and V.

* ``decode_attention_fp4``: q ``[B, QH, D]``, one query token per sequence;
* ``speculative_decode_attention_fp4``: q ``[B, QH, M, D]``, M <= 16 drafts,
  the cache's last M keys; ``causal=True`` hides from draft m the drafts after it.

``kv_indptr`` holds each sequence's length (as for the 16-bit paged calls, the
reference's kernels/decode.py:203-331 and kernels/speculative_decode.py:228-365);
lengths past the block table's width count as that.  q is fp16 or bf16: the type
of the rows that the cache was written from (``fp4_cache``), in which its values
are exact.  They are expanded in registers on their way to the MFMA, softmax
statistics are fp32, and the softmax weights enter the product with V as two
16-bit parts, so the result is the exact attention over the cached values to
within its own rounding.  A row without keys is NaN, as in the 16-bit calls.

The computation runs in ``libfa2.so`` (``fa2_fp4_decode``, include/fa2_ops.h); no
fallback.
"""

from __future__ import annotations

import torch

from . import _fa2, _ops
from ._launch import DTYPES, ext, in_32_bits, index_tensor, rows_ok, stride_of, table
from .fp4_cache import check_cache

# As kernels/decode.py: the C++ extension launches when it is built.
USE_EXT = True


def decode_attention_fp4(
    q: torch.Tensor,
    k_cache,
    v_cache,
    *,
    kv_indptr: torch.Tensor,
    k_block_table: torch.Tensor,
    v_block_table: torch.Tensor,
) -> torch.Tensor:
    """See the module docstring."""
    return _decode("decode_attention_fp4", q, k_cache, v_cache, kv_indptr, k_block_table,
                   v_block_table, False, 3)


def speculative_decode_attention_fp4(
    q: torch.Tensor,
    k_cache,
    v_cache,
    *,
    causal: bool = False,
    kv_indptr: torch.Tensor,
    k_block_table: torch.Tensor,
    v_block_table: torch.Tensor,
) -> torch.Tensor:
    """See the module docstring."""
    return _decode("speculative_decode_attention_fp4", q, k_cache, v_cache, kv_indptr,
                   k_block_table, v_block_table, bool(causal), 4)


def _decode(name, q, k_cache, v_cache, lens, k_table, v_table, causal, dims):
    x = ext() if USE_EXT else None
    if x is not None and v_cache is not None:
        rc, out = x.fp4_decode(q, *k_cache, *v_cache, lens, k_table, v_table, causal, dims)
        if rc == 0:
            return out
        if rc > 0:
            raise _ops.OpsError(name, rc)
    # (the extension makes these checks itself and leaves the errors to them)
    if q.dim() != dims:
        raise ValueError(f"{name}: q must be {'[B, QH, D]' if dims == 3 else '[B, QH, M, D]'}")
    if dims == 4:
        assert q.shape[2] <= 16, "Speculative decode is intended for small draft lengths (M <= 16)."
    if v_cache is None:
        raise ValueError(f"{name}: v_cache is missing")
    kc, ks, vc, vs = check_cache(name, k_cache, v_cache)
    assert q.device == kc.device == lens.device == k_table.device == v_table.device, (
        "Tensors must be on the same device")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"{name}: unsupported dtype {q.dtype} (float16, bfloat16)")
    B, QH, D = q.shape[0], q.shape[1], q.shape[-1]
    KVH = kc.shape[1]
    if D != kc.shape[3] * 2:
        raise ValueError(f"{name}: q's head_dim {D} is not the cache's ({kc.shape[3] * 2})")
    if QH == 0 or QH % KVH != 0:
        raise ValueError(f"{name}: q_heads ({QH}) must be a multiple of kv_heads ({KVH})")
    if (lens.numel() < B or k_table.dim() != 2 or v_table.dim() != 2 or k_table.shape[0] < B
            or v_table.shape[0] < B):
        raise ValueError(f"{name}: kv_indptr and the block tables need {B} rows")
    return _run(name, q, kc, ks, vc, vs, lens, k_table, v_table, causal)


def _run(name, q, kc, ks, vc, vs, lens, k_table, v_table, causal, workspace=None):
    """The ctypes launch; ``workspace`` (tests only) is a uint8 device buffer
    used instead of an allocation."""
    dev = q.device
    q4 = q.unsqueeze(2) if q.dim() == 3 else q
    B, QH, M, D = q4.shape
    if not rows_ok(q4) or (M > 1 and stride_of(q4, 1) != M * stride_of(q4, 2)):
        q4 = q4.clone(memory_format=torch.contiguous_format)
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    o4 = out.unsqueeze(2) if q.dim() == 3 else out
    li = index_tensor(in_32_bits(lens), dev)
    kt, vt = table(in_32_bits(k_table), dev), table(in_32_bits(v_table), dev)
    p = _ops.Fp4DecodeParams()
    p.dtype = DTYPES[q.dtype]
    p.mask = _fa2.MASK_BOTTOM_RIGHT if causal else _fa2.MASK_NONE
    p.batch, p.q_heads, p.kv_heads, p.head_dim, p.q_len = B, QH, kc.shape[1], D, M
    p.page_size, p.num_pages = kc.shape[2], kc.shape[0]
    p.table_width = min(kt.shape[1], vt.shape[1])
    p.k_table_stride, p.v_table_stride = kt.stride(0), vt.stride(0)
    for t, pre in ((q4, "q"), (o4, "o")):
        setattr(p, pre + "_sb", stride_of(t, 0))
        setattr(p, pre + "_sh", stride_of(t, 1))
        setattr(p, pre + "_ss", stride_of(t, 2 if M > 1 else 1))
    p.q, p.o = q4.data_ptr(), out.data_ptr()
    p.k_codes, p.k_scales = kc.data_ptr(), ks.data_ptr()
    p.v_codes, p.v_scales = vc.data_ptr(), vs.data_ptr()
    p.kv_lens, p.k_block_table, p.v_block_table = li.data_ptr(), kt.data_ptr(), vt.data_ptr()
    p.softmax_scale = D ** -0.5
    with torch.cuda.device(dev):
        n = _ops.decode_workspace_size(name, p)
        if n:
            ws = workspace if workspace is not None else torch.empty(n, dtype=torch.uint8,
                                                                     device=dev)
            if ws.numel() < n or ws.device != dev:
                raise ValueError(f"workspace needs {n} bytes on {dev}")
            p.workspace, p.workspace_bytes = ws.data_ptr(), n
        _ops.call(name, "fa2_fp4_decode", p, torch.cuda.current_stream().cuda_stream)
    return out
