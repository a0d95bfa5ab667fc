"""The paged KV cache held in 4 bits on MI355X: its layout, its writer and its
reader (``decode_fp4`` holds the attention over it).

The 4-bit sibling of ``paged_cache``: the same block tables, lengths and prefix
sums (the format of the reference's paged kernels, harsh-vsingh/triton-kernels
kernels/decode.py:130-149), values in OCP MX FP4.  One cache (K or V) is an
:class:`Fp4Cache` of two contiguous uint8 tensors::

    codes   [pages, KVH, page, D / 2]     value d: nibble d % 2 (0 low) of byte d // 2
    scales  [pages, KVH, page, D / 32]    2 ** (scale - 127) of block d // 32; 255: NaN

A nibble is E2M1 (sign, two exponent bits, one of mantissa: 0 .5 1 1.5 2 3 4 6).
D is 64, 128 or 256; 4.25 bits a value.  A page holds the rows of each kv head
together, since the attention reads one head at a time: 16 rows of 128 dims are
1 KB of codes.  gfx950 makes two values per instruction, scale included, so
readers pay next to nothing for the format and add no rounding of their own.

* :func:`paged_kv_append_fp4` - quantise new rows into the caches;
* :func:`paged_kv_gather_fp4` - rows back in 16 or 32 bits, token-major, the
  K/V that ``flash_attention_v2`` takes for a prefill chunk over the context;
* :func:`allocate_fp4_cache` - an empty cache.

Quantisation of a block of 32: the least power of two at which the largest
value is at most 6 after rounding, each value to the nearest code, ties to even.
Powers are kept in 2 ** -23 ... 2 ** 13 for fp16 rows and 2 ** -100 ... 2 ** 125
for bf16 and fp32 rows, so that every cached value is exact in the rows' type;
past 49152 fp16 rows saturate.  Inside that range a value is off by at most 1/5 of
its block's largest (5 steps become 4).  A block with an infinity or NaN is NaN.

Tables, lengths, starts and prefix sums are int32; other integer types are
converted, int64 saturating, so that what is outside a pool stays outside.  The
computation runs in ``libfa2.so`` (include/fa2_ops.h); no fallback.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _ops
from ._launch import DTYPES, aligned, ext, in_32_bits, index_tensor, stride_of, table

# As kernels/decode.py: the C++ extension launches when it is built.
USE_EXT = True

FP4_HEAD_DIMS = (64, 128, 256)


class Fp4Cache(NamedTuple):
    """K or V in 4 bits; every entry point also takes a plain pair."""

    codes: torch.Tensor
    scales: torch.Tensor


def allocate_fp4_cache(num_pages: int, page_size: int, kv_heads: int, head_dim: int,
                       device="cuda") -> Fp4Cache:
    """A cache of zeros (K and V take one each)."""
    if head_dim not in FP4_HEAD_DIMS:
        raise ValueError(f"allocate_fp4_cache: head_dim {head_dim} not supported "
                         f"(supported: {FP4_HEAD_DIMS})")
    if num_pages <= 0 or page_size <= 0 or kv_heads <= 0:
        raise ValueError("allocate_fp4_cache: sizes must be positive")
    return Fp4Cache(*(torch.zeros((num_pages, kv_heads, page_size, n), dtype=torch.uint8,
                                  device=device) for n in (head_dim // 2, head_dim // 32)))


def check_cache(name: str, k_cache, v_cache):
    """The four tensors of a K and a V cache (V may be None) after their checks."""
    kc, ks = k_cache
    vc, vs = v_cache if v_cache is not None else (None, None)
    ts = (kc, ks) if vc is None else (kc, ks, vc, vs)
    for t in ts:
        assert t.device == kc.device, "Tensors must be on the same device"
        if t.dtype != torch.uint8:
            raise TypeError(f"{name}: codes and scales must be uint8")
        if t.dim() != 4 or not t.is_contiguous():
            raise ValueError(f"{name}: codes and scales must be contiguous 4-D tensors")
    assert kc.is_cuda, "Tensors must be on a CUDA device"
    d = kc.shape[3] * 2
    if d not in FP4_HEAD_DIMS:
        raise ValueError(f"{name}: head_dim {d} not supported (supported: {FP4_HEAD_DIMS})")
    if ks.shape != (*kc.shape[:3], d // 32):
        raise ValueError(f"{name}: scales must be {(*kc.shape[:3], d // 32)}")
    if vc is not None and (vc.shape != kc.shape or vs.shape != ks.shape):
        raise ValueError(f"{name}: the K and V caches must have equal shapes")
    if 0 in kc.shape:
        raise ValueError(f"{name}: an empty cache")
    return kc, ks, vc, vs


def _check_rows(name, kc, vc, k_table, v_table, indptr, start_pos):
    """The checks that the writer and the reader share; the number of sequences."""
    has_v = vc is not None
    assert kc.device == k_table.device == indptr.device, "Tensors must be on the same device"
    if (v_table is None) == has_v:
        raise ValueError(f"{name}: pass the V arguments together")
    B = indptr.numel() - 1
    if B < 0 or k_table.dim() != 2 or k_table.shape[0] < B or (
            has_v and (v_table.dim() != 2 or v_table.shape[0] < B)):
        raise ValueError(f"{name}: the block tables need one row per sequence")
    if start_pos is not None and start_pos.numel() < B:
        raise ValueError(f"{name}: start_pos needs one entry per sequence")
    return B


def paged_kv_append_fp4(
    k_cache,
    v_cache,
    k_block_table: torch.Tensor,
    v_block_table: torch.Tensor | None,
    k_new: torch.Tensor,
    v_new: torch.Tensor | None,
    new_indptr: torch.Tensor,
    start_pos: torch.Tensor | None = None,
) -> None:
    """Quantise ``k_new`` / ``v_new`` rows into the caches, in place.

    ``k_cache`` / ``v_cache``: :class:`Fp4Cache`; ``k_new`` / ``v_new``: ``[T, KVH,
    D]`` fp16, bf16 or fp32, each with strides of its own (rows contiguous);
    ``new_indptr``: ``[B + 1]`` prefix sums over the new rows; ``start_pos``:
    ``[B]`` logical position of each sequence's first new row (``None``: 0);
    tables ``[B, width]``.  The V arguments may all be ``None`` (K only).  Rows
    whose logical page is past the table width, or whose table entry is outside
    the cache, are not written; no two rows of a call may share a place.
    """
    name = "paged_kv_append_fp4"
    x = ext() if USE_EXT else None
    if x is not None:
        rc = x.fp4_append(*k_cache, *(v_cache if v_cache is not None else (None, None)),
                          k_block_table, v_block_table, k_new, v_new, new_indptr, start_pos)
        if rc == 0:
            return
        if rc > 0:
            raise _ops.OpsError(name, rc)
    # (the extension makes these checks itself and leaves the errors to them)
    kc, ks, vc, vs = check_cache(name, k_cache, v_cache)
    if (v_new is None) != (vc is None):
        raise ValueError(f"{name}: pass the V arguments together")
    B = _check_rows(name, kc, vc, k_block_table, v_block_table, new_indptr, start_pos)
    if k_new.dtype not in DTYPES:
        raise TypeError(f"{name}: unsupported dtype {k_new.dtype} (float16, bfloat16, float32)")
    H, D = kc.shape[1], kc.shape[3] * 2
    assert k_new.device == kc.device and (v_new is None or v_new.device == kc.device), (
        "Tensors must be on the same device")
    if k_new.dim() != 3 or k_new.shape[1:] != (H, D):
        raise ValueError(f"{name}: new rows must be [T, {H}, {D}]")
    if v_new is not None and (v_new.shape != k_new.shape or v_new.dtype != k_new.dtype):
        raise ValueError(f"{name}: k_new and v_new must have equal shapes and dtypes")
    k_new = aligned(k_new)
    v_new = aligned(v_new) if v_new is not None else None
    _rows(name, "fa2_fp4_append", kc, ks, vc, vs, k_block_table, v_block_table, k_new, v_new,
          new_indptr, start_pos, B)


def paged_kv_gather_fp4(
    k_cache,
    v_cache,
    k_block_table: torch.Tensor,
    v_block_table: torch.Tensor | None,
    indptr: torch.Tensor,
    num_rows: int,
    start_pos: torch.Tensor | None = None,
    *,
    dtype: torch.dtype = torch.bfloat16,
    out=None,
):
    """Rows of the caches in ``dtype``: (k, v) ``[num_rows, KVH, D]`` each; exact in the
    type of the rows that were written, in bf16 for fp16 rows too, and in fp32.  (fp16
    rounds what bf16 or fp32 rows left outside 2 ** -24 ... 65504: to its own small
    numbers, zero or infinity.)

    Row ``indptr[b] + j`` is logical row ``start_pos[b] + j`` (``None``: from 0) of
    sequence b; with ``indptr`` as ``kv_indptr`` the result is the ragged K/V of
    ``flash_attention_v2``.  ``num_rows`` is ``indptr[B]``, which the host passes so
    that nothing waits for the device.  Rows past the table width or with a table
    entry outside the cache are zeros; rows that no sequence holds are left as
    they are in ``out`` (a pair of contiguous ``[num_rows, KVH, D]`` tensors,
    returned, whose type stands in ``dtype``'s place; ``None``: new ones, in which
    such rows hold anything).  ``v_cache`` and ``v_block_table`` may both be ``None``:
    then v is ``None``.
    """
    name = "paged_kv_gather_fp4"
    x = ext() if USE_EXT else None
    if x is not None and out is None:
        rc, k, v = x.fp4_gather(*k_cache, *(v_cache if v_cache is not None else (None, None)),
                                k_block_table, v_block_table, num_rows, dtype, indptr, start_pos)
        if rc == 0:
            return k, v
        if rc > 0:
            raise _ops.OpsError(name, rc)
    # (the extension makes these checks itself and leaves the errors to them)
    kc, ks, vc, vs = check_cache(name, k_cache, v_cache)
    B = _check_rows(name, kc, vc, k_block_table, v_block_table, indptr, start_pos)
    shape = (int(num_rows), kc.shape[1], kc.shape[3] * 2)
    if shape[0] < 0:
        raise ValueError(f"{name}: num_rows must not be negative")
    if out is None:
        if dtype not in DTYPES:
            raise TypeError(f"{name}: unsupported dtype {dtype} (float16, bfloat16, float32)")
        k = torch.empty(shape, dtype=dtype, device=kc.device)
        v = torch.empty(shape, dtype=dtype, device=kc.device) if vc is not None else None
    else:
        k, v = out
        if (v is None) != (vc is None):
            raise ValueError(f"{name}: pass the V arguments together")
        for t in (k,) if v is None else (k, v):
            assert t.device == kc.device, "Tensors must be on the same device"
            if t.dtype not in DTYPES or t.dtype != k.dtype:
                raise TypeError(f"{name}: out must be float16, bfloat16 or float32, k and v alike")
            if t.shape != shape or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{name}: out must be contiguous {list(shape)} tensors")
    if x is not None:
        _ops.check(name, x.fp4_gather_into(kc, ks, vc, vs, k_block_table, v_block_table, k, v,
                                           indptr, start_pos))
    else:
        _rows(name, "fa2_fp4_gather", kc, ks, vc, vs, k_block_table, v_block_table, k, v, indptr,
              start_pos, B)
    return k, v


def _rows(name, entry, kc, ks, vc, vs, k_table, v_table, k, v, indptr, start_pos, B):
    """The ctypes launch of the writer and the reader."""
    dev = kc.device
    ip = index_tensor(in_32_bits(indptr), dev)
    sp = index_tensor(in_32_bits(start_pos), dev) if start_pos is not None else None
    kt = table(in_32_bits(k_table), dev)
    p = _ops.Fp4RowsParams()
    p.dtype = DTYPES[k.dtype]
    p.batch, p.kv_heads, p.head_dim, p.num_rows = B, kc.shape[1], k.shape[2], k.shape[0]
    p.page_size, p.num_pages, p.table_width = kc.shape[2], kc.shape[0], kt.shape[1]
    p.k_table_stride = kt.stride(0)
    p.k_ts, p.k_hs = stride_of(k, 0), stride_of(k, 1)
    p.k, p.k_codes, p.k_scales = k.data_ptr(), kc.data_ptr(), ks.data_ptr()
    p.indptr, p.k_block_table = ip.data_ptr(), kt.data_ptr()
    if sp is not None:
        p.start_pos = sp.data_ptr()
    if vc is not None:
        vt = table(in_32_bits(v_table), dev)
        p.table_width = min(kt.shape[1], vt.shape[1])
        p.v_table_stride = vt.stride(0)
        p.v_ts, p.v_hs = stride_of(v, 0), stride_of(v, 1)
        p.v, p.v_codes, p.v_scales = v.data_ptr(), vc.data_ptr(), vs.data_ptr()
        p.v_block_table = vt.data_ptr()
    with torch.cuda.device(dev):
        _ops.call(name, entry, p, torch.cuda.current_stream().cuda_stream)
