"""The paged cache of latent attention on MI355X: its layout and its writer
(``latent_decode`` and ``latent_attention`` hold the attention).

A token's keys and values of all heads come from one row: a latent vector of
``latent_dim`` values, normalised, and a key part of 64 values that all heads share,
rotated to the token's position::

    cache  [pages, page_size, latent_dim + 64]   fp16 or bf16, contiguous

``latent_dim`` is 256 or 512.  Block tables, lengths and prefix sums are those of the
16-bit caches (the format of the reference's paged kernels,
harsh-vsingh/triton-kernels kernels/decode.py:130-149).  The computation runs in
``libfa2.so`` (``fa2_latent_append``, include/fa2_latent.h); no fallback, and no
backward pass, like the rest of the package.
"""

from __future__ import annotations

import torch

from . import _latent, _ops
from ._launch import DTYPES, aligned, ext, in_32_bits, index_tensor, stride_of, table

# As kernels/decode.py: the C++ extension launches when it is built.
USE_EXT = True

HALF = (torch.float16, torch.bfloat16)


def check_latent_dim(name: str, latent_dim: int, width: int) -> None:
    if latent_dim not in _latent.LATENT_DIMS or width != latent_dim + _latent.ROPE_DIM:
        raise ValueError(f"{name}: rows of {width} values with latent_dim {latent_dim} are not "
                         f"supported (latent_dim {_latent.LATENT_DIMS}, "
                         f"{_latent.ROPE_DIM} more a row)")


def allocate_latent_cache(num_pages: int, page_size: int, latent_dim: int,
                          dtype: torch.dtype = torch.bfloat16, device="cuda") -> torch.Tensor:
    """A cache of zeros."""
    name = "allocate_latent_cache"
    check_latent_dim(name, latent_dim, latent_dim + _latent.ROPE_DIM)
    if dtype not in HALF:
        raise TypeError(f"{name}: unsupported dtype {dtype} (float16, bfloat16)")
    if num_pages <= 0 or page_size <= 0:
        raise ValueError(f"{name}: sizes must be positive")
    return torch.zeros((num_pages, page_size, latent_dim + _latent.ROPE_DIM), dtype=dtype,
                       device=device)


def check_cache(name: str, cache: torch.Tensor) -> None:
    assert cache.is_cuda, "Tensors must be on a CUDA device"
    if cache.dtype not in HALF:
        raise TypeError(f"{name}: unsupported dtype {cache.dtype} (float16, bfloat16)")
    if cache.dim() != 3 or not cache.is_contiguous() or cache.data_ptr() % 16:
        raise ValueError(f"{name}: the cache must be a contiguous [pages, page_size, width] tensor "
                         "from a 16-byte boundary")
    if 0 in cache.shape:
        raise ValueError(f"{name}: an empty cache")


def paged_latent_append(
    cache: torch.Tensor,
    block_table: torch.Tensor,
    rows: torch.Tensor,
    new_indptr: torch.Tensor,
    weight: torch.Tensor,
    rope_table: torch.Tensor,
    start_pos: torch.Tensor | None = None,
    *,
    eps: float = 1e-6,
    interleaved: bool = False,
    return_rows: bool = False,
):
    """Finish new rows and write them into the cache, in place.

    ``rows`` ``[T, latent_dim + 64]`` (any row stride whose rows start on 16 bytes, such as
    a view of a fused projection's output; other tensors are copied first) holds the
    projections ``(c, r)`` of the new tokens, ``new_indptr`` ``[B + 1]`` prefix sums over
    them, ``start_pos`` ``[B]`` the logical position of each sequence's first new row
    (``None``: 0), ``block_table`` ``[B, width]`` its pages.  What is written is
    ``c * rsqrt(mean(c ** 2) + eps) * weight`` and r rotated to the row's position, as
    :func:`qk_norm_rope` rotates (``interleaved``: neighbouring pairs), with
    ``rope_table`` float32 ``[positions, 64]`` from :func:`build_rope_table`; computed in
    fp32, rounded once.  ``weight``: ``[latent_dim]`` of the rows' type or float32.

    Rows whose logical page is past the table, or whose table entry is outside the
    cache, are not written; a position outside the rope table makes the row NaN; no two
    rows of a call may share a place.  With ``return_rows`` the finished rows are
    returned, contiguous ``[T, latent_dim + 64]`` (those that no sequence holds are
    anything): what a prefill expands to keys and values.
    """
    name = "paged_latent_append"
    x = ext() if USE_EXT else None
    if x is not None:
        rc, out = x.latent_append(cache, block_table, rows, new_indptr, weight, rope_table,
                                  start_pos, eps, interleaved, return_rows)
        if rc == 0:
            return out
        if rc > 0:
            raise _ops.OpsError(name, rc)
    # (the extension makes these checks itself and leaves the errors to them)
    check_cache(name, cache)
    dev, width = cache.device, cache.shape[2]
    latent = width - _latent.ROPE_DIM
    check_latent_dim(name, latent, width)
    assert all(t.device == dev for t in (block_table, rows, new_indptr, weight, rope_table)) and (
        start_pos is None or start_pos.device == dev), "Tensors must be on the same device"
    if rows.dtype != cache.dtype:
        raise TypeError(f"{name}: rows must be {cache.dtype}, as the cache")
    if rows.dim() != 2 or rows.shape[1] != width:
        raise ValueError(f"{name}: rows must be [T, {width}]")
    if weight.dtype not in (rows.dtype, torch.float32):
        raise TypeError(f"{name}: weight must be {rows.dtype} or torch.float32")
    if weight.shape != (latent,):
        raise ValueError(f"{name}: weight must be [{latent}]")
    if rope_table.dtype != torch.float32 or rope_table.dim() != 2:
        raise TypeError(f"{name}: rope_table must be float32 [positions, {_latent.ROPE_DIM}]")
    if rope_table.shape[1] != _latent.ROPE_DIM:
        raise ValueError(f"{name}: rope_table must be [positions, {_latent.ROPE_DIM}]")
    if not eps >= 0:
        raise ValueError(f"{name}: eps must not be negative")
    B = new_indptr.numel() - 1
    if B < 0 or block_table.dim() != 2 or block_table.shape[0] < B:
        raise ValueError(f"{name}: the block table needs one row per sequence")
    if start_pos is not None and start_pos.numel() < B:
        raise ValueError(f"{name}: start_pos needs one entry per sequence")
    rows = aligned(rows)
    weight, rope_table = (
        t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(
            memory_format=torch.contiguous_format) for t in (weight, rope_table))
    ip, bt = index_tensor(in_32_bits(new_indptr), dev), table(in_32_bits(block_table), dev)
    sp = index_tensor(in_32_bits(start_pos), dev) if start_pos is not None else None
    out = torch.empty(rows.shape, dtype=rows.dtype, device=dev) if return_rows else None
    p = _latent.LatentAppendParams()
    p.dtype, p.weight_dtype = DTYPES[rows.dtype], DTYPES[weight.dtype]
    p.interleaved, p.eps = int(bool(interleaved)), float(eps)
    p.batch, p.num_rows, p.latent_dim, p.rope_dim = B, rows.shape[0], latent, _latent.ROPE_DIM
    p.page_size, p.num_pages = cache.shape[1], cache.shape[0]
    p.table_width, p.table_stride = bt.shape[1], bt.stride(0)
    p.positions, p.rope_stride, p.x_ts = rope_table.shape[0], _latent.ROPE_DIM, stride_of(rows, 0)
    p.x, p.cache, p.weight = rows.data_ptr(), cache.data_ptr(), weight.data_ptr()
    p.rope, p.indptr, p.block_table = rope_table.data_ptr(), ip.data_ptr(), bt.data_ptr()
    if sp is not None:
        p.start_pos = sp.data_ptr()
    if out is not None:
        p.rows_out = out.data_ptr()
    with torch.cuda.device(dev):
        _latent.call(name, "fa2_latent_append", p, torch.cuda.current_stream().cuda_stream)
    return out
