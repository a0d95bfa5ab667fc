"""``tree_decode_attention`` on MI355X: attention of drafts that form a tree, over a
dense, ragged or paged 16-bit K/V cache.

The sibling of ``speculative_decode_attention`` (the reference's
kernels/speculative_decode.py:228-365) for drafts that are alternatives of one another:
M <= 64 query tokens per sequence, whose keys are the cache's last M; draft m sees every
key before them and the drafts d with ``tree_mask[..., m, d]`` (its ancestors and
itself).  A chain of drafts is the lower triangle.

* dense  - q ``[B,QH,M,D]``, k/v ``[B,KVH,N,D]``;
* ragged - q ``[B,QH,M,D]``, k/v ``[total_kv,KVH,D]``, ``kv_indptr`` prefix
  sums ``[B+1]``;
* paged  - q ``[B,QH,M,D]``, k/v caches ``[pages*page,KVH,D]`` (or
  ``[pages,page,KVH,D]``), ``kv_indptr`` = context LENGTHS ``[B]`` (drafts counted),
  ``k/v_block_table`` ``[B, max_blocks]``.

``tree_mask``: bool ``[M, M]`` for all sequences or ``[B, M, M]``.  fp16 or bf16, D 64,
128 or 256.  Masks, layouts and numerics are otherwise those of
``speculative_decode_attention``; lengths past the block table's width count as that,
table entries are clamped into the caches, and a draft that sees no key is NaN; values that
the mask hides are multiplied by zero, so they have to be finite (those behind a sequence's
end need not be).  The computation runs in ``libfa2.so`` (``fa2_tree_decode``, include/fa2_latent.h); no fallback.
"""

from __future__ import annotations

import torch

from . import _fa2, _latent, _ops
from ._launch import DTYPES, aligned, ext, in_32_bits, index_tensor, stride_of, strides, table
from .latent_decode import check_tree, run_decode, tree_strides

# As kernels/decode.py: the C++ extension launches when it is built.
USE_EXT = True

TREE_HEAD_DIMS = (64, 128, 256)


def tree_decode_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    tree_mask: torch.Tensor,
    *,
    kv_indptr: torch.Tensor | None = None,
    k_block_table: torch.Tensor | None = None,
    v_block_table: torch.Tensor | None = None,
    kv_page_size: int | None = None,
) -> torch.Tensor:
    """See the module docstring; ``[B, QH, M, D]``."""
    name = "tree_decode_attention"
    x = ext() if USE_EXT else None
    if x is not None:
        rc, out = x.tree_decode(q, k, v, tree_mask, kv_indptr, k_block_table, v_block_table,
                                kv_page_size)
        if rc == 0:
            return out
        if rc > 0:
            raise _ops.OpsError(name, rc)
    # (the extension makes these checks itself and leaves the errors to them)
    assert q.dtype == k.dtype == v.dtype, "Tensors must have the same dtype"
    assert q.device == k.device == v.device, "Tensors must be on the same device"
    assert q.is_cuda, "Tensors must be on a CUDA device"
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"{name}: unsupported dtype {q.dtype} (float16, bfloat16)")
    if q.dim() != 4:
        raise ValueError(f"{name}: q must be [B, QH, M, D]")
    B, QH, M, D = q.shape
    if D not in TREE_HEAD_DIMS:
        raise ValueError(f"{name}: head_dim {D} not supported (supported: {TREE_HEAD_DIMS})")
    paged = k_block_table is not None
    if k.shape != v.shape or k.shape[-1] != D:
        raise ValueError(f"{name}: k and v must have equal shapes with head_dim {D}")
    if paged:
        assert v_block_table is not None
        assert kv_page_size is not None
        assert kv_indptr is not None, (
            "kv_indptr (sequence context lengths) must be provided for paged mode."
        )
        layout = _fa2.LAYOUT_PAGED
        if k.dim() not in (3, 4) or kv_page_size <= 0 or (k.dim() == 4
                                                          and k.shape[1] != kv_page_size):
            raise ValueError(f"{name}: caches must be [pages * page, KVH, D] or "
                             "[pages, page, KVH, D]")
        if k_block_table.dim() != 2 or v_block_table.dim() != 2:
            raise ValueError(f"{name}: block tables must be [B, max_blocks]")
        if (kv_indptr.numel() < B or k_block_table.shape[0] < B or v_block_table.shape[0] < B):
            raise ValueError(f"{name}: kv_indptr and the block tables need {B} rows")
        assert q.device == kv_indptr.device == k_block_table.device == v_block_table.device, (
            "Tensors must be on the same device")
    elif kv_indptr is not None:
        layout = _fa2.LAYOUT_RAGGED
        if k.dim() != 3:
            raise ValueError(f"{name}: k and v must be [total_kv, KVH, D]")
        if kv_indptr.numel() < B + 1:
            raise ValueError(f"{name}: kv_indptr needs {B + 1} prefix sums")
        assert q.device == kv_indptr.device, "Tensors must be on the same device"
    else:
        layout = _fa2.LAYOUT_DENSE
        if k.dim() != 4 or k.shape[0] != B:
            raise ValueError(f"{name}: k and v must be [{B}, KVH, N, D]")
    KVH = k.shape[1] if layout != _fa2.LAYOUT_PAGED or k.dim() == 3 else k.shape[2]
    if QH == 0 or KVH == 0 or QH % KVH != 0:
        raise ValueError(f"{name}: q_heads ({QH}) must be a multiple of kv_heads ({KVH})")
    tree_mask = check_tree(name, tree_mask, B, M, q.device)
    return _run(name, q, k, v, tree_mask, layout, kv_indptr, k_block_table, v_block_table,
                kv_page_size)


def _run(name, q, k, v, tree, layout, kv_indptr, k_table, v_table, page_size, workspace=None):
    """The ctypes launch; ``workspace`` (tests only) is a uint8 device buffer
    used instead of an allocation."""
    dev = q.device
    if layout == _fa2.LAYOUT_PAGED and k.dim() == 4:
        k, v = (t.reshape(-1, t.shape[2], t.shape[3]) for t in (k, v))
    q, k, v = aligned(q), aligned(k), aligned(v)
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    p = _latent.TreeDecodeParams()
    p.layout, p.dtype = layout, DTYPES[q.dtype]
    p.batch, p.q_heads, p.q_len, p.head_dim = q.shape
    p.kv_heads = k.shape[1]
    p.kv_len = k.shape[2] if layout == _fa2.LAYOUT_DENSE else k.shape[0]
    p.q_sb, p.q_sh, p.q_ss = strides(q)
    p.k_sb, p.k_sh, p.k_ss = strides(k)
    p.v_sb, p.v_sh, p.v_ss = strides(v)
    p.o_sb, p.o_sh, p.o_ss = strides(out)
    p.q, p.k, p.v, p.o = (t.data_ptr() for t in (q, k, v, out))
    if layout != _fa2.LAYOUT_DENSE:
        ki = index_tensor(in_32_bits(kv_indptr), dev)
        p.kv_indptr = ki.data_ptr()
    if layout == _fa2.LAYOUT_PAGED:
        kt, vt = table(in_32_bits(k_table), dev), table(in_32_bits(v_table), dev)
        p.page_size, p.table_width = int(page_size), min(kt.shape[1], vt.shape[1])
        p.k_table_stride, p.v_table_stride = kt.stride(0), vt.stride(0)
        p.k_block_table, p.v_block_table = kt.data_ptr(), vt.data_ptr()
    p.tree_sb, p.tree_sr = tree_strides(tree)
    p.tree = tree.data_ptr()
    p.softmax_scale = q.shape[3] ** -0.5
    run_decode(name, "fa2_tree_decode", p, dev, workspace)
    return out
