"""``latent_decode_attention`` on MI355X: attention of one or more query tokens per
sequence over a latent cache (``latent_cache``), in the absorbed form.

The keys' up-projection is folded into the queries and the values' one is applied to
the result, so every head attends to the cached rows themselves: for token m of head h,
with ``x_n = (c_n, r_n)`` the sequence's rows::

    out = sum_n p_n c_n,   p = softmax_n(softmax_scale * q . x_n)

* ``q`` ``[B, QH, latent_dim + 64]``: one token per sequence; any strides whose rows
  start on 16 bytes (heads outside, as a batched product leaves them);
* ``q`` ``[B, QH, M, latent_dim + 64]``: the cache's last M rows are theirs.
  ``causal=True`` hides from token m those after it; ``tree_mask`` (bool ``[M, M]`` or
  ``[B, M, M]``, M <= 64) says instead which of them token m sees
  (``tree_decode_attention`` has the same mask over K/V caches).

``kv_indptr`` holds each sequence's length (as for the paged decode calls, the
reference's kernels/decode.py:203-331); lengths past the block table's width count as
that.  ``softmax_scale`` is the model's, that of the expanded keys.  16-bit MFMA with fp32
accumulation and softmax statistics; only the softmax weights are rounded to the
tensors' type for the product with the latents, and summed as rounded.  A row that sees
no key is NaN, as in the other decode calls; rows of a sequence that the mask hides are
multiplied by zero, so their latents have to be finite (what lies behind the sequence's end
need not be).  The computation runs in ``libfa2.so``
(``fa2_latent_decode``, include/fa2_latent.h); no fallback.
"""

from __future__ import annotations

import math

import torch

from . import _fa2, _latent, _ops
from ._launch import DTYPES, aligned, ext, in_32_bits, index_tensor, stride_of, table
from .latent_cache import check_cache, check_latent_dim

# As kernels/decode.py: the C++ extension launches when it is built.
USE_EXT = True


def check_tree(name: str, tree: torch.Tensor, batch: int, m: int, device) -> torch.Tensor:
    """``tree_mask`` as the kernels take it: bytes, drafts of a row side by side."""
    assert tree.device == device, "Tensors must be on the same device"
    if tree.dtype not in (torch.bool, torch.uint8):
        raise TypeError(f"{name}: tree_mask must be bool")
    if m > _latent.TREE_MAX:
        raise ValueError(f"{name}: trees hold at most {_latent.TREE_MAX} drafts")
    if tree.shape not in ((m, m), (batch, m, m)):
        raise ValueError(f"{name}: tree_mask must be [{m}, {m}] or [{batch}, {m}, {m}]")
    return tree if m <= 1 or tree.stride(-1) == 1 else tree.contiguous()


def tree_strides(tree: torch.Tensor):
    """(batch, draft) strides."""
    return (stride_of(tree, 0) if tree.dim() == 3 else 0), stride_of(tree, tree.dim() - 2)


def latent_decode_attention(
    q: torch.Tensor,
    cache: torch.Tensor,
    *,
    latent_dim: int,
    softmax_scale: float,
    kv_indptr: torch.Tensor,
    block_table: torch.Tensor,
    causal: bool = False,
    tree_mask: torch.Tensor | None = None,
) -> torch.Tensor:
    """See the module docstring; ``[B, QH, latent_dim]`` or ``[B, QH, M, latent_dim]``."""
    name = "latent_decode_attention"
    x = ext() if USE_EXT else None
    if x is not None:
        rc, out = x.latent_decode(q, cache, latent_dim, softmax_scale, kv_indptr, block_table,
                                  bool(causal), tree_mask)
        if rc == 0:
            return out
        if rc > 0:
            raise _ops.OpsError(name, rc)
    # (the extension makes these checks itself and leaves the errors to them)
    if q.dim() not in (3, 4):
        raise ValueError(f"{name}: q must be [B, QH, width] or [B, QH, M, width]")
    check_cache(name, cache)
    check_latent_dim(name, latent_dim, cache.shape[2])
    if q.dtype != cache.dtype:
        raise TypeError(f"{name}: q must be {cache.dtype}, as the cache")
    if q.shape[-1] != cache.shape[2]:
        raise ValueError(f"{name}: q's rows must be the cache's ({cache.shape[2]} values)")
    assert q.device == cache.device == kv_indptr.device == block_table.device, (
        "Tensors must be on the same device")
    B, QH = q.shape[:2]
    if QH == 0:
        raise ValueError(f"{name}: q has no heads")
    if kv_indptr.numel() < B or block_table.dim() != 2 or block_table.shape[0] < B:
        raise ValueError(f"{name}: kv_indptr and the block table need {B} rows")
    if not (softmax_scale > 0 and math.isfinite(softmax_scale)):
        raise ValueError(f"{name}: softmax_scale must be above zero and finite")
    if tree_mask is not None:
        tree_mask = check_tree(name, tree_mask, B, q.shape[2] if q.dim() == 4 else 1, q.device)
    return _run(name, q, cache, latent_dim, softmax_scale, kv_indptr, block_table, causal,
                tree_mask)


def _run(name, q, cache, latent_dim, softmax_scale, lens, block_table, causal, tree,
         workspace=None):
    """The ctypes launch; ``workspace`` (tests only) is a uint8 device buffer
    used instead of an allocation."""
    dev = q.device
    q4 = aligned(q.unsqueeze(2) if q.dim() == 3 else q)
    B, QH, M, W = q4.shape
    out = torch.empty(q.shape[:-1] + (latent_dim,), dtype=q.dtype, device=dev)
    o4 = out.unsqueeze(2) if q.dim() == 3 else out
    li, bt = index_tensor(in_32_bits(lens), dev), table(in_32_bits(block_table), dev)
    p = _latent.LatentDecodeParams()
    p.dtype = DTYPES[q.dtype]
    p.mask = (_latent.MASK_TREE if tree is not None else
              _fa2.MASK_BOTTOM_RIGHT if causal else _fa2.MASK_NONE)
    p.batch, p.q_heads, p.q_len = B, QH, M
    p.latent_dim, p.rope_dim = latent_dim, W - latent_dim
    p.page_size, p.num_pages = cache.shape[1], cache.shape[0]
    p.table_width, p.table_stride = bt.shape[1], bt.stride(0)
    p.q_sb, p.q_sh, p.q_ss = (stride_of(q4, i) for i in range(3))
    p.o_sb, p.o_sh, p.o_ss = (stride_of(o4, i) for i in range(3))
    p.q, p.o, p.cache = q4.data_ptr(), out.data_ptr(), cache.data_ptr()
    p.kv_lens, p.block_table = li.data_ptr(), bt.data_ptr()
    if tree is not None:
        p.tree_sb, p.tree_sr = tree_strides(tree)
        p.tree = tree.data_ptr()
    p.softmax_scale = float(softmax_scale)
    run_decode(name, "fa2_latent_decode", p, dev, workspace)
    return out


def run_decode(name, entry, p, dev, workspace) -> None:
    """Workspace and launch of the decode calls on torch's current stream of ``dev``."""
    with torch.cuda.device(dev):
        n = _latent.workspace_size(name, entry, p)
        if n:
            ws = workspace if workspace is not None else torch.empty(n, dtype=torch.uint8,
                                                                     device=dev)
            if ws.numel() < n or ws.device != dev:
                raise ValueError(f"workspace needs {n} bytes on {dev}")
            p.workspace, p.workspace_bytes = ws.data_ptr(), n
        _latent.call(name, entry, p, torch.cuda.current_stream().cuda_stream)
