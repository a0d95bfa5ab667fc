"""``qk_norm_rope`` on MI355X: the RMS norm of every query and key head and the
rotation of its position, in one pass over both.

It stands between a model's projections and the attention entry points: the
reference's kernels (harsh-vsingh/triton-kernels) take finished queries and
keys.  For each head row x of ``head_dim`` values::

    y = x * rsqrt(mean(x ** 2) + eps) * weight
    (a, b) -> (a * cos - b * sin, b * cos + a * sin)

over the pairs (i, i + R/2) of y's first R values, or (2i, 2i + 1) with
``interleaved``; cos and sin of the pair and the token's position come from a
table (:func:`build_rope_table`), whose width is R.  The arithmetic is fp32
whatever the tensors' type, rounded once at the end (so a bf16 or fp32 row whose
sum of squares passes fp32's range, values around 2 ** 60, gives zeros).  The
computation runs in ``libfa2.so`` (``fa2_norm_rope``, include/fa2_ops.h); no
fallback, and no backward pass, like the rest of the package.
"""

from __future__ import annotations

import torch

from . import _ops
from ._launch import DTYPES, aligned, check_dtype_and_dim, ext, strides

# As kernels/decode.py: the C++ extension launches when it is built.
USE_EXT = True

_NAME = "qk_norm_rope"


def build_rope_table(max_positions: int, rotary_dim: int, *, base: float = 10000.0,
                     device="cuda") -> torch.Tensor:
    """The table of :func:`qk_norm_rope`: float32 ``[max_positions, rotary_dim]``,
    cosines of ``position * base ** (-2 i / rotary_dim)`` in the first half of a
    row, sines in the second.  The angles are computed in float64 (an fp32
    angle of position 100000 is off by 0.004)."""
    if rotary_dim <= 0 or rotary_dim % 16:
        raise ValueError(f"build_rope_table: rotary_dim {rotary_dim} must be a positive multiple "
                         "of 16")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    angle = (torch.arange(max_positions, dtype=torch.float64, device=device)[:, None]
             * float(base) ** (-i / rotary_dim))
    return torch.cat([angle.cos(), angle.sin()], 1).to(torch.float32)


def qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    rope_table: torch.Tensor,
    positions: torch.Tensor,
    *,
    eps: float = 1e-6,
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Normalised and rotated (q, k), as new contiguous tensors of the shapes given.

    ``q`` and ``k`` are each token-major ``[T, H, D]`` (ragged prefill, decode,
    ``paged_kv_append``) or ``[B, H, M, D]`` (dense, paged and speculative
    queries), T = B * M with token b * M + m; any strides with contiguous rows
    that start on 16 bytes, such as views of a fused projection's output (other
    tensors are copied first).  ``q_weight`` / ``k_weight``: ``[D]``, of q's type
    or float32.  ``rope_table``: float32 ``[P, R]``, R <= D a multiple of 16.
    ``positions``: T integers (int32 or int64, any shape), a token's row of the
    table; a token whose position is outside ``[0, P)`` becomes NaN.
    """
    x = ext() if USE_EXT else None
    if x is not None:
        rc, q_out, k_out = x.norm_rope(q, k, q_weight, k_weight, rope_table, positions, eps,
                                       interleaved)
        if rc == 0:
            return q_out, k_out
        if rc > 0:
            raise _ops.OpsError(_NAME, rc)
    # (the extension makes these checks itself and leaves the errors to them)
    assert q.dtype == k.dtype, "Tensors must have the same dtype"
    assert (q.device == k.device == q_weight.device == k_weight.device == rope_table.device
            == positions.device), "Tensors must be on the same device"
    assert q.is_cuda, "Tensors must be on a CUDA device"
    if q.dim() not in (3, 4) or k.dim() not in (3, 4):
        raise ValueError(f"{_NAME}: q and k must be [T, H, D] or [B, H, M, D]")
    D = q.shape[-1]
    check_dtype_and_dim(_NAME, q.dtype, D)
    T = q.shape[0] if q.dim() == 3 else q.shape[0] * q.shape[2]
    Tk = k.shape[0] if k.dim() == 3 else k.shape[0] * k.shape[2]
    if k.shape[-1] != D or Tk != T:
        raise ValueError(f"{_NAME}: k must have q's head_dim ({D}) and tokens ({T})")
    if q_weight.shape != (D,) or k_weight.shape != (D,):
        raise ValueError(f"{_NAME}: weights must be [{D}]")
    if q_weight.dtype != k_weight.dtype or q_weight.dtype not in (q.dtype, torch.float32):
        raise TypeError(f"{_NAME}: weights must both be {q.dtype} or torch.float32")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{_NAME}: positions must be int32 or int64")
    if positions.numel() != T:
        raise ValueError(f"{_NAME}: positions must hold one integer for each of {T} tokens")
    if rope_table.dtype != torch.float32 or rope_table.dim() != 2:
        raise TypeError(f"{_NAME}: rope_table must be float32 [positions, rotary_dim]")
    R = rope_table.shape[1]
    if R > D or R % 16:
        raise ValueError(f"{_NAME}: rotary_dim {R} must be a multiple of 16, at most {D}")
    if not eps >= 0:
        raise ValueError(f"{_NAME}: eps must not be negative")
    q, k = aligned(q), aligned(k)
    q_weight, k_weight, rope_table = (
        t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(
            memory_format=torch.contiguous_format) for t in (q_weight, k_weight, rope_table))
    positions = positions.contiguous()
    q_out, k_out = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
    p = _ops.NormRopeParams()
    p.dtype, p.weight_dtype = DTYPES[q.dtype], DTYPES[q_weight.dtype]
    p.interleaved, p.eps = int(bool(interleaved)), float(eps)
    p.tokens, p.q_heads, p.kv_heads, p.head_dim = T, q.shape[1], k.shape[1], D
    p.rotary_dim, p.positions, p.rope_stride = R, rope_table.shape[0], R
    p.q_rows = q.shape[2] if q.dim() == 4 else T
    p.k_rows = k.shape[2] if k.dim() == 4 else T
    p.q_sb, p.q_sh, p.q_ss = strides(q)
    p.k_sb, p.k_sh, p.k_ss = strides(k)
    p.qo_sb, p.qo_sh, p.qo_ss = strides(q_out)
    p.ko_sb, p.ko_sh, p.ko_ss = strides(k_out)
    p.q, p.k, p.q_out, p.k_out = (t.data_ptr() for t in (q, k, q_out, k_out))
    p.q_weight, p.k_weight = q_weight.data_ptr(), k_weight.data_ptr()
    p.rope, p.position = rope_table.data_ptr(), positions.data_ptr()
    p.position_64 = int(positions.dtype == torch.int64)
    with torch.cuda.device(q.device):
        _ops.call(_NAME, "fa2_norm_rope", p, torch.cuda.current_stream().cuda_stream)
    return q_out, k_out
