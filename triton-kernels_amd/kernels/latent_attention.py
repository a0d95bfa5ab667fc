"""``latent_attention`` on MI355X: prefill attention of a latent-attention model, in the
expanded form.

Every head has keys and values of its own, up-projected from the latents, and the keys
end in a part that all heads share (the rotated part of the cached rows,
``latent_cache``)::

    out[m, h] = sum_n p_n v[n, h],   p = softmax_n(scale * (q[m, h] . (k[n, h], k_rope[n])))

* dense  - q ``[B,H,M,D+64]``, k / v ``[B,H,N,D]``, k_rope ``[B,N,64]``;
* ragged - q ``[Tq,H,D+64]``, k / v ``[Tk,H,D]``, k_rope ``[Tk,64]``, ``q_indptr`` /
  ``kv_indptr`` prefix sums ``[B+1]``.

D is 64 or 128 (keys without the shared part, and values), fp16 or bf16; rows of any
strides that start on 16 bytes are read in place, such as k and v as views of one
up-projection and k_rope as a view of the finished rows.  ``is_causal`` and
``causal_alignment`` are those of ``flash_attention_v2`` (the reference's
kernels/attention.py:749-927), whose kernel and numerics these are; ``softmax_scale``:
``(D + 64) ** -0.5`` unless given.  Values that the mask hides from a row may be multiplied by
zero, so they have to be finite (what lies behind a sequence's end need not be).  The
computation runs in ``libfa2.so`` (``fa2_latent_prefill``, include/fa2_latent.h); no fallback.
"""

from __future__ import annotations

import math

import torch

from . import _fa2, _latent, _ops
from ._launch import DTYPES, aligned, ext, in_32_bits, index_tensor, stride_of, strides
from .latent_decode import run_decode

# As kernels/decode.py: the C++ extension launches when it is built.
USE_EXT = True

LATENT_HEAD_DIMS = (64, 128)


def latent_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    k_rope: torch.Tensor,
    v: torch.Tensor,
    is_causal: bool = False,
    *,
    q_indptr: torch.Tensor | None = None,
    kv_indptr: torch.Tensor | None = None,
    softmax_scale: float | None = None,
    causal_alignment: str = "top_left",
) -> torch.Tensor:
    """See the module docstring; q's shape with D values a row."""
    name = "latent_attention"
    if causal_alignment not in ("top_left", "bottom_right"):
        raise ValueError(f"{name}: causal_alignment must be 'top_left' or 'bottom_right'")
    mask = (_fa2.MASK_NONE if not is_causal else _fa2.MASK_TOP_LEFT
            if causal_alignment == "top_left" else _fa2.MASK_BOTTOM_RIGHT)
    x = ext() if USE_EXT else None
    if x is not None:
        rc, out = x.latent_prefill(q, k, k_rope, v, mask, q_indptr, kv_indptr, softmax_scale)
        if rc == 0:
            return out
        if rc > 0:
            raise _ops.OpsError(name, rc)
    # (the extension makes these checks itself and leaves the errors to them)
    assert q.dtype == k.dtype == k_rope.dtype == v.dtype, "Tensors must have the same dtype"
    assert q.device == k.device == k_rope.device == v.device, "Tensors must be on the same device"
    assert q.is_cuda, "Tensors must be on a CUDA device"
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"{name}: unsupported dtype {q.dtype} (float16, bfloat16)")
    ragged = q_indptr is not None or kv_indptr is not None
    dims = 3 if ragged else 4
    if ragged and (q_indptr is None or kv_indptr is None):
        raise ValueError(f"{name}: pass q_indptr and kv_indptr together")
    if q.dim() != dims or k.dim() != dims or v.dim() != dims or k_rope.dim() != dims - 1:
        raise ValueError(f"{name}: q, k, v must be " + (
            "[T, H, D] and k_rope [T, 64]" if ragged else "[B, H, L, D] and k_rope [B, L, 64]"))
    D = k.shape[-1]
    if D not in LATENT_HEAD_DIMS:
        raise ValueError(f"{name}: head_dim {D} not supported (supported: {LATENT_HEAD_DIMS})")
    if q.shape[-1] != D + _latent.ROPE_DIM or k_rope.shape[-1] != _latent.ROPE_DIM:
        raise ValueError(f"{name}: q's rows must have {D + _latent.ROPE_DIM} values and k_rope's "
                         f"{_latent.ROPE_DIM}")
    H = q.shape[1]
    rows = k.shape[:1] if ragged else (k.shape[0], k.shape[2])
    if k.shape != v.shape or k.shape[1] != H or k_rope.shape[:-1] != rows or (
            not ragged and k.shape[0] != q.shape[0]):
        raise ValueError(f"{name}: k and v must have equal shapes with q's heads ({H}), k_rope "
                         "their tokens")
    if H == 0:
        raise ValueError(f"{name}: q has no heads")
    if ragged:
        assert q.device == q_indptr.device == kv_indptr.device, (
            "Tensors must be on the same device")
        if q_indptr.numel() != kv_indptr.numel() or q_indptr.numel() == 0:
            raise ValueError(f"{name}: q_indptr and kv_indptr must hold B + 1 prefix sums each")
    if softmax_scale is not None and not (softmax_scale > 0 and math.isfinite(softmax_scale)):
        raise ValueError(f"{name}: softmax_scale must be above zero and finite")
    return _run(name, q, k, k_rope, v, mask, q_indptr, kv_indptr, softmax_scale)


def _run(name, q, k, k_rope, v, mask, q_indptr, kv_indptr, softmax_scale, workspace=None):
    """The ctypes launch; ``workspace`` (tests only) is a uint8 device buffer
    used instead of an allocation."""
    dev = q.device
    q, k, k_rope, v = aligned(q), aligned(k), aligned(k_rope), aligned(v)
    D = k.shape[-1]
    ragged = q_indptr is not None
    out = torch.empty(q.shape[:-1] + (D,), dtype=q.dtype, device=dev)
    p = _latent.LatentPrefillParams()
    p.layout = _fa2.LAYOUT_RAGGED if ragged else _fa2.LAYOUT_DENSE
    p.dtype, p.mask = DTYPES[q.dtype], mask
    p.heads, p.head_dim, p.rope_dim = q.shape[1], D, _latent.ROPE_DIM
    if ragged:
        qi, ki = (index_tensor(in_32_bits(t), dev) for t in (q_indptr, kv_indptr))
        p.q_indptr, p.kv_indptr = qi.data_ptr(), ki.data_ptr()
        p.batch, p.q_len, p.kv_len = q_indptr.numel() - 1, q.shape[0], k.shape[0]
    else:
        p.batch, p.q_len, p.kv_len = q.shape[0], q.shape[2], k.shape[2]
    p.q_sb, p.q_sh, p.q_ss = strides(q)
    p.k_sb, p.k_sh, p.k_ss = strides(k)
    p.v_sb, p.v_sh, p.v_ss = strides(v)
    p.o_sb, p.o_sh, p.o_ss = strides(out)
    p.kr_sb = 0 if ragged else stride_of(k_rope, 0)
    p.kr_ss = stride_of(k_rope, k_rope.dim() - 2)
    p.q, p.k, p.kr, p.v, p.o = (t.data_ptr() for t in (q, k, k_rope, v, out))
    p.softmax_scale = float(softmax_scale) if softmax_scale is not None else q.shape[-1] ** -0.5
    run_decode(name, "fa2_latent_prefill", p, dev, workspace)
    return out
