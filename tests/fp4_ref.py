"""Plain 64-bit forms of the operators around the attention, and the error
bounds that the GPU tests hold the kernels to.

Bounds (u = 2^-24, half a step of fp32; h = finfo(dtype).eps / 2, half a step of
the output's type), all per element:

* cache values: exact.
* qk_norm_rope: the sum of D squares is off by at most D u of itself, so the
  factor by D u / 2; 1 / sqrt, the products with x and weight and those of the
  rotation add under 8 u.  Off by (|a cos| + |b sin|) (D / 2 + 8) u, and h of the
  result for its own rounding.
* attention: a score is a sum of D products, off by at most dS = scale * (D + 4)
  * 2 u * max_j sum_d |q_d k_jd|, which moves each weight by that factor; the
  exponent's own rounding and v_exp_f32 add under 8 u to a weight (x e^-x < 1).
  Two parts of a weight leave h^2 of it.  Sums of n keys: 32 at once in an
  MFMA, then one rounding per step, merges after them: under (n / 16 + 64) 2 u.
  All of these are of A = sum_j p_j |v_j|, and both the sum of weights and the
  weighted sum have them: twice.  And h of the result.  fp16 outputs are
  multiples of 2^-24 at least: half of that on top.
"""

from __future__ import annotations

import math

import torch

U = 2.0 ** -24
E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def quantize(x):
    """(values float64, nibbles uint8, scale bytes) of rows [..., D], by search
    over the codes in 64 bits."""
    lo, hi = (-23, 13) if x.dtype == torch.float16 else (-100, 125)
    y = x.double().unflatten(-1, (-1, 32))
    a = y.abs().amax(-1)
    ok = torch.isfinite(y).all(-1)
    a = torch.where(ok, a, 1.0)
    # floor(log2 a) from frexp's exponent, exact in 64 bits
    mant, ex = torch.frexp(a)
    e = ex.long() - 1 - 2 + (mant >= 0.875).long()
    e = torch.where(a > 0, e, lo).clamp(lo, hi)
    step = torch.ldexp(torch.ones_like(a), e)
    r = torch.where(ok.unsqueeze(-1), (y / step.unsqueeze(-1)), 0.0)
    dist = (r.abs().unsqueeze(-1) - E2M1).abs()
    best = dist.amin(-1, keepdim=True)
    near = dist == best
    code = torch.arange(8)
    # of two codes as near, the even one
    code = torch.where(near & (code % 2 == 0), code, torch.where(near, code + 100, 1000)).amin(-1)
    code = code % 100
    nib = code + 8 * torch.signbit(r).long()
    nib = torch.where(ok.unsqueeze(-1), nib, 0)
    val = E2M1[code] * torch.where(torch.signbit(r), -1.0, 1.0) * step.unsqueeze(-1)
    val = torch.where(ok.unsqueeze(-1), val, math.nan)
    scale = torch.where(ok, e + 127, 255).to(torch.uint8)
    return val.flatten(-2), nib.to(torch.uint8).flatten(-2), scale


def pack(nib):
    return nib[..., 0::2] | (nib[..., 1::2] << 4)


def cached_values(codes, scales):
    """float64 values of codes [..., D/2] and scales [..., D/32] (CPU)."""
    nib = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    v = E2M1[nib & 7] * torch.where(nib >= 8, -1.0, 1.0)
    f = torch.ldexp(torch.ones(scales.shape, dtype=torch.float64), scales.long() - 127)
    f = torch.where(scales == 255, math.nan, f)
    return v * f.repeat_interleave(32, -1)


def norm_rope(x, w, table, pos, interleaved, eps):
    """(values, bound) of token-major rows x [T, H, D] in 64 bits."""
    y = x.double()
    D, R = y.shape[-1], table.shape[1]
    y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
    z, m = y.clone(), y.abs()
    pos = pos.flatten().long()
    bad = (pos < 0) | (pos >= table.shape[0])
    cs = table.double()[pos.clamp(0, max(table.shape[0] - 1, 0))][:, None] if R else None
    if R:
        c, s = cs[..., :R // 2], cs[..., R // 2:]
        ia = torch.arange(0, R, 2) if interleaved else torch.arange(R // 2)
        ib = ia + 1 if interleaved else ia + R // 2
        a, b = y[..., ia], y[..., ib]
        z[..., ia], z[..., ib] = a * c - b * s, b * c + a * s
        m[..., ia], m[..., ib] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    z[bad] = math.nan
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    return z, half_step(x.dtype) * z.abs() + m * (D / 2 + 8) * U + tiny


def attention(q, ks, vs, causal):
    """(values, bound) [QH, M, D] of one sequence in 64 bits: q [QH, M, D], cache
    values ks, vs [L, KVH, D] (float64), drafts the last M keys where causal."""
    QH, M, D = q.shape
    L, KVH, _ = ks.shape
    out = torch.full((QH, M, D), math.nan, dtype=torch.float64)
    tol = torch.zeros_like(out)
    h = half_step(q.dtype)
    scale = D ** -0.5
    for head in range(QH):
        k, v = ks[:, head // (QH // KVH)], vs[:, head // (QH // KVH)]
        x = q[head].double()
        for i in range(M):
            n = L - M + i + 1 if causal else L
            if n <= 0:
                continue
            s = k[:n] @ x[i] * scale
            p = torch.softmax(s, 0)
            o = p @ v[:n]
            size = (k[:n].abs() @ x[i].abs()).max() * scale
            rel = 2 * (size * (D + 4) * 2 * U + 8 * U + h * h + (n / 16 + 64) * 2 * U)
            out[head, i] = o
            tol[head, i] = h * o.abs() + p @ v[:n].abs() * rel
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    return out, tol + tiny


def within(got, want, tol):
    """Assert |got - want| <= tol and the same NaN places."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), "NaN in other places"
    over = ((got - want).abs() - tol)[~nan]
    if over.numel():
        worst = over.max().item()
        assert worst <= 0, f"off by {worst} more than the bound"
