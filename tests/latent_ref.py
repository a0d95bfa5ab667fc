"""64-bit restatements of latent attention and of attention for trees of drafts, with
bounds of what the kernels' arithmetic may add.

``attention64`` takes keys and values as one head's rows.  Its bound counts, relative to
A = sum_n w_n |v_n| (w the exact weights): the rounding of each weight to the tensors'
type, u = eps / 2, once in the numerator and once in the sum (2 u); the scores' fp32
sums, which change a weight by the factor exp(e) with
e <= (2 + dims) 2^-24 scale sum_d |q_d k_d| + 4 2^-24 |score| + 2^-22 (exponent and its
scaling), again twice; fp32 sums over n keys, (n + 64) 2^-24 each; then u |o| for the
output and the type's smallest number.
"""

import math

import torch


def attention64(q, k, v, sees, scale, dtype):
    """(output, bound) of rows q [R, Dk] over k [N, Dk], v [N, Dv] (all float64);
    ``sees`` bool [R, N]; NaN rows where nothing is seen."""
    n = k.shape[0]
    u = torch.finfo(dtype).eps / 2
    logits = (q @ k.T) * scale
    size = (q.abs() @ k.abs().T) * scale
    logits = logits.masked_fill(~sees, -math.inf)
    w = torch.softmax(logits, -1)
    o = torch.where(sees.any(-1, keepdim=True), w @ v, math.nan)
    a = w @ v.abs()
    size = torch.where(sees, size, 0.0).amax(-1, keepdim=True) if n else torch.zeros_like(o[:, :1])
    e = (q.shape[1] + 6) * 2.0 ** -24 * size + 2.0 ** -22
    rel = 2 * (u + e + (n + 64) * 2.0 ** -24)
    return o, 1.02 * rel * a + u * o.abs() * 1.02 + torch.finfo(dtype).smallest_normal


def visible(n, m, causal, tree):
    """bool [m, n]: what each of m tokens, the last of n keys, sees."""
    sees = torch.ones(m, n, dtype=torch.bool)
    draft = torch.arange(n) - (n - m)
    for i in range(m):
        for x in range(max(0, n - m), n):
            d = int(draft[x])
            if tree is not None:
                sees[i, x] = bool(tree[i, d])
            elif causal:
                sees[i, x] = d <= i
    return sees


def check(got, want, bound, what=""):
    """NaN where NaN is wanted, within the bound elsewhere."""
    got = got.double().cpu()
    want, bound = want.cpu(), bound.cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN rows"
    off = ((got - want).abs() - bound).nan_to_num(nan=-1.0)
    assert not (off > 0).any(), (
        f"{what}: {int((off > 0).sum())} of {off.numel()} off, by {off.max().item():.3e} at most; "
        f"largest error {(got - want).abs().nan_to_num().max().item():.3e}")


def random_tree(m, seed, generator=None):
    """bool [m, m]: each draft sees itself and its ancestors."""
    g = torch.Generator().manual_seed(seed)
    sees = torch.zeros(m, m, dtype=torch.bool)
    for i in range(m):
        p = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
        if p >= 0:
            sees[i] = sees[p]
        sees[i, i] = True
    return sees


def pages_of(lens, page, seed, spare=2, width=0, fill=-1):
    """A shuffled block table [B, width] (padded with ``fill``) and the pool's pages."""
    need = [(n + page - 1) // page for n in lens]
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(sum(need) + spare, generator=g)
    t = torch.full((len(lens), max(need + [width, 1])), fill, dtype=torch.int32)
    at = 0
    for b, c in enumerate(need):
        t[b, :c] = perm[at:at + c].to(torch.int32)
        at += c
    return t, sum(need) + spare


def finished_rows64(x, weight, rope, positions, eps, interleaved):
    """(rows, bound per unit of rounding) of the cache's writer: x [T, R + 64] float64."""
    r = weight.shape[0]
    c, z = x[:, :r], x[:, r:]
    y = torch.empty_like(x)
    size = torch.empty_like(x)
    y[:, :r] = c / torch.sqrt(c.square().mean(-1, keepdim=True) + eps) * weight
    size[:, :r] = y[:, :r].abs()
    half = z.shape[1] // 2
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        cs, sn = rope[positions, i], rope[positions, half + i]
        y[:, r + a] = z[:, a] * cs - z[:, b] * sn
        y[:, r + b] = z[:, b] * cs + z[:, a] * sn
        size[:, r + a] = (z[:, a] * cs).abs() + (z[:, b] * sn).abs()
        size[:, r + b] = (z[:, b] * cs).abs() + (z[:, a] * sn).abs()
    return y, size
