"""Attention for trees of drafts over values that are not finite."""

import math

import pytest
import torch

import kernels
from test_tree_decode_gpu import make

pytestmark = pytest.mark.gpu

BF, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("layout", ["dense", "ragged", "paged"])
@pytest.mark.parametrize("dtype,n,hq,hkv,m,d,page", [
    (BF, 1, 2, 2, 1, 64, 16), (F16, 63, 4, 1, 2, 128, 16), (BF, 64, 4, 2, 3, 64, 8),
    (BF, 65, 4, 1, 4, 256, 16), (F16, 300, 8, 2, 4, 128, 5), (BF, 1300, 2, 1, 2, 64, 64),
    (BF, 100, 4, 1, 17, 64, 16),    # 68 rows
    (F16, 97, 2, 1, 16, 128, 24),   # 32 rows
    (BF, 700, 4, 1, 61, 128, 16),   # two q-blocks, units cut
    (F16, 70, 2, 1, 20, 256, 16), (BF, 33, 2, 1, 64, 256, 16),
])
def test_infinite_value_of_the_last_key(layout, dtype, n, hq, hkv, m, d, page):
    """sum p v with an infinite v under a weight above zero is infinite; the last key's
    neighbours in its tile, behind the sequence's end, add nothing to that."""
    n = max(n, m)
    q, _, vs, _, (k, v), kw = make(layout, dtype, [n, n], hq, hkv, m, d, page)
    t = torch.ones(m, m, dtype=torch.bool, device="cuda")  # every row sees the last key
    ref = kernels.tree_decode_attention(q, k, v, t, **kw)
    assert ref.isfinite().all()
    bad = v.clone()
    if layout == "dense":
        bad[1, :, n - 1, 5] = -math.inf
    elif layout == "ragged":
        bad[2 * n - 1, :, 5] = -math.inf
    else:
        at = kw["v_block_table"][1, (n - 1) // page]
        bad[at, (n - 1) % page, :, 5] = -math.inf
    o = kernels.tree_decode_attention(q, k, bad, t, **kw)
    assert (o[1, ..., 5] == -math.inf).all()
    o[1, ..., 5] = ref[1, ..., 5]
    assert torch.equal(o, ref)
