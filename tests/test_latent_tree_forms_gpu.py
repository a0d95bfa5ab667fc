"""Latent attention and attention for trees of drafts where calls differ from the usual
ones: NaN keys that some rows see, K and V of different strides, rows that start on 16 but
not on 32 bytes, many dense sequences, rows past 4 GiB, and the prefill's plans in workspaces of
any content, in graphs and on a second stream."""

import importlib
import math

import pytest
import torch

import kernels
from kernels import _fa2
from test_latent_gpu import (append_case, decode_case, decode_check, i32, prefill_case,
                             prefill_check, randn)
from test_tree_decode_gpu import make, verify

pytestmark = pytest.mark.gpu

attn_mod = importlib.import_module("kernels.latent_attention")
BF = torch.bfloat16


# ---- keys that are not finite ---------------------------------------------------------

@pytest.mark.parametrize("layout", ["dense", "ragged", "paged"])
@pytest.mark.parametrize("n,m,d", [(100, 4, 128), (100, 40, 64), (1300, 5, 64), (90, 20, 256)])
def test_tree_keys_that_are_not_finite(layout, n, m, d):
    """A NaN key makes the rows that see it NaN and no others."""
    q, _, _, t, (k, v), kw = make(layout, BF, [n, n], 4, 2, m, d)
    t = t.cuda()
    ref = kernels.tree_decode_attention(q, k, v, t, **kw)

    def with_nan(j):
        x = k.clone()
        if layout == "dense":
            x[0, 1, j, 3] = math.nan
        elif layout == "ragged":
            x[j, 1, 3] = math.nan
        else:
            x[kw["k_block_table"][0, j // 16], j % 16, 1, 3] = math.nan
        return kernels.tree_decode_attention(q, x, v, t, **kw)
    for draft in (0, m // 2, m - 1):
        o = with_nan(n - m + draft)
        sees = t[0, :, draft]
        assert o[0, 2:, sees].isnan().all()
        want = ref.clone()
        want[0, 2:, sees] = o[0, 2:, sees]
        assert torch.equal(o.nan_to_num(7.0), want.nan_to_num(7.0))
    o = with_nan(n - m - 1)  # of the context
    assert o[0, 2:].isnan().all()
    assert torch.equal(o[0, :2], ref[0, :2]) and torch.equal(o[1], ref[1])


@pytest.mark.parametrize("latent,hq,m", [(512, 4, 3), (512, 16, 8), (256, 3, 5), (256, 32, 6)])
def test_latent_keys_that_are_not_finite(latent, hq, m):
    """The shared key part of a draft: NaN for the rows that see it only."""
    lens, page = [100, 40], 16
    q, cache, table, t = decode_case(latent, BF, lens, hq, m, page, tree=True)

    def call(c):
        return kernels.latent_decode_attention(q, c.cuda(), latent_dim=latent, softmax_scale=0.07,
                                               kv_indptr=i32(lens), block_table=table.cuda(),
                                               tree_mask=t.cuda())
    ref = call(cache)
    for draft in (0, m - 1):
        j = lens[0] - m + draft
        bad = cache.clone()
        bad[table[0, j // page].long(), j % page, latent + 2] = math.nan
        o = call(bad)
        sees = t[0, :, draft].cuda()
        assert o[0, :, sees].isnan().all()
        assert torch.equal(o[0, :, ~sees], ref[0, :, ~sees]) and torch.equal(o[1], ref[1])


@pytest.mark.parametrize("q_lens,kv_lens,h", [([5, 70], [70, 100], 3), ([20], [2700], 2),
                                              ([1100, 1000], [590, 1010], 52)],
                         ids=["blocks", "split", "pairs"])
def test_prefill_values_and_keys_that_are_not_finite(q_lens, kv_lens, h):
    """The last key, behind which a tile has nothing: an infinite value is infinite in the
    result, a NaN in the shared part NaN, and the other sequences keep their bits."""
    q, k, kr, v = prefill_case(64, BF, q_lens, kv_lens, h)
    qi, ki = (i32([0] + x).cumsum(0).to(torch.int32) for x in (q_lens, kv_lens))
    ref = kernels.latent_attention(q, k, kr, v, q_indptr=qi, kv_indptr=ki)
    m, n = q_lens[0], kv_lens[0]
    bad = v.clone()
    bad[n - 1, :, 5] = math.inf
    o = kernels.latent_attention(q, k, kr, bad, q_indptr=qi, kv_indptr=ki)
    assert (o[:m, :, 5] == math.inf).all()
    o[:m, :, 5] = ref[:m, :, 5]
    assert torch.equal(o, ref)
    bad = kr.clone()
    bad[n - 1, 9] = math.nan
    o = kernels.latent_attention(q, k, bad, v, q_indptr=qi, kv_indptr=ki)
    assert o[:m].isnan().all() and torch.equal(o[m:], ref[m:])
    if m <= n:  # causal: for the last row alone
        f = dict(is_causal=True, causal_alignment="bottom_right", q_indptr=qi, kv_indptr=ki)
        ref = kernels.latent_attention(q, k, kr, v, **f)
        o = kernels.latent_attention(q, k, bad, v, **f)
        assert o[m - 1].isnan().all()
        assert torch.equal(o[:m - 1], ref[:m - 1]) and torch.equal(o[m:], ref[m:])


# ---- strides --------------------------------------------------------------------------

def widened(x, more):
    """x as a view of rows with ``more`` values behind each head's, NaN."""
    wide = torch.full(x.shape[:-1] + (x.shape[-1] + more,), math.nan, dtype=x.dtype, device="cuda")
    wide[..., :x.shape[-1]] = x
    return wide[..., :x.shape[-1]]


@pytest.mark.parametrize("layout", ["dense", "ragged", "paged"])
@pytest.mark.parametrize("lens,hq,hkv,m,d", [
    ([130, 130], 4, 1, 3, 64), ([130, 130], 4, 1, 3, 128), ([700, 700], 3, 3, 5, 64),
    ([130, 130], 4, 1, 24, 64), ([200, 200], 6, 3, 61, 128), ([90, 90], 2, 1, 20, 256),
])
def test_strides_of_k_and_v(layout, lens, hq, hkv, m, d):
    """K and V of strides of their own, rows 16 bytes off 32-byte boundaries among them."""
    q, ks, vs, t, (k, v), kw = make(layout, BF, lens, hq, hkv, m, d)
    t = t.cuda()
    ref = kernels.tree_decode_attention(q, k, v, t, **kw)
    verify(ref, q, ks, vs, t.cpu())
    for a, b in ((8, 0), (0, 24), (8, 40), (16, 8)):
        wk, wv = widened(k, a), widened(v, b)
        assert torch.equal(kernels.tree_decode_attention(q, wk, wv, t, **kw), ref), (a, b)


# ---- many dense sequences -------------------------------------------------------------

@pytest.mark.parametrize("b,n,hq,hkv,m,d", [
    (70, 2100, 2, 1, 3, 64),    # more than a wave's lanes, units cut
    (70, 2100, 2, 1, 24, 64), (300, 130, 2, 2, 5, 64), (66, 1000, 4, 1, 40, 128),
])
def test_many_dense_sequences(b, n, hq, hkv, m, d):
    q, ks, vs, t, (k, v), kw = make("dense", BF, [n] * b, hq, hkv, m, d)
    verify(kernels.tree_decode_attention(q, k, v, t.cuda(), **kw), q, ks, vs, t)


# ---- the prefill's plans --------------------------------------------------------------

PLANS = [([20], [2700], 2),                                         # keys split
         ([2] * 40, [30] * 40, 16),                                 # a list, no splits
         ([500, 600, 300, 700, 40], [500, 700, 300, 900, 1100], 24)]  # pairs, claimed


@pytest.mark.parametrize("q_lens,kv_lens,h", PLANS, ids=["split", "list", "claimed"])
def test_prefill_plans(q_lens, kv_lens, h):
    q, k, kr, v = prefill_case(128, BF, q_lens, kv_lens, h)
    qi, ki = (i32([0] + x).cumsum(0).to(torch.int32) for x in (q_lens, kv_lens))
    f = dict(is_causal=True, causal_alignment="bottom_right", q_indptr=qi, kv_indptr=ki)
    ref = kernels.latent_attention(q, k, kr, v, **f)
    prefill_check(ref, q, k, kr, v, q_lens, kv_lens, "bottom_right", 192 ** -0.5)
    for fill in (0, 255, 1):
        ws = torch.full((2 ** 26,), fill, dtype=torch.uint8, device="cuda")
        for _ in range(2):  # the second call finds what the first one left
            got = attn_mod._run("x", q, k, kr, v, _fa2.MASK_BOTTOM_RIGHT, qi, ki, None,
                                workspace=ws)
            assert torch.equal(got, ref), fill
    with pytest.raises(ValueError):
        attn_mod._run("x", q, k, kr, v, _fa2.MASK_BOTTOM_RIGHT, qi, ki, None, workspace=ws[:64])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            a = kernels.latent_attention(q, k, kr, v, **f)
    b = kernels.latent_attention(q, k, kr, v, **f)
    torch.cuda.synchronize()
    assert torch.equal(a, ref) and torch.equal(b, ref)
    graph, out = torch.cuda.CUDAGraph(), [None, None]
    v2 = randn(*v.shape, dtype=BF, seed=77).cuda()
    ref2 = kernels.latent_attention(q, k, kr, v2, **f)
    with torch.cuda.graph(graph):
        out[0] = kernels.latent_attention(q, k, kr, v, **f)
        out[1] = kernels.latent_attention(q, k, kr, v2, **f)
    for i in range(4):
        out[0].zero_()
        out[1].zero_()
        graph.replay()
        other = kernels.latent_attention(q, k, kr, v, **f)
        torch.cuda.synchronize()
        assert torch.equal(out[0], ref) and torch.equal(out[1], ref2), i
        assert torch.equal(other, ref), i


@pytest.mark.parametrize("q_lens,kv_lens,h", [([40, 200], [1300, 260], 2),
                                              ([1100, 500], [1300, 800], 52)],
                         ids=["blocks", "pairs"])
def test_prefill_rows_past_4_gib(q_lens, kv_lens, h):
    """The shared part in rows 2 or 4 MB apart, ragged and dense."""
    q, k, kr, v = prefill_case(64, BF, q_lens, kv_lens, h)
    qi, ki = (i32([0] + x).cumsum(0).to(torch.int32) for x in (q_lens, kv_lens))
    f = dict(is_causal=True, causal_alignment="bottom_right")
    far = torch.zeros(kr.shape[0], 2 ** 21, dtype=BF, device="cuda")[:, 2 ** 20:2 ** 20 + 64]
    far.copy_(kr)
    assert far.stride(0) * 2 * (far.shape[0] - 1) > 2 ** 32
    ref = kernels.latent_attention(q, k, kr, v, q_indptr=qi, kv_indptr=ki, **f)
    prefill_check(ref, q, k, kr, v, q_lens, kv_lens, "bottom_right", 128 ** -0.5)
    o = kernels.latent_attention(q, k, far, v, q_indptr=qi, kv_indptr=ki, **f)
    assert torch.equal(o, ref)
    m, n = q_lens[0], kv_lens[0]
    qd, kd, vd = (x[None, :c].transpose(1, 2) for x, c in ((q, m), (k, n), (v, n)))
    near = kernels.latent_attention(qd, kd, kr[None, :n], vd, **f)
    assert torch.equal(kernels.latent_attention(qd, kd, far[None, :n], vd, **f), near)
    # keys and values of the heads as far apart
    up = torch.zeros(k.shape[0], 2 ** 20, dtype=BF, device="cuda")[:, :h * 128].unflatten(1, (h, 128))
    up[..., :64], up[..., 64:] = k, v
    o = kernels.latent_attention(q, up[..., :64], kr, up[..., 64:], q_indptr=qi, kv_indptr=ki, **f)
    assert torch.equal(o, ref)


# ---- graphs whose inputs change between replays ----------------------------------------

def capture(f):
    f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f()
    return graph, out


def test_append_in_a_graph():
    """A captured append writes what its buffers hold at the replay."""
    lens, starts, page = [1, 3, 0, 40], [0, 15, 7, 100], 16
    x, w, rope, table, cache, _ = append_case(512, BF, [64] * 4, [200] * 4, page)
    table, sp = table.cuda(), i32(starts)
    ip = i32([0] + lens).cumsum(0).to(torch.int32)
    first = cache.clone()
    graph, rows = capture(lambda: kernels.paged_latent_append(cache, table, x, ip, w, rope, sp,
                                                              return_rows=True))
    for i, (ln, st) in enumerate([(lens, starts), ([2, 2, 2, 2], [9, 0, 31, 190]),
                                  ([64] * 4, [100, 0, 199, 5]), ([0, 0, 0, 0], [1] * 4)]):
        ip.copy_(i32([0] + ln).cumsum(0))
        sp.copy_(i32(st))
        x.copy_(randn(*x.shape, dtype=BF, seed=50 + i))
        cache.copy_(first)
        graph.replay()
        eager = first.clone()
        want = kernels.paged_latent_append(eager, table, x, ip, w, rope, sp, return_rows=True)
        torch.cuda.synchronize()
        assert torch.equal(cache, eager) and torch.equal(rows[:sum(ln)], want[:sum(ln)]), i


@pytest.mark.parametrize("latent,hq,m", [(512, 128, 0), (512, 16, 0), (256, 32, 7)])
def test_latent_decode_in_a_graph(latent, hq, m):
    """A captured decode call goes by the lengths, the table, the queries and the mask of
    the replay: whole units, cut ones and empty ones from one plan."""
    page, b, width = 16, 4, 200
    q, cache, table, t = decode_case(latent, BF, [width * page] * b, hq, m, page, tree=m > 0)
    c, bt, li = cache.cuda(), table.cuda(), i32([1] * b)
    t = t.cuda() if m else None
    f = dict(latent_dim=latent, softmax_scale=0.07, kv_indptr=li, block_table=bt, tree_mask=t)
    graph, out = capture(lambda: kernels.latent_decode_attention(q, c, **f))
    for i, lens in enumerate([[3200] * 4, [1, 40, 64, 65], [3100, 0, 700, 2], [10] * 4,
                              [5000, -1, 129, 3200]]):
        li.copy_(i32(lens))
        q.copy_(randn(*q.shape, dtype=BF, seed=90 + i))
        bt.copy_(bt.roll(1, 0).clone())
        if m:
            t.copy_(t.roll(1, 0).clone())
        out.zero_()
        graph.replay()
        want = kernels.latent_decode_attention(q, c, **f)
        torch.cuda.synchronize()
        assert torch.equal(out.nan_to_num(7.0), want.nan_to_num(7.0)), i
        fresh = decode_case(latent, BF, [width * page] * b, hq, m, page, tree=m > 0)[1]
        held = [min(max(n, 0), width * page) for n in lens]
        decode_check(out, q, fresh, bt.cpu(), held, latent, 0.07, False,
                     t.cpu() if m else None, page)


@pytest.mark.parametrize("m,hq,hkv,d", [(9, 8, 2, 128), (3, 4, 4, 64), (20, 4, 1, 256)])
def test_tree_decode_in_a_graph(m, hq, hkv, d):
    q, ks, vs, t, (k, v), kw = make("paged", BF, [2600, 2600, 2600], hq, hkv, m, d)
    t, li = t.cuda(), kw["kv_indptr"]
    graph, out = capture(lambda: kernels.tree_decode_attention(q, k, v, t, **kw))
    for i, lens in enumerate([[2600, 1, 300], [0, 64, 63], [2600] * 3, [30, 2000, 1000]]):
        li.copy_(i32(lens))
        q.copy_(randn(*q.shape, dtype=BF, seed=40 + i))
        t.copy_(t.roll(1, 0).clone())
        out.zero_()
        graph.replay()
        want = kernels.tree_decode_attention(q, k, v, t, **kw)
        torch.cuda.synchronize()
        assert torch.equal(out.nan_to_num(7.0), want.nan_to_num(7.0)), i
        verify(out, q, [x[:n] for x, n in zip(ks, lens)], [x[:n] for x, n in zip(vs, lens)],
               t.cpu())


@pytest.mark.parametrize("h", [2, 24], ids=["blocks", "claimed"])
def test_prefill_in_a_graph(h):
    """A captured ragged prefill goes by the prefix sums of the replay."""
    tq, tk = 2140, 3700
    q, k, kr, v = prefill_case(128, BF, [tq], [tk], h)
    qi, ki = torch.zeros(4, dtype=torch.int32, device="cuda"), i32([0] * 4)
    f = dict(is_causal=True, causal_alignment="bottom_right", q_indptr=qi, kv_indptr=ki)
    graph, out = capture(lambda: kernels.latent_attention(q, k, kr, v, **f))
    for i, (ql, kl) in enumerate([([500, 600, 1040], [500, 700, 2500]), ([2140, 0, 0], [2140, 5, 0]),
                                  ([1, 2, 3], [3000, 2, 600]), ([130, 300, 7], [130, 300, 9])]):
        qi.copy_(i32([0] + ql).cumsum(0))
        ki.copy_(i32([0] + kl).cumsum(0))
        q.copy_(randn(*q.shape, dtype=BF, seed=60 + i))
        out.zero_()
        graph.replay()
        want = kernels.latent_attention(q, k, kr, v, **f)
        torch.cuda.synchronize()
        n, nk = sum(ql), sum(kl)
        assert torch.equal(out[:n].nan_to_num(7.0), want[:n].nan_to_num(7.0)), i
        assert (out[n:] == 0).all()  # rows of nobody are left as they were
        prefill_check(out[:n], q[:n], k[:nk], kr[:nk], v[:nk], ql, kl, "bottom_right",
                      192 ** -0.5)
