"""Attention for trees of drafts over 16-bit K/V caches, against the 64-bit restatement
of tests/latent_ref.py (whose bounds count roundings), and a serving loop over it and the
latent cache."""

import importlib
import math

import pytest
import torch

import kernels
from kernels import _fa2
from latent_ref import attention64, check, pages_of, random_tree, visible

pytestmark = pytest.mark.gpu

tree_mod = importlib.import_module("kernels.tree_decode")
BF, F16 = torch.bfloat16, torch.float16


def randn(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.fixture(params=[True, False], ids=["ext", "ctypes"])
def path(request, monkeypatch):
    monkeypatch.setattr(tree_mod, "USE_EXT", request.param)
    return request.param


def make(layout, dtype, lens, hq, hkv, m, d, page=16, seed=0):
    """q, per-sequence K and V [n, hkv, d] (cpu), trees, and the call's arguments."""
    ks = [randn(n, hkv, d, dtype=dtype, seed=seed + 10 * b + 1) for b, n in enumerate(lens)]
    vs = [randn(n, hkv, d, dtype=dtype, seed=seed + 10 * b + 2) for b, n in enumerate(lens)]
    q = randn(len(lens), hq, m, d, dtype=dtype, seed=seed).cuda()
    t = torch.stack([random_tree(m, seed + b) for b in range(len(lens))])
    if layout == "dense":
        assert len(set(lens)) == 1
        return q, ks, vs, t, [torch.stack(x).transpose(1, 2).cuda() for x in (ks, vs)], {}
    if layout == "ragged":
        ip = i32([0] + lens).cumsum(0).to(torch.int32)
        return q, ks, vs, t, [torch.cat(x).cuda() for x in (ks, vs)], dict(kv_indptr=ip)
    pools, tables = [], []
    for i, xs in enumerate((ks, vs)):
        table, pages = pages_of(lens, page, seed + i)
        pool = torch.full((pages, page, hkv, d), math.nan, dtype=dtype)
        for b, x in enumerate(xs):
            at = torch.arange(lens[b])
            pool[table[b].long()[at // page], at % page] = x
        pools.append(pool.cuda())
        tables.append(table.cuda())
    return q, ks, vs, t, pools, dict(kv_indptr=i32(lens), k_block_table=tables[0],
                                     v_block_table=tables[1], kv_page_size=page)


def verify(o, q, ks, vs, trees):
    b, hq, m, d = q.shape
    hkv = ks[0].shape[1]
    for x in range(b):
        n = ks[x].shape[0]
        sees = visible(n, m, False, trees[x])
        for h in range(hq):
            g = h // (hq // hkv)
            want, bound = attention64(q[x, h].double().cpu(), ks[x][:, g].double(),
                                      vs[x][:, g].double(), sees, d ** -0.5, q.dtype)
            check(o[x, h], want, bound, f"sequence {x} ({n} keys), head {h}")


@pytest.mark.parametrize("layout", ["dense", "ragged", "paged"])
@pytest.mark.parametrize("dtype,lens,hq,hkv,m,d,page", [
    (BF, [100, 100], 4, 2, 5, 128, 16),
    (F16, [65, 65, 65], 2, 2, 1, 64, 16),
    (BF, [300, 300], 8, 2, 16, 64, 5),       # 64 rows
    (F16, [130, 130], 8, 1, 13, 128, 8),     # 104 rows
    (BF, [700], 8, 2, 64, 128, 16),          # two q-blocks
    (BF, [90, 90], 4, 4, 33, 256, 24),
    (F16, [64, 64], 6, 2, 61, 256, 64),
    (BF, [20, 20], 4, 2, 37, 64, 16),        # fewer keys than drafts
    (F16, [0, 0], 2, 1, 3, 128, 16),         # no keys
])
def test_layouts(path, layout, dtype, lens, hq, hkv, m, d, page):
    q, ks, vs, t, (k, v), kw = make(layout, dtype, lens, hq, hkv, m, d, page)
    if layout == "paged" and not sum(lens):
        kw["k_block_table"], kw["v_block_table"] = (torch.zeros(2, 1, dtype=torch.int32,
                                                                device="cuda"),) * 2
    o = kernels.tree_decode_attention(q, k, v, t.cuda(), **kw)
    assert o.shape == q.shape and o.is_contiguous()
    verify(o, q, ks, vs, t)


@pytest.mark.parametrize("layout", ["ragged", "paged"])
@pytest.mark.parametrize("lens,hq,hkv,m,d", [
    ([1, 0, 31, 32, 33, 63, 64, 65, 129], 4, 2, 7, 128),
    ([2500, 40, 3100, 16], 8, 2, 16, 128),   # units cut by segments
    ([1500, 900], 8, 8, 13, 64), ([5000], 16, 1, 61, 128), ([2000, 17], 8, 2, 20, 256),
    ([100 + i for i in range(150)], 2, 2, 3, 64),
    ([30] * 66 + [2600, 0, 900], 4, 2, 24, 128),  # more than a wave's lanes, units cut
    ([2600] + [64] * 70, 8, 1, 17, 64),
])
def test_lengths(layout, lens, hq, hkv, m, d):
    q, ks, vs, t, (k, v), kw = make(layout, BF, lens, hq, hkv, m, d)
    verify(kernels.tree_decode_attention(q, k, v, t.cuda(), **kw), q, ks, vs, t)


def test_windows_and_long_tables():
    """More block-table entries than LDS holds; pages of one row."""
    q, ks, vs, t, (k, v), kw = make("paged", F16, [2600, 1], 2, 1, 4, 64, page=1)
    verify(kernels.tree_decode_attention(q, k, v, t.cuda(), **kw), q, ks, vs, t)


def test_chain_is_speculative_decode(path):
    """The lower triangle is speculative_decode_attention's causal mask."""
    for dtype in (BF, F16):
        for m, hq, hkv, d in ((8, 8, 2, 128), (16, 4, 4, 64)):
            q, ks, vs, _, (k, v), kw = make("paged", dtype, [300, 77, 1000], hq, hkv, m, d)
            # (that call reads the rows behind a sequence's end under a zero weight)
            k, v = k.nan_to_num(), v.nan_to_num()
            chain = torch.ones(m, m, dtype=torch.bool, device="cuda").tril()
            o = kernels.tree_decode_attention(q, k, v, chain, **kw)
            verify(o, q, ks, vs, [chain.cpu()] * 3)
            s = kernels.speculative_decode_attention(q, k, v, causal=True, **kw)
            verify(s, q, ks, vs, [chain.cpu()] * 3)


def test_same_bits(path):
    """Strided queries, K/V and masks, 3-D caches, wide types, entries outside the caches
    behind the end, another stream, graphs, workspaces of any content."""
    lens, m = [300, 2100, 64], 9
    q, ks, vs, t, (k, v), kw = make("paged", BF, lens, 8, 2, m, 128)
    t = t.cuda()

    def call(q=q, k=k, v=v, t=t, **more):
        return kernels.tree_decode_attention(q, k, v, t, **{**kw, **more})
    ref = call()
    verify(ref, q, ks, vs, t.cpu())
    assert torch.equal(call(q=q.transpose(1, 2).contiguous().transpose(1, 2)), ref)
    assert torch.equal(call(k=k.flatten(0, 1), v=v.flatten(0, 1)), ref)
    kv = torch.cat([k, v], 2)  # K and V side by side in one pool
    assert torch.equal(call(k=kv[:, :, :2], v=kv[:, :, 2:], k_block_table=kw["k_block_table"]), ref)
    assert torch.equal(call(t=t.to(torch.uint8) * 3), ref)
    assert torch.equal(call(t=t.transpose(1, 2).contiguous().transpose(1, 2)), ref)
    wide = {n: torch.nn.functional.pad(kw[n].long(), (0, 9), value=2 ** 40)
            for n in ("k_block_table", "v_block_table")}
    assert torch.equal(call(kv_indptr=kw["kv_indptr"].long(), **wide), ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = call()
    b = call()
    torch.cuda.synchronize()
    assert torch.equal(a, ref) and torch.equal(b, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        out.zero_()
        graph.replay()
        other = call()
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and torch.equal(other, ref), i
    for fill in (0, 255):
        ws = torch.full((2 ** 27,), fill, dtype=torch.uint8, device="cuda")
        got = tree_mod._run("x", q, k, v, t, _fa2.LAYOUT_PAGED, kw["kv_indptr"],
                            kw["k_block_table"], kw["v_block_table"], 16, workspace=ws)
        assert torch.equal(got, ref)
    # one mask for all sequences
    assert torch.equal(call(t=t[1]), call(t=t[1].expand(3, -1, -1)))


def test_empty_rows(path):
    """A mask row without drafts sees the context, or nothing where there is none."""
    q, ks, vs, _, (k, v), kw = make("ragged", F16, [6, 40], 4, 2, 6, 128)
    t = torch.zeros(2, 6, 6, dtype=torch.bool)
    t[:, 2, 4] = True  # (not a tree: any mask is taken)
    o = kernels.tree_decode_attention(q, k, v, t.cuda(), **kw)
    verify(o, q, ks, vs, t)
    assert o[0, :, 0].isnan().all() and not o[0, :, 2].isnan().any() and not o[1].isnan().any()


def test_pool_past_4_gib():
    page, hkv, d, m = 64, 8, 128, 4
    pages = (2 ** 32 + 2 ** 28) // (page * hkv * d * 2)
    pool = torch.zeros(pages, page, hkv, d, dtype=BF, device="cuda")
    table = i32([[pages - 1, pages - 2]])
    ks = randn(70, hkv, d, dtype=BF, seed=1)
    pool[pages - 1], pool[pages - 2, :6] = ks[:64].cuda(), ks[64:].cuda()
    q = randn(1, 8, m, d, dtype=BF).cuda()
    t = random_tree(m, 3)
    o = kernels.tree_decode_attention(q, pool, pool, t.cuda(), kv_indptr=i32([70]),
                                      k_block_table=table, v_block_table=table, kv_page_size=page)
    verify(o, q, [ks], [ks], [t])


def test_refusals(path):
    q, ks, vs, t, (k, v), kw = make("paged", BF, [40, 40], 8, 2, 5, 128)
    qd, _, _, _, (kd, vd), _ = make("dense", BF, [40, 40], 8, 2, 5, 128)
    t = t.cuda()

    def call(q=q, k=k, v=v, t=t, **more):
        return kernels.tree_decode_attention(q, k, v, t, **{**kw, **more})
    cases = [
        (AssertionError, dict(q=q.half())), (AssertionError, dict(v=v.cpu())),
        (TypeError, dict(q=q.float(), k=k.float(), v=v.float())), (ValueError, dict(q=q[0])),
        (ValueError, dict(q=q[..., :96], k=k[..., :96], v=v[..., :96])),
        (ValueError, dict(q=q[..., :64])), (ValueError, dict(v=v[:, :, :1])),
        (ValueError, dict(q=q[:, :7])), (ValueError, dict(q=q[:, :0])),
        (AssertionError, dict(v_block_table=None)), (AssertionError, dict(kv_page_size=None)),
        (AssertionError, dict(kv_indptr=None)), (ValueError, dict(kv_page_size=8)),
        (ValueError, dict(kv_page_size=0)), (ValueError, dict(kv_indptr=kw["kv_indptr"][:1])),
        (ValueError, dict(k_block_table=kw["k_block_table"][:1])),
        (ValueError, dict(v_block_table=kw["v_block_table"][0])),
        (TypeError, dict(t=t.float())), (ValueError, dict(t=t[:1])), (ValueError, dict(t=t[0, :3])),
        (AssertionError, dict(t=t.cpu())), (AssertionError, dict(kv_indptr=kw["kv_indptr"].cpu())),
        (ValueError, dict(q=torch.zeros(2, 8, 65, 128, dtype=BF, device="cuda"),
                          t=torch.ones(65, 65, dtype=torch.bool, device="cuda"))),
    ]
    for err, more in cases:
        with pytest.raises(err):
            call(**more)
    with pytest.raises(ValueError):
        kernels.tree_decode_attention(qd[:1], kd, vd, t[0])
    with pytest.raises(ValueError):
        kernels.tree_decode_attention(qd, kd, vd, t, kv_indptr=i32([0, 40, 80]))
    with pytest.raises(ValueError):
        kernels.tree_decode_attention(qd, kd[0].transpose(0, 1), vd[0].transpose(0, 1), t,
                                      kv_indptr=i32([0, 40]))
    with pytest.raises(RuntimeError):  # caches of less than a page
        kernels.tree_decode_attention(q, k.flatten(0, 1)[:8], v.flatten(0, 1)[:8], t, **kw)


def test_serving_loop():
    """A layer of a latent-attention model: prompts prefilled in the expanded form, a
    decode step and a step that verifies trees of drafts in the absorbed form, all from one
    cache; the absorbed results, projected, are the expanded ones."""
    h, d, latent, page, b = 16, 128, 512, 16, 3
    dtype, scale = BF, 192 ** -0.5
    g = torch.Generator().manual_seed(5)
    w_k = (torch.randn(latent, h, d, generator=g) / latent ** 0.5).to(dtype).cuda()
    w_v = (torch.randn(latent, h, d, generator=g) / latent ** 0.5).to(dtype).cuda()
    weight = torch.ones(latent, dtype=dtype, device="cuda")
    rope = kernels.build_rope_table(512, 64, device="cuda")
    m = 5
    lens, steps = [70, 1, 130], [1, m]
    table, pages = pages_of([n + 1 + m for n in lens], page, 0)
    cache, bt = kernels.allocate_latent_cache(pages, page, latent, dtype), table.cuda()
    trees = torch.stack([random_tree(m, x) for x in range(b)])
    x = [randn(n + 1 + m, latent + 64, dtype=dtype, seed=n).cuda() for n in lens]
    qs = [randn(n + 1 + m, h, d + 64, dtype=dtype, seed=n + 1).cuda() for n in lens]

    def append(lo, counts, rows=False):
        ip = i32([0] + counts).cumsum(0).to(torch.int32)
        new = torch.cat([x[i][lo[i]:lo[i] + counts[i]] for i in range(b)])
        return ip, kernels.paged_latent_append(cache, bt, new, ip, weight, rope, i32(lo),
                                               return_rows=rows)

    def up(rows):  # keys and values of the heads
        c = rows[:, :latent]
        return (torch.matmul(c, w_k.flatten(1)).unflatten(1, (h, d)),
                torch.matmul(c, w_v.flatten(1)).unflatten(1, (h, d)))

    # the prompts
    ip, rows = append([0] * b, lens, rows=True)
    k, v = up(rows)
    o = kernels.latent_attention(torch.cat([q[:n] for q, n in zip(qs, lens)]), k, rows[:, latent:],
                                 v, True, q_indptr=ip, kv_indptr=ip)
    every = [rows[ip[i]:ip[i + 1]] for i in range(b)]
    for i in range(b):
        want = reference(qs[i][:lens[i]], every[i], w_k, w_v, scale,
                         visible(lens[i], lens[i], True, None))
        close(o[ip[i]:ip[i + 1]], want)
    # one token, then a tree of drafts
    at = list(lens)
    for count in steps:
        _, rows = append(at, [count] * b, rows=True)
        every = [torch.cat([e, rows[i * count:(i + 1) * count]]) for i, e in enumerate(every)]
        q = torch.stack([qs[i][at[i]:at[i] + count] for i in range(b)]).transpose(1, 2)
        absorbed = torch.matmul(q[..., :d].transpose(0, 1).flatten(1, 2),
                                w_k.permute(1, 2, 0).contiguous())
        absorbed = torch.cat([absorbed.unflatten(1, (b, count)).transpose(0, 1), q[..., d:]], -1)
        at = [n + count for n in at]
        f = dict(latent_dim=latent, softmax_scale=scale, kv_indptr=i32(at), block_table=bt)
        if count == 1:
            o = kernels.latent_decode_attention(absorbed[:, :, 0], cache, **f).unsqueeze(2)
        else:
            o = kernels.latent_decode_attention(absorbed, cache, tree_mask=trees.cuda(), **f)
        heads = torch.matmul(o.transpose(0, 1).flatten(1, 2), w_v.transpose(0, 1).contiguous())
        heads = heads.unflatten(1, (b, count)).transpose(0, 1)  # [b, h, count, d]
        for i in range(b):
            want = reference(q[i].transpose(0, 1), every[i], w_k, w_v, scale,
                             visible(at[i], count, False, trees[i] if count > 1 else None))
            close(heads[i].transpose(0, 1), want)


def reference(q, rows, w_k, w_v, scale, sees):
    """[m, h, d] in 64 bits, from the cached rows and the projections themselves."""
    rows, q = rows.double().cpu(), q.double().cpu()
    latent = w_k.shape[0]
    out = torch.empty(q.shape[0], q.shape[1], w_v.shape[2], dtype=torch.float64)
    for h in range(q.shape[1]):
        keys = torch.cat([rows[:, :latent] @ w_k[:, h].double().cpu(), rows[:, latent:]], -1)
        p = ((q[:, h] @ keys.T) * scale).masked_fill(~sees, -math.inf).softmax(-1)
        out[:, h] = p @ (rows[:, :latent] @ w_v[:, h].double().cpu())
    return out


def close(got, want):
    """Chains of bf16 roundings: the projected keys (or queries), values (or outputs)
    and the weights, 2^-8 of the row's size each at most; scores of about 1 move by
    2^-8 of the keys' size, 2 sqrt(d) 2^-8 at scale d^-1/2."""
    got = got.double().cpu()
    size = want.abs().amax(-1, keepdim=True)
    assert ((got - want).abs() <= 16 * 2.0 ** -8 * size).all()
