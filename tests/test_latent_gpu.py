"""Latent attention on the GPU: the cache's writer, the absorbed and the expanded form,
against the 64-bit restatements of tests/latent_ref.py (whose bounds count roundings)."""

import importlib
import math

import pytest
import torch

import kernels
from kernels import _latent
from latent_ref import attention64, check, finished_rows64, pages_of, random_tree, visible

pytestmark = pytest.mark.gpu

cache_mod = importlib.import_module("kernels.latent_cache")
decode_mod = importlib.import_module("kernels.latent_decode")
attn_mod = importlib.import_module("kernels.latent_attention")
BF, F16 = torch.bfloat16, torch.float16


def randn(*shape, dtype=torch.float32, seed=0, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return (size * torch.randn(shape, generator=g)).to(dtype)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.fixture(params=[True, False], ids=["ext", "ctypes"])
def path(request, monkeypatch):
    """Both launch paths."""
    for m in (cache_mod, decode_mod, attn_mod):
        monkeypatch.setattr(m, "USE_EXT", request.param)
    return request.param


# ---- the writer ----------------------------------------------------------------------

def append_case(latent, dtype, lens, starts, page, *, inter=False, w32=False, seed=0, stride=0,
                positions=4096, spare_rows=3):
    width = latent + 64
    t = sum(lens) + spare_rows  # rows behind the last sequence
    x = randn(t, width + stride, dtype=dtype, seed=seed).cuda()[:, :width]
    w = (1 + 0.1 * randn(latent, seed=seed + 1)).to(torch.float32 if w32 else dtype).cuda()
    rope = kernels.build_rope_table(positions, 64, device="cuda")
    table, pages = pages_of([a + b for a, b in zip(starts, lens)], page, seed + 2)
    cache = randn(pages, page, width, dtype=dtype, seed=seed + 3).cuda()
    ip = i32([0] + lens).cumsum(0).to(torch.int32)
    return x, w, rope, table, cache, ip


def append_check(x, w, rope, table, before, cache, rows, lens, starts, page, inter, eps=1e-6):
    dtype = cache.dtype
    u = torch.finfo(dtype).eps / 2
    want = before.double().cpu()
    bound = torch.zeros_like(want)
    done, seen = [], []
    t0 = 0
    for b, n in enumerate(lens):
        pos = torch.arange(starts[b], starts[b] + n)
        y, size = finished_rows64(x[t0:t0 + n].double().cpu(), w.double().cpu(),
                                  rope.double().cpu(), pos, eps, inter)
        # u for the result; the sum of squares of up to 512 values, its root and three
        # products: 600 half steps of fp32 at most, of the terms of a rotation too
        lim = u * y.abs() + 600 * 2.0 ** -24 * size + torch.finfo(dtype).smallest_normal * u * 2
        at = table[b].long()[pos // page], pos % page
        want[at], bound[at] = y, 1.01 * lim
        done.append(y)
        seen.append(1.01 * lim)
        t0 += n
    check(cache, want, bound, "cache")
    if rows is not None:
        check(rows[:t0], torch.cat(done), torch.cat(seen), "rows")


@pytest.mark.parametrize("latent,dtype,lens,starts,page,inter,w32,stride", [
    (512, BF, [1], [0], 16, False, False, 0),
    (512, BF, [1] * 64, list(range(5, 69)), 16, False, False, 512),
    (256, F16, [1, 0, 3, 17, 0], [0, 4, 15, 100, 2], 16, True, False, 8),
    (512, F16, [130, 1, 0, 61], [7, 0, 3, 1000], 5, False, True, 64),
    (256, BF, [2, 33, 64, 1, 1], [31, 32, 0, 63, 64], 32, True, True, 0),
    (256, BF, [1, 0, 2] * 40, [3, 1, 9] * 40, 1, False, False, 0),       # 120 sequences
    (512, BF, [0, 1, 0, 0, 2] * 1000, [1, 2, 0, 4, 5] * 1000, 8, False, False, 0),  # 5000
])
def test_append(path, latent, dtype, lens, starts, page, inter, w32, stride):
    x, w, rope, table, cache, ip = append_case(latent, dtype, lens, starts, page, w32=w32,
                                               stride=stride)
    before = cache.clone()
    rows = kernels.paged_latent_append(cache, table.cuda(), x, ip, w, rope, i32(starts),
                                       interleaved=inter, return_rows=True)
    append_check(x, w, rope, table, before, cache, rows, lens, starts, page, inter)
    again = before.clone()
    assert kernels.paged_latent_append(again, table.cuda(), x, ip, w, rope, i32(starts),
                                       interleaved=inter) is None
    assert torch.equal(again, cache)


def test_append_places(path):
    """No starts; positions without a page, outside the pool or past the rope table; wide
    index types; no rows and no sequences."""
    lens, page = [40, 3, 2], 16
    x, w, rope, table, cache, ip = append_case(512, BF, lens, [0, 0, 0], page, positions=35)
    table[0, 1] = -1                 # rows 16 .. 31 of the first sequence
    table[1, 0] = cache.shape[0]     # the second one
    before = cache.clone()
    rows = kernels.paged_latent_append(cache, table.cuda(), x, ip, w, rope, return_rows=True)
    want = before.clone()
    want[table[0, 0].long()] = rows[:16]
    want[table[0, 2].long(), :8] = rows[32:40]
    want[table[2, 0].long(), :2] = rows[43:45]
    assert torch.equal(cache.view(torch.int16), want.view(torch.int16))
    assert rows[35:40].isnan().all() and not rows[:35].isnan().any()  # no such position
    # a table one page wide: the rest has no place; indices past 32 bits stay outside
    for t in (table[:, :1].clone(), table[:, :1].long() + 2 ** 32):
        c = before.clone()
        kernels.paged_latent_append(c, t.cuda(), x, ip.long(), w, rope)
        want = before.clone()
        if t.dtype == torch.int32:
            want[table[0, 0].long()] = rows[:16]
            want[table[2, 0].long(), :2] = rows[43:45]
        assert torch.equal(c, want)
    c = before.clone()
    kernels.paged_latent_append(c, table.cuda(), x, ip, w, rope, i32([-50, -3, 2 ** 30]))
    assert torch.equal(c, before)
    kernels.paged_latent_append(c, table.cuda(), x[:0], ip * 0, w, rope)
    kernels.paged_latent_append(c, table[:0].cuda(), x, ip[:1], w, rope)
    assert torch.equal(c, before)


def test_append_before_the_first_sequence(path):
    """Prefix sums that start past row 0: the rows before are nobody's."""
    x, w, rope, table, cache, ip = append_case(256, F16, [4, 5], [0, 2], 16)
    whole, part = cache.clone(), cache.clone()
    kernels.paged_latent_append(whole, table.cuda(), x[2:], ip, w, rope, i32([0, 2]))
    kernels.paged_latent_append(part, table.cuda(), x, ip + 2, w, rope, i32([0, 2]))
    assert torch.equal(whole, part)


def test_append_past_4_gib():
    """Pages whose bytes lie past 32 bits."""
    page, width = 64, 576
    pages = (2 ** 32 + 2 ** 28) // (page * width * 2)
    cache = torch.zeros(pages, page, width, dtype=BF, device="cuda")
    table = i32([[pages - 1], [pages - 3]])
    x, w, rope, _, _, _ = append_case(512, BF, [3, 2], [5, 0], page)
    rows = kernels.paged_latent_append(cache, table, x, i32([0, 3, 5]), w, rope, i32([5, 0]),
                                       return_rows=True)
    assert torch.equal(cache[pages - 1, 5:8], rows[:3])
    assert torch.equal(cache[pages - 3, :2], rows[3:5])
    assert int((cache[pages - 4:] != 0).any(-1).sum()) == 5
    q = randn(2, 16, width, dtype=BF).cuda()
    o = kernels.latent_decode_attention(q, cache, latent_dim=512, softmax_scale=0.1,
                                        kv_indptr=i32([7, 2]), block_table=table)
    for b, n in enumerate((7, 2)):
        rows64 = cache[table[b, 0], :n].double().cpu()
        want, bound = attention64(q[b].double().cpu(), rows64, rows64[:, :512],
                                  torch.ones(16, n, dtype=torch.bool), 0.1, BF)
        check(o[b], want, bound)


# ---- the absorbed form -----------------------------------------------------------------

def decode_case(latent, dtype, lens, hq, m, page, *, seed=0, tree=False, size=1.0, width=0,
                head_major=False, shared=False, fill=-1):
    table, pages = pages_of(lens, page, seed, width=width, fill=fill)
    cache = randn(pages, page, latent + 64, dtype=dtype, seed=seed + 1, size=size)
    # what lies behind a sequence's end, and pages of nobody, are NaN
    held = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        at = torch.arange(n)
        held[table[b].long()[at // page], at % page] = True
    cache[~held] = math.nan
    dims = (len(lens), hq, m, latent + 64) if m else (len(lens), hq, latent + 64)
    q = randn(*dims, dtype=dtype, seed=seed + 2).cuda()
    if head_major:  # as a product over the heads leaves them
        q = q.transpose(0, 1).contiguous().transpose(0, 1)
    t = None
    if tree:
        t = torch.stack([random_tree(m, seed + 3 + b) for b in range(1 if shared else len(lens))])
        t = t[0] if shared else t
    return q, cache, table, t


def decode_check(o, q, cache, table, lens, latent, scale, causal, tree, page):
    q4 = q.unsqueeze(2) if q.dim() == 3 else q
    o4 = o.unsqueeze(2) if o.dim() == 3 else o
    m = q4.shape[2]
    for b, n in enumerate(lens):
        at = torch.arange(n)
        rows = cache[table[b].long()[at // page], at % page].double()
        t = None if tree is None else tree if tree.dim() == 2 else tree[b]
        sees = visible(n, m, causal, t)
        x = q4[b].transpose(0, 1).double().cpu()  # [m, hq, width]
        for i in range(m):
            want, bound = attention64(x[i], rows, rows[:, :latent],
                                      sees[i].expand(x.shape[1], -1), scale, q.dtype)
            check(o4[b, :, i], want, bound, f"sequence {b} ({n} keys), token {i}")


@pytest.mark.parametrize("latent,dtype,lens,hq,m,page,causal,tree", [
    (512, BF, [1], 16, 0, 16, False, False),
    (512, F16, [0, 31, 32, 33, 64, 65], 16, 0, 16, False, False),
    (512, BF, [5, 700], 1, 0, 16, False, False),
    (512, BF, [300, 17, 1000], 33, 0, 5, False, False),
    (512, F16, [300, 0, 777], 64, 0, 64, False, False),
    (512, BF, [900, 63], 128, 0, 16, False, False),
    (512, BF, [129, 500], 65, 0, 24, False, False),
    (256, F16, [1, 500, 2000], 16, 0, 16, False, False),
    (256, BF, [1, 95, 96, 97], 40, 0, 32, False, False),
    (256, F16, [333, 1200], 128, 0, 7, False, False),
    (512, BF, [3, 100, 650], 16, 3, 16, True, False),
    (512, BF, [2, 100, 650], 16, 5, 16, False, False),   # fewer keys than tokens
    (512, F16, [2, 0, 300, 64], 128, 2, 16, True, False),
    (512, BF, [70, 300], 24, 16, 16, True, False),       # 384 rows
    (256, BF, [5, 65, 400], 32, 6, 16, False, True),
    (512, F16, [40, 33, 300], 8, 31, 8, False, True),
    (512, BF, [64, 100, 64], 2, 64, 16, False, True),
    (256, F16, [10, 200], 3, 37, 1, False, True),        # fewer keys than drafts
    (256, BF, [90, 513], 4, 200, 16, True, False),       # a chunk of a prompt
])
def test_decode(path, latent, dtype, lens, hq, m, page, causal, tree):
    q, cache, table, t = decode_case(latent, dtype, lens, hq, m, page, tree=tree)
    o = kernels.latent_decode_attention(q, cache.cuda(), latent_dim=latent, softmax_scale=0.072,
                                        kv_indptr=i32(lens), block_table=table.cuda(),
                                        causal=causal, tree_mask=t.cuda() if tree else None)
    assert o.shape == q.shape[:-1] + (latent,) and o.is_contiguous()
    decode_check(o, q, cache, table, lens, latent, 0.072, causal, t, page)


@pytest.mark.parametrize("lens,hq,page", [
    ([3000, 100, 2500, 1], 16, 16),           # units cut by segments
    ([4097], 128, 16), ([20000], 16, 16), ([9000], 16, 3),  # windows of block-table entries
    ([600, 40, 1300, 90] * 70, 16, 16),       # more sequences than CUs
    ([40] * 66 + [2600, 0, 1, 900], 48, 16),  # more than a wave's lanes, units cut
    ([70] * 65 + [3000], 128, 16),
])
def test_decode_shares(lens, hq, page):
    q, cache, table, _ = decode_case(256, BF, lens, hq, 0, page)
    o = kernels.latent_decode_attention(q, cache.cuda(), latent_dim=256, softmax_scale=0.072,
                                        kv_indptr=i32(lens), block_table=table.cuda())
    decode_check(o, q, cache, table, lens, 256, 0.072, False, None, page)


@pytest.mark.parametrize("latent,hq", [(512, 16), (512, 128), (256, 64)])
def test_decode_layouts(path, latent, hq):
    """Head-major queries, one tree for all, byte masks, strided masks, wide tables of
    any fill, lengths past the table, 64-bit indices: the same bits."""
    lens, page = [300, 61, 150], 16
    q, cache, table, t = decode_case(latent, BF, lens, hq, 4, page, tree=True, shared=True,
                                     width=40, fill=2 ** 31 - 1)
    c = cache.cuda()

    def call(q, tree, lens, table):
        return kernels.latent_decode_attention(q, c, latent_dim=latent, softmax_scale=0.05,
                                               kv_indptr=lens, block_table=table, tree_mask=tree)
    ref = call(q, t.cuda(), i32(lens), table.cuda())
    decode_check(ref, q, cache, table, lens, latent, 0.05, False, t, page)
    hm = q.permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3)
    assert torch.equal(call(hm, t.cuda(), i32(lens), table.cuda()), ref)
    wide = torch.zeros(len(lens), hq, 4, q.shape[-1] + 4, dtype=BF, device="cuda")
    wide[..., 2:-2] = q  # rows off 16 bytes: copied first
    assert torch.equal(call(wide[..., 2:-2], t.cuda(), i32(lens), table.cuda()), ref)
    per = t.expand(3, -1, -1).contiguous().cuda()
    assert torch.equal(call(q, per, i32(lens), table.cuda()), ref)
    assert torch.equal(call(q, per.to(torch.uint8) * 7, i32(lens), table.cuda()), ref)
    big = torch.zeros(3, 9, 9, dtype=torch.bool, device="cuda")
    big[:, 2:6, 3:7] = per
    assert torch.equal(call(q, big[:, 2:6, 3:7], i32(lens), table.cuda()), ref)
    assert torch.equal(call(q, per.transpose(1, 2).contiguous().transpose(1, 2), i32(lens),
                            table.cuda()), ref)
    assert torch.equal(call(q, t.cuda(), i32(lens).long(), table.long().cuda()), ref)
    # a chain of drafts is the lower triangle
    chain = kernels.latent_decode_attention(q, c, latent_dim=latent, softmax_scale=0.05,
                                            kv_indptr=i32(lens), block_table=table.cuda(),
                                            causal=True)
    assert torch.equal(call(q, torch.ones(4, 4, dtype=torch.bool).tril().cuda(), i32(lens),
                            table.cuda()), chain)
    # lengths past the table: what it holds
    short = table[:, :3].cuda()
    a = call(q, t.cuda(), i32([48, 48, 48]), short)
    assert torch.equal(call(q, t.cuda(), i32([300, 49, 2 ** 31 - 1]), short), a)


def test_decode_masks_and_ends(path):
    """Drafts that see nothing of a sequence without context; scores at the ends of the
    range; weights far below the largest."""
    q, cache, table, _ = decode_case(512, F16, [5, 69], 16, 5, 16)
    t = torch.zeros(2, 5, 5, dtype=torch.bool)
    t[0, 1:, 1] = True
    o = kernels.latent_decode_attention(q, cache.cuda(), latent_dim=512, softmax_scale=0.05,
                                        kv_indptr=i32([5, 69]), block_table=table.cuda(),
                                        tree_mask=t.cuda())
    decode_check(o, q, cache, table, [5, 69], 512, 0.05, False, t, 16)
    assert o[0, :, 0].isnan().all() and not o[0, :, 1:].isnan().any()
    # one key far above 2000 others: they count 2^-20 each
    lens = [2001]
    q, cache, table, _ = decode_case(256, F16, lens, 16, 0, 16)
    flat = torch.zeros(2001, 320)
    flat[:, :256] = randn(2001, 256, seed=9)
    flat[:, 256] = 0.0
    flat[700, 256] = 20.0
    q[:] = 0
    q[..., 256] = 1.0
    at = torch.arange(2001)
    cache[table[0].long()[at // 16], at % 16] = flat.to(F16)
    for scale in (math.log(2.0), 2.0 ** -20, 60000.0):
        o = kernels.latent_decode_attention(q, cache.cuda(), latent_dim=256, softmax_scale=scale,
                                            kv_indptr=i32(lens), block_table=table.cuda())
        decode_check(o, q, cache, table, lens, 256, scale, False, None, 16)


def test_decode_nothing(path):
    q, cache, table, _ = decode_case(512, BF, [4, 4], 16, 0, 16)
    f = dict(latent_dim=512, softmax_scale=0.1, kv_indptr=i32([4, 4]), block_table=table.cuda())
    assert kernels.latent_decode_attention(q[:0], cache.cuda(), **f).shape == (0, 16, 512)
    q4 = q.unsqueeze(2)
    assert kernels.latent_decode_attention(q4[:, :, :0], cache.cuda(), **f).shape == (2, 16, 0, 512)
    f["block_table"] = table[:, :0].cuda()
    assert kernels.latent_decode_attention(q, cache.cuda(), **f).isnan().all()
    f["block_table"], f["kv_indptr"] = table.cuda(), i32([-3, 0])
    assert kernels.latent_decode_attention(q, cache.cuda(), **f).isnan().all()


@pytest.mark.parametrize("latent,hq", [(512, 128), (512, 16), (256, 128)])
def test_decode_graph_streams_and_workspaces(latent, hq):
    """Captured and replayed with other work between, on another stream, two calls at
    once, in workspaces of any content: the same bits."""
    lens, page = [2500, 40, 3100, 700], 16
    q, cache, table, _ = decode_case(latent, BF, lens, hq, 0, page)
    c, li, bt = cache.cuda(), i32(lens), table.cuda()
    f = dict(latent_dim=latent, softmax_scale=0.07, kv_indptr=li, block_table=bt)
    ref = kernels.latent_decode_attention(q, c, **f)
    decode_check(ref, q, cache, table, lens, latent, 0.07, False, None, page)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            a = kernels.latent_decode_attention(q, c, **f)
    b = kernels.latent_decode_attention(q, c, **f)
    torch.cuda.synchronize()
    assert torch.equal(a, ref) and torch.equal(b, ref)
    graph = torch.cuda.CUDAGraph()
    out = [None, None]
    with torch.cuda.graph(graph):
        out[0] = kernels.latent_decode_attention(q, c, **f)
        out[1] = kernels.latent_decode_attention(q.flip(0), c, **f)
    for i in range(4):
        out[0].zero_()
        graph.replay()
        other = kernels.latent_decode_attention(q, c, **f)
        torch.cuda.synchronize()
        assert torch.equal(out[0], ref) and torch.equal(other, ref), i
    for fill in (0, 255, 1):
        ws = torch.full((2 ** 28,), fill, dtype=torch.uint8, device="cuda")
        got = decode_mod._run("x", q, c, latent, 0.07, li, bt, False, None, workspace=ws)
        assert torch.equal(got, ref)
    with pytest.raises(ValueError):
        decode_mod._run("x", q, c, latent, 0.07, li, bt, False, None, workspace=ws[:64])


# ---- the expanded form -----------------------------------------------------------------

def prefill_case(d, dtype, q_lens, kv_lens, h, seed=0):
    up = randn(sum(kv_lens), h, 2 * d, dtype=dtype, seed=seed).cuda()
    rows = randn(sum(kv_lens), 512 + 64, dtype=dtype, seed=seed + 1).cuda()
    q = randn(sum(q_lens), h, d + 64, dtype=dtype, seed=seed + 2).cuda()
    return q, up[..., :d], rows[:, 512:], up[..., d:]


def sees_of(m, n, mask):
    i, j = torch.arange(m)[:, None], torch.arange(n)
    if mask == "none":
        return torch.ones(m, n, dtype=torch.bool)
    return j <= i + (n - m if mask == "bottom_right" else 0)


def prefill_check(o, q, k, kr, v, q_lens, kv_lens, mask, scale):
    q0 = k0 = 0
    for m, n in zip(q_lens, kv_lens):
        sees = sees_of(m, n, mask)
        for h in range(q.shape[1]):
            keys = torch.cat([k[k0:k0 + n, h], kr[k0:k0 + n]], -1).double().cpu()
            want, bound = attention64(q[q0:q0 + m, h].double().cpu(), keys,
                                      v[k0:k0 + n, h].double().cpu(), sees, scale, q.dtype)
            check(o[q0:q0 + m, h], want, bound, f"{m} over {n}, head {h}")
        q0, k0 = q0 + m, k0 + n


MASKS = [("none", {}), ("top_left", dict(is_causal=True)),
         ("bottom_right", dict(is_causal=True, causal_alignment="bottom_right"))]


@pytest.mark.parametrize("mask,kw", MASKS, ids=[m for m, _ in MASKS])
@pytest.mark.parametrize("d,dtype,q_lens,kv_lens,h", [
    (128, BF, [1], [1], 1),
    (128, F16, [333], [333], 3),
    (64, BF, [1, 0, 129, 64, 0], [5, 9, 129, 200, 0], 4),
    (128, BF, [257, 3, 0, 128], [300, 0, 40, 1000], 2),   # keys missing, queries missing
    (64, F16, [40], [2500], 2),                            # splits
    (128, BF, [500, 600, 300, 700, 40], [500, 700, 300, 900, 1100], 24),  # units claimed
    (128, F16, [2] * 40, [30] * 40, 16),                   # a plan, one q-block each
    (64, BF, [1100, 30], [600, 90], 64),                   # pairs, some of one q-block
])
def test_prefill_ragged(path, d, dtype, q_lens, kv_lens, h, mask, kw):
    q, k, kr, v = prefill_case(d, dtype, q_lens, kv_lens, h)
    qi, ki = (i32([0] + x).cumsum(0).to(torch.int32) for x in (q_lens, kv_lens))
    o = kernels.latent_attention(q, k, kr, v, q_indptr=qi, kv_indptr=ki, **kw)
    assert o.shape == q.shape[:-1] + (d,)
    prefill_check(o, q, k, kr, v, q_lens, kv_lens, mask, (d + 64) ** -0.5)


@pytest.mark.parametrize("mask,kw", MASKS, ids=[m for m, _ in MASKS])
@pytest.mark.parametrize("b,h,m,n,d,dtype", [
    (1, 2, 1, 1, 128, BF), (2, 3, 100, 100, 64, F16), (3, 2, 65, 129, 128, BF),
    (1, 2, 40, 4500, 128, F16), (2, 4, 300, 260, 128, BF), (1, 1, 3, 0, 64, BF),
    (2, 48, 520, 333, 64, BF), (1, 88, 513, 600, 128, F16),  # pairs of q-blocks
])
def test_prefill_dense(path, b, h, m, n, d, dtype, mask, kw):
    q, k, kr, v = prefill_case(d, dtype, [m] * b, [n] * b, h)
    qd = q.unflatten(0, (b, m)).transpose(1, 2)
    kd, vd = (x.unflatten(0, (b, n)).transpose(1, 2) for x in (k, v))
    o = kernels.latent_attention(qd, kd, kr.unflatten(0, (b, n)), vd, softmax_scale=0.06, **kw)
    assert o.shape == (b, h, m, d)
    prefill_check(o.transpose(1, 2).flatten(0, 1), q, k, kr, v, [m] * b, [n] * b, mask, 0.06)


def test_prefill_graph_streams_and_layouts():
    q_lens, kv_lens = [300, 17], [300, 2600]
    q, k, kr, v = prefill_case(128, BF, q_lens, kv_lens, 4)
    qi, ki = (i32([0] + x).cumsum(0).to(torch.int32) for x in (q_lens, kv_lens))
    f = dict(is_causal=True, causal_alignment="bottom_right", q_indptr=qi, kv_indptr=ki)
    ref = kernels.latent_attention(q, k, kr, v, **f)
    prefill_check(ref, q, k, kr, v, q_lens, kv_lens, "bottom_right", 192 ** -0.5)
    off = torch.zeros(kr.shape[0], 68, dtype=BF, device="cuda")
    off[:, 2:66] = kr  # rows off 16 bytes: copied first
    assert torch.equal(kernels.latent_attention(q, k.contiguous(), off[:, 2:66], v, **f), ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = kernels.latent_attention(q, k, kr, v, **f)
    side.synchronize()
    assert torch.equal(a, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kernels.latent_attention(q, k, kr, v, **f)
    for i in range(4):
        out.zero_()
        graph.replay()
        other = kernels.latent_attention(q, k, kr, v, **f)
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and torch.equal(other, ref), i
    # rows behind the last sequence are left out
    more = torch.cat([q, q[:5]])
    assert torch.equal(kernels.latent_attention(more, k, kr, v, **f)[:317], ref)


@pytest.mark.parametrize("mask,kw", MASKS, ids=[m for m, _ in MASKS])
@pytest.mark.parametrize("q_lens,kv_lens,h", [
    ([130, 40], [300, 70], 2), ([20], [2700], 2), ([1100, 1000], [590, 610], 52),
])
def test_prefill_neighbours(q_lens, kv_lens, h, mask, kw):
    """What lies behind a sequence's rows is not seen: NaN between the sequences, ragged
    (a sequence of nobody's queries) and dense (views of longer tensors)."""
    d, gap = 64, 37
    kn, qn = sum(kv_lens) + gap * len(kv_lens), sum(q_lens)
    _, k, kr, v = prefill_case(d, BF, [1], [kn], h)
    q = randn(qn, h, d + 64, dtype=BF, seed=4).cuda()
    at, held = 0, torch.zeros(kn, dtype=torch.bool, device="cuda")
    ki, qi = [0], [0]
    for m, n in zip(q_lens, kv_lens):
        held[at:at + n] = True
        at += n + gap
        ki += [at - gap, at]
        qi += [qi[-1] + m] * 2
    for x in (k, kr, v):
        x[~held] = math.nan
    o = kernels.latent_attention(q, k, kr, v, q_indptr=i32(qi), kv_indptr=i32(ki), **kw)
    prefill_check(o, q, k[held], kr[held], v[held], q_lens, kv_lens, mask, 128 ** -0.5)
    m, n = q_lens[0], kv_lens[0]
    k, kr, v = k[:n + gap], kr[:n + gap], v[:n + gap]
    dense = kernels.latent_attention(q[None, :m].transpose(1, 2), k[None, :n].transpose(1, 2),
                                     kr[None, :n], v[None, :n].transpose(1, 2), **kw)
    prefill_check(dense[0].transpose(0, 1), q[:m], k, kr, v, [m], [n], mask, 128 ** -0.5)


# ---- refusals on the device, both paths ---------------------------------------------------

def test_refusals(path):
    q, cache, table, _ = decode_case(512, BF, [40, 9], 16, 3, 16)
    c, bt, li = cache.cuda(), table.cuda(), i32([40, 9])

    def dec(q=q, c=c, **kw):
        f = dict(latent_dim=512, softmax_scale=0.1, kv_indptr=li, block_table=bt)
        f.update(kw)
        return kernels.latent_decode_attention(q, c, **f)
    t = torch.ones(3, 3, dtype=torch.bool, device="cuda")
    for err, kw in [
        (ValueError, dict(q=q[0, 0])), (ValueError, dict(latent_dim=256)),
        (ValueError, dict(latent_dim=576)), (TypeError, dict(q=q.half())),
        (TypeError, dict(c=c.float(), q=q.float())), (ValueError, dict(q=q[..., :512])),
        (ValueError, dict(q=q[:, :0])), (ValueError, dict(kv_indptr=li[:1])),
        (ValueError, dict(block_table=bt[:1])), (ValueError, dict(block_table=bt[0])),
        (ValueError, dict(softmax_scale=0.0)), (ValueError, dict(softmax_scale=math.inf)),
        (ValueError, dict(c=c[:, :, :])) if False else (ValueError, dict(c=c[:, :8])),
        (ValueError, dict(c=c[:0])), (TypeError, dict(tree_mask=t.int())),
        (ValueError, dict(tree_mask=t[:2])), (ValueError, dict(tree_mask=t.expand(3, 3, 3))),
        (ValueError, dict(q=torch.zeros(2, 1, 65, 576, dtype=BF, device="cuda"),
                          tree_mask=torch.ones(65, 65, dtype=torch.bool, device="cuda"))),
        (AssertionError, dict(kv_indptr=li.cpu())), (AssertionError, dict(tree_mask=t.cpu())),
    ]:
        with pytest.raises(err):
            dec(**kw)
    x, w, rope, table, cache, ip = append_case(512, BF, [4], [0], 16)
    bt = table.cuda()

    def app(cache=cache, bt=bt, x=x, ip=ip, w=w, rope=rope, sp=None, **kw):
        return kernels.paged_latent_append(cache, bt, x, ip, w, rope, sp, **kw)
    for err, kw in [
        (TypeError, dict(cache=cache.float(), x=x.float())), (TypeError, dict(x=x.half())),
        (ValueError, dict(x=x[:, :512])), (ValueError, dict(cache=cache[..., :512].contiguous())),
        (ValueError, dict(w=w[:256])), (TypeError, dict(w=w.half())),
        (TypeError, dict(rope=rope.half())), (ValueError, dict(rope=rope[:, :32])),
        (ValueError, dict(eps=-1.0)), (ValueError, dict(bt=bt[:0])), (ValueError, dict(ip=ip[:0])),
        (ValueError, dict(sp=i32([]))), (AssertionError, dict(ip=ip.cpu())),
        (ValueError, dict(cache=cache[:, :8])),
    ]:
        with pytest.raises(err):
            app(**kw)
    q, k, kr, v = prefill_case(128, BF, [5], [5], 2)
    ki = i32([0, 5])

    def pre(q=q, k=k, kr=kr, v=v, **kw):
        f = dict(q_indptr=ki, kv_indptr=ki)
        f.update(kw)
        return kernels.latent_attention(q, k, kr, v, **f)
    for err, kw in [
        (AssertionError, dict(k=k.half())), (TypeError, dict(zip(("q", "k", "kr", "v"),
                                                                 (x.float() for x in (q, k, kr, v))))),
        (ValueError, dict(kv_indptr=None)), (ValueError, dict(q_indptr=None)),
        (ValueError, dict(q_indptr=i32([0, 2, 5]))), (ValueError, dict(q=q[..., :128])),
        (ValueError, dict(kr=kr[:4])), (ValueError, dict(kr=kr[:, :32])),
        (ValueError, dict(v=v[:4])), (ValueError, dict(k=k[..., :32], v=v[..., :32])),
        (ValueError, dict(k=k[:, :1], v=v[:, :1])), (ValueError, dict(softmax_scale=-1.0)),
        (ValueError, dict(q_indptr=None, kv_indptr=None)),
        (AssertionError, dict(q_indptr=ki.cpu())),
    ]:
        with pytest.raises(err):
            pre(**kw)
