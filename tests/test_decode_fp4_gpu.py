"""decode_attention_fp4 and speculative_decode_attention_fp4 against the
attention over the cached values in 64 bits (bounds: fp4_ref).

The pools hold NaN scales and arbitrary codes wherever no sequence has a row, so a
read that counts a row too many shows."""

import math

import pytest
import torch

import fp4_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need an MI355X")


class Case:
    """A batch: queries, a cache of random codes and scales, shuffled tables."""

    def __init__(self, lens, QH, KVH, D, M, dtype, page, seed, spread=2, causal=False):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.page, self.causal, self.M = lens, page, causal, M
        B = len(lens)
        self.q = torch.randn(B, QH, max(M, 1), D, generator=g).to(dtype)
        need = [-(-n // page) for n in lens]
        pages, width = sum(need) + 2, max(need + [1])
        self.caches, self.tables = [], []
        for _ in range(2):
            codes = torch.randint(0, 256, (pages, KVH, page, D // 2), generator=g, dtype=torch.uint8)
            scales = torch.full((pages, KVH, page, D // 32), 255, dtype=torch.uint8)
            perm, t, at = torch.randperm(pages, generator=g), torch.full((B, width), -1), 0
            for b, n in enumerate(need):
                t[b, :n] = perm[at:at + n]
                at += n
                for i in range(n):
                    rows = min(page, lens[b] - i * page)
                    scales[t[b, i], :, :rows] = torch.randint(
                        127 - 2 - spread, 127 - 1, (KVH, rows, D // 32), generator=g,
                        dtype=torch.uint8)
            self.caches.append([codes, scales])
            self.tables.append(t.to(torch.int32))

    def dev(self):
        return dict(q=self.q.cuda() if self.M else self.q[:, :, 0].contiguous().cuda(),
                    k_cache=tuple(t.cuda() for t in self.caches[0]),
                    v_cache=tuple(t.cuda() for t in self.caches[1]),
                    kv_indptr=torch.tensor(self.lens, dtype=torch.int32).cuda(),
                    k_block_table=self.tables[0].cuda(), v_block_table=self.tables[1].cuda())

    def call(self, **kw):
        from kernels import decode_attention_fp4, speculative_decode_attention_fp4
        d = self.dev() | kw
        if self.M:
            return speculative_decode_attention_fp4(d.pop("q"), d.pop("k_cache"),
                                                    d.pop("v_cache"), causal=self.causal, **d)
        return decode_attention_fp4(d.pop("q"), d.pop("k_cache"), d.pop("v_cache"), **d)

    def values(self, b):
        out = []
        n = self.lens[b]
        at = torch.arange(n)
        for (codes, scales), t in zip(self.caches, self.tables):
            pg = t[b].long()[at // self.page] if n else at
            out.append(R.cached_values(codes[pg, :, at % self.page], scales[pg, :, at % self.page]))
        return out

    def check(self, out):
        out = out.cpu() if self.M else out.cpu().unsqueeze(2)
        for b in range(len(self.lens)):
            want, tol = R.attention(self.q[b], *self.values(b), self.causal)
            R.within(out[b], want, tol)


DTYPES = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("QH,KVH", [(1, 1), (8, 2), (5, 5), (16, 1), (24, 1), (40, 2)])
@pytest.mark.parametrize("page", [16, 5])
def test_small_lengths(dtype, D, QH, KVH, page):
    """Lengths of zero, one and around a block, a tile and a page."""
    c = Case([0, 1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 130], QH, KVH, D, 0, dtype, page, D + QH)
    c.check(c.call())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,QH,KVH,M", [(64, 8, 8, 8), (64, 8, 2, 3), (128, 4, 1, 5), (128, 8, 2, 16),
                                        (128, 3, 3, 16), (256, 4, 2, 7), (128, 16, 1, 2)])
@pytest.mark.parametrize("causal", [False, True])
def test_drafts(dtype, D, QH, KVH, M, causal):
    """Drafts, also where the sequence is shorter than they are (rows without
    keys), and at the ends of blocks and tiles."""
    lens = [0, 1, M - 1, M, M + 1, 16, 31, 32, 33, 47, 300]
    c = Case(lens, QH, KVH, D, M, dtype, 16, D + M, causal=causal)
    c.check(c.call())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,QH,KVH,M,page,lens", [
    (128, 8, 2, 0, 16, [5000, 1, 3100, 770]),       # pieces of cut units
    (128, 4, 1, 0, 64, [9001]),                      # one long sequence, many pieces
    (64, 8, 8, 0, 16, [2500] * 5),
    (256, 4, 1, 0, 32, [4100, 200]),
    (128, 8, 1, 4, 16, [3000, 40, 1500]),            # 32 rows
    (128, 24, 1, 4, 16, [2100, 64]),                 # q-blocks
    (64, 4, 2, 0, 1, [1700, 600]),                   # windows: more pages than the LDS table
    (128, 4, 2, 0, 3, [2000, 1999]),
    (64, 2, 1, 0, 16, [20000]),                      # more pages per piece than the LDS table?
    (128, 16, 16, 0, 16, [700 + 13 * i for i in range(40)]),  # whole units
])
def test_long(dtype, D, QH, KVH, M, page, lens):
    c = Case(lens, QH, KVH, D, M, dtype, page, 11, causal=bool(M))
    c.check(c.call())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("QH,KVH,M", [(24, 1, 0), (16, 4, 5), (8, 2, 8), (24, 1, 4), (34, 2, 1),
                                       (40, 1, 16)])
@pytest.mark.parametrize("page", [16, 5])
def test_wide_tables(dtype, D, QH, KVH, M, page):
    """More than 16 rows where the tables could hold many keys (q-blocks of 32 up to
    D128), and the same with tables of just the pages (q-blocks of 16)."""
    c = Case([0, 1, 33, 2000, M, 130, 1100], QH, KVH, D, M, dtype, page, 23, causal=bool(M))
    c.check(c.call())
    width = -(-(1 << 20) // (page * KVH))  # 7 * 2^14 tiles of 64 keys and more
    wide = [torch.full((7, width), -1, dtype=torch.int32) for _ in range(2)]
    for w, t in zip(wide, c.tables):
        w[:, :t.shape[1]] = t
    c.check(c.call(k_block_table=wide[0].cuda(), v_block_table=wide[1].cuda()))


@pytest.mark.parametrize("D,KVH,page,lens", [
    (128, 16, 16, [60 + 59 * (i * 7 % 50) for i in range(50)]),     # several units a workgroup
    (128, 1, 16, [2900 if i % 9 == 0 else 40 + i for i in range(70)]),  # more than 64 sequences
    (64, 16, 48, [2900 if i % 9 == 0 else 40 + i for i in range(66)]),
    (128, 2, 48, [5000, 100, 2047]),
    (256, 8, 16, [3000 if i % 5 == 0 else 7 * i for i in range(33)]),
    (64, 8, 16, [1030] * 16),                                       # equal units
    (128, 1, 16, [1030 + i for i in range(64)]),
    (64, 300, 16, [200, 1, 77, 640]),                               # more heads than CUs
])
def test_shares(D, KVH, page, lens):
    """Workgroups with several units and units with several workgroups."""
    c = Case(lens, 2 * KVH, KVH, D, 0, torch.bfloat16, page, 24)
    out = c.call().cpu().unsqueeze(2)
    for b in range(0, len(lens), 3):
        want, tol = R.attention(c.q[b], *c.values(b), False)
        R.within(out[b], want, tol)


@pytest.mark.parametrize("D", [64, 128])
def test_windows_inside_a_piece(D):
    """Units stay whole and span several windows of the LDS block table."""
    B = 200
    lens = [1200 + (7 * i) % 40 for i in range(B)]
    c = Case(lens, 4, 4, D, 0, torch.bfloat16, 2, 12)
    out = c.call().cpu().unsqueeze(2)
    for b in (0, 1, 99, 150, 199):
        want, tol = R.attention(c.q[b], *c.values(b), False)
        R.within(out[b], want, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_nan_blocks(dtype, D):
    """A NaN block of K makes the rows that see its key NaN, one of V 32 of their
    values; rows that do not see it are untouched."""
    M, lens = 4, [70, 64, 33, 900, 3]
    c = Case(lens, 4, 2, D, M, dtype, 16, 13, causal=True)

    def poison(which, b, n, head, block):
        codes, scales = c.caches[which]
        pg = c.tables[which][b, n // 16].item()
        scales[pg, head, n % 16, block] = 255

    poison(1, 0, 68, 0, D // 32 - 1)  # a draft that two drafts see
    poison(1, 0, 66, 1, 0)            # the first draft
    poison(1, 1, 63, 0, 1)            # the last one
    poison(1, 1, 10, 1, 1)            # a key that all see
    poison(0, 2, 31, 0, 0)            # K: the third draft
    poison(1, 3, 899, 1, 0)
    poison(1, 4, 2, 0, 0)
    c.check(c.call())


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_at_the_ends_of_the_type(dtype):
    """Largest scales: scores far past the exponent's range, outputs near the
    type's maximum; smallest scales."""
    c = Case([100, 333], 4, 2, 128, 0, dtype, 16, 14)
    top = 127 + 13 if dtype == torch.float16 else 127 + 60
    for codes, scales in c.caches:
        scales[scales != 255] = top
    c.check(c.call())
    low = 127 - 23 if dtype == torch.float16 else 127 - 100
    for codes, scales in c.caches:
        scales[scales != 255] = low
    c.check(c.call())


def test_lengths_past_the_table_and_bad_entries():
    """A length past the table's keys counts as those; entries outside the pool
    are read from inside it and change no other sequence."""
    c = Case([48, 20, 90], 4, 2, 128, 0, torch.bfloat16, 16, 15)
    d = c.dev()
    want = c.call()
    lens = torch.tensor([48, 20, 100000], dtype=torch.int32).cuda()
    full = Case([48, 20, 96], 4, 2, 128, 0, torch.bfloat16, 16, 15)
    full.caches, full.tables = c.caches, c.tables
    for codes, scales in full.caches:
        scales[scales == 255] = 126
    out = full.call(kv_indptr=lens)
    full.check(out)
    entries = torch.tensor([10 ** 9, -5, 2 ** 31 - 1, -2 ** 31, 7, 6], dtype=torch.int32)
    kt, vt = d["k_block_table"].clone(), d["v_block_table"].clone()
    kt[2] = vt[2] = entries.cuda()
    out = c.call(k_block_table=kt, v_block_table=vt)
    assert torch.equal(out[:2], want[:2])


def test_strides_and_index_types():
    from kernels import decode_attention_fp4, speculative_decode_attention_fp4
    c = Case([300, 41], 8, 2, 128, 3, torch.float16, 16, 16, causal=True)
    want, d = c.call(), c.dev()
    q = d["q"]
    tm = q.transpose(1, 2).contiguous().transpose(1, 2)       # token-major memory
    wide = torch.empty(2, 8, 3, 256, dtype=q.dtype, device="cuda")[..., :128].copy_(q)
    off = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape).copy_(q)
    tab = torch.cat([d["k_block_table"]] * 2, 1)[:, :d["k_block_table"].shape[1]]
    for x in (tm, wide, off):
        got = c.call(q=x, kv_indptr=d["kv_indptr"].long(), k_block_table=tab,
                     v_block_table=d["v_block_table"].long())
        assert got.shape == want.shape and got.is_contiguous() and torch.equal(got, want)
    one = speculative_decode_attention_fp4(q[:, :, 2:], d["k_cache"], d["v_cache"],
                                           **{n: d[n] for n in ("kv_indptr", "k_block_table",
                                                                "v_block_table")})
    sq = decode_attention_fp4(q[:, :, 2], d["k_cache"], d["v_cache"],
                              **{n: d[n] for n in ("kv_indptr", "k_block_table",
                                                   "v_block_table")})
    assert torch.equal(one[:, :, 0], sq)


@pytest.mark.parametrize("drafts", [False, True])
@pytest.mark.parametrize("bad", ["dims", "dtype", "head_dim", "heads", "lens", "rows", "v", "codes",
                                 "pages", "scales", "device", "drafts"])
def test_refusals(drafts, bad):
    """Each is refused on the host, with and without the extension."""
    import kernels.decode_fp4 as m
    c = Case([40, 3], 4, 2, 128, 3 if drafts else 0, torch.float16, 16, 25)
    d = c.dev()
    q, k, v = d.pop("q"), d.pop("k_cache"), d.pop("v_cache")
    if bad == "dims":
        q = q[0]
    elif bad == "dtype":
        q = q.float()
    elif bad == "head_dim":
        q = q[..., :64]
    elif bad == "heads":
        q = q[:, :3]
    elif bad == "lens":
        d["kv_indptr"] = d["kv_indptr"][:1]
    elif bad == "rows":
        d["v_block_table"] = d["v_block_table"][:1]
    elif bad == "v":
        v = None
    elif bad == "codes":
        v = (v[0].float(), v[1])
    elif bad == "pages":
        v = (v[0][1:], v[1][1:])
    elif bad == "scales":
        k = (k[0], k[1][..., :3])
    elif bad == "device":
        d["kv_indptr"] = d["kv_indptr"].cpu()
    elif not drafts:
        q = q.unsqueeze(2)
    else:
        q = q[:, :, :1].expand(-1, -1, 17, -1)
    call = m.speculative_decode_attention_fp4 if drafts else m.decode_attention_fp4
    for use in (True, False):
        m.USE_EXT = use
        try:
            with pytest.raises((ValueError, TypeError, AssertionError, RuntimeError)):
                call(q, k, v, **d)
        finally:
            m.USE_EXT = True
    torch.cuda.synchronize()


def test_empty_batch():
    from kernels import decode_attention_fp4
    c = Case([5], 4, 2, 64, 0, torch.float16, 16, 17)
    d = c.dev()
    out = decode_attention_fp4(d["q"][:0], d["k_cache"], d["v_cache"], kv_indptr=d["kv_indptr"][:0],
                               k_block_table=d["k_block_table"][:0],
                               v_block_table=d["v_block_table"][:0])
    assert out.shape == (0, 4, 64)


def test_offsets_past_32_bits():
    """Pages beyond 2^32 bytes of codes."""
    from kernels import allocate_fp4_cache, decode_attention_fp4
    H, D, page, pages = 8, 256, 64, 70000
    kc = allocate_fp4_cache(pages, page, H, D)
    g = torch.Generator().manual_seed(1)
    n = 100
    codes = torch.randint(0, 256, (2, H, page, D // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(124, 127, (2, H, page, D // 32), generator=g, dtype=torch.uint8)
    kc.codes[pages - 2:].copy_(codes)
    kc.scales[pages - 2:].copy_(scales)
    t = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32)
    q = torch.randn(1, 16, D, generator=g).to(torch.bfloat16)
    out = decode_attention_fp4(q.cuda(), kc, kc, kv_indptr=torch.tensor([n], device="cuda"),
                               k_block_table=t.cuda(), v_block_table=t.cuda())
    v = R.cached_values(codes, scales)[[1, 0]].transpose(1, 2).flatten(0, 1)[:n]
    want, tol = R.attention(q[0].unsqueeze(1), v, v, False)
    R.within(out[0].unsqueeze(1), want, tol)


def test_results_repeat_and_paths_agree():
    """Cut units: the same bits every time, without the extension, on another
    stream, with a dirty workspace, and in replays of a graph between eager
    calls; two graphs that share a pool."""
    import kernels.decode_fp4 as m
    c = Case([5000, 3, 2600], 8, 2, 128, 0, torch.bfloat16, 16, 18)
    d = c.dev()
    args = [d[n] for n in ("q", "k_cache", "v_cache")]
    kw = {n: d[n] for n in ("kv_indptr", "k_block_table", "v_block_table")}
    want = m.decode_attention_fp4(*args, **kw)
    for _ in range(5):
        assert torch.equal(m.decode_attention_fp4(*args, **kw), want)
    m.USE_EXT = False
    try:
        assert torch.equal(m.decode_attention_fp4(*args, **kw), want)
    finally:
        m.USE_EXT = True
    dirty = torch.full((1 << 28,), 0xA5, dtype=torch.uint8, device="cuda")
    flat = [t for p in (args[1], args[2]) for t in p]
    for _ in range(2):
        got = m._run("decode_attention_fp4", args[0], *flat, *kw.values(), False, workspace=dirty)
        assert torch.equal(got, want)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = m.decode_attention_fp4(*args, **kw)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got, want)
    graphs, held = [torch.cuda.CUDAGraph() for _ in range(2)], []
    pool = torch.cuda.graph_pool_handle()
    torch.cuda.synchronize()
    for gr in graphs:
        with torch.cuda.graph(gr, pool=pool):
            held.append(m.decode_attention_fp4(*args, **kw))
    for i in range(4):
        args[0].copy_(torch.randn(args[0].shape, generator=torch.Generator().manual_seed(i)))
        eager = m.decode_attention_fp4(*args, **kw)
        for gr, h in zip(graphs, held):
            gr.replay()
            got = h.clone()
            torch.cuda.synchronize()
            assert torch.equal(got, eager), i


def test_two_calls_at_once():
    """Two streams, each with its own workspace."""
    cases = [Case([5000, 2000], 8, 2, 128, 0, torch.bfloat16, 16, s) for s in (19, 20)]
    devs = [c.dev() for c in cases]
    want = [c.call(**d) for c, d in zip(cases, devs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(cases[i].call(**devs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert torch.equal(out, want[i])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [0, 3])
def test_serving_steps(dtype, M):
    """The operators as a serving loop runs them: norms and rotation, append,
    attention over the 4-bit cache, step after step; then a prefill chunk of
    flash_attention_v2 over the gathered context."""
    from kernels import (Fp4Cache, allocate_fp4_cache, build_rope_table, decode_attention_fp4,
                         flash_attention_v2, paged_kv_append_fp4, paged_kv_gather_fp4,
                         qk_norm_rope, speculative_decode_attention_fp4)
    B, QH, KVH, D, page, steps, T = 3, 8, 2, 128, 16, 4, max(M, 1)
    g = torch.Generator().manual_seed(21)
    prompt = [37, 1, 64]
    width = 12
    kt, vt = (torch.randperm(B * width, generator=g).view(B, width).to(torch.int32).cuda()
              for _ in range(2))
    kc, vc = (allocate_fp4_cache(B * width, page, KVH, D) for _ in range(2))
    table = build_rope_table(256, D, device="cuda")
    w = (1 + 0.1 * torch.randn(2, D, generator=g)).to(dtype).cuda()

    def project(n):
        return torch.randn(n, QH + 2 * KVH, D, generator=g).to(dtype).cuda()

    def plain_cache(k, v, ks, vs, at):
        t = 0
        for b, n in enumerate(at):
            ks[b] = torch.cat([ks[b], R.quantize(k[t:t + n].cpu())[0]])
            vs[b] = torch.cat([vs[b], R.quantize(v[t:t + n].cpu())[0]])
            t += n

    ks = [torch.empty(0, KVH, D, dtype=torch.float64) for _ in range(B)]
    vs = list(ks)
    lens = [0] * B
    for step in range(1 + steps):
        new = prompt if step == 0 else [T] * B
        qkv = project(sum(new))
        pos = torch.cat([torch.arange(s, s + n) for s, n in zip(lens, new)]).cuda()
        q, k, v = qkv[:, :QH], qkv[:, QH:QH + KVH], qkv[:, QH + KVH:]
        drafts = step > 0 and M
        if drafts:
            q = q.unflatten(0, (B, M)).transpose(1, 2)
        q, k = qk_norm_rope(q, k, w[0], w[1], table, pos)
        ip = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
        paged_kv_append_fp4(kc, vc, kt, vt, k, v, ip,
                            start_pos=torch.tensor(lens, dtype=torch.int32).cuda())
        plain_cache(k, v, ks, vs, new)
        lens = [a + b for a, b in zip(lens, new)]
        if step == 0:
            continue
        kw = dict(kv_indptr=torch.tensor(lens, dtype=torch.int32).cuda(), k_block_table=kt,
                  v_block_table=vt)
        if M:
            out = speculative_decode_attention_fp4(q, kc, vc, causal=True, **kw)
        else:
            out = decode_attention_fp4(q, kc, vc, **kw).unsqueeze(2)
            q = q.unsqueeze(2)
        for b in range(B):
            want, tol = R.attention(q[b].cpu(), ks[b], vs[b], bool(M))
            R.within(out[b], want, tol)
    # a chunk of queries over the whole context, causal from its end
    chunk = [5, 1, 9]
    q = torch.randn(sum(chunk), QH, D, generator=g).to(dtype)
    ip = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    qi = torch.tensor([0] + chunk).cumsum(0).to(torch.int32).cuda()
    k, v = paged_kv_gather_fp4(kc, vc, kt, vt, ip, sum(lens), dtype=dtype)
    assert torch.equal(k.cpu().double(), torch.cat(ks))
    out = flash_attention_v2(q.cuda(), k, v, is_causal=True, q_indptr=qi, kv_indptr=ip,
                             causal_alignment="bottom_right")
    t = 0
    for b, n in enumerate(chunk):
        x = q[t:t + n].transpose(0, 1)
        want, tol = R.attention(x, ks[b], vs[b], True)
        # (flash_attention_v2 rounds its weights to the type: h of A, in both sums)
        h = R.half_step(dtype)
        size = torch.stack([vs[b].abs().amax((0, 2))[i // (QH // KVH)] for i in range(QH)])
        R.within(out[t:t + n].transpose(0, 1), want, tol + 2 * h * size[:, None, None])
        t += n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("M", [0, 3])
@pytest.mark.parametrize("quanta", [2.49, 16.49, 100.4])
def test_small_weights(dtype, D, M, quanta):
    """Weights far below the largest count in full: every wave's first tile has a key
    that takes nearly all of the softmax and whose value is zero, so the output is
    the sum of weights of ``quanta`` * 2^-24 of the largest (2^-24: the least that fp16
    holds).  All terms are positive: A of fp4_ref's bound is the output."""
    QH, KVH, n = 4, 2, 768
    c = Case([n, n - 5], QH, KVH, D, M, dtype, 16, 26, causal=bool(M))
    lead = math.log(2.0 ** 24 / quanta)  # of the score, over zeros
    # a key of D values 3: its score is 3 * sqrt(D) * the query's value
    c.q = torch.full((2, QH, max(M, 1), D), lead / (3 * D ** 0.5)).to(dtype)
    for i, (codes, scales) in enumerate(c.caches):
        codes[:] = 0 if i == 0 else 0x22                        # K 0, V 1
        scales[:] = 127
        for b in range(2):
            for j in range(8):
                pg = c.tables[i][b, 32 * j // 16].item()
                codes[pg, :, 0] = 0x55 if i == 0 else 0         # K 3, V 0
    out = c.call()
    c.check(out)
    assert (out > 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("M", [0, 2])
@pytest.mark.parametrize("lens", [[100, 333], [5000, 64], [700] * 5])
def test_one_key_far_above_the_others(dtype, D, M, lens):
    """Scores at the largest scales, far past the exponent's range.  A key of +-6 with
    the queries' signs scores 6 sum |q_d|, which with these queries passes every other
    key by half of that at least (checked), the scores' errors by far less: its
    weight is one, all others are zero, and the output is its row of V, a number of
    the type, times (1 + 2 u) at most: that number."""
    H = 3
    c = Case(lens, H, H, D, M, dtype, 16, 27)
    c.q[:, :, 1:] = c.q[:, :, :1] * 0.5  # (drafts of one direction: one key for all)
    top = 127 + 13 if dtype == torch.float16 else 127 + 60
    for codes, scales in c.caches:
        scales[scales != 255] = top
    at = [n * (i % 3) // 2 if i % 3 < 2 else n - 1 for i, n in enumerate(lens)]
    codes, scales = c.caches[0]
    for b, j in enumerate(at):
        pg = c.tables[0][b, j // 16].item()
        nib = 7 + 8 * torch.signbit(c.q[b, :, 0]).to(torch.uint8)
        codes[pg, :, j % 16] = R.pack(nib)
    out = c.call()
    out = out.cpu() if M else out.cpu().unsqueeze(2)
    for b, j in enumerate(at):
        k, v = c.values(b)
        s = torch.einsum("hmd,nhd->hmn", c.q[b].double(), k)
        rest = s.clone()
        rest[..., j] = -math.inf
        assert (rest.amax(-1) < 0.5 * s[..., j]).all()
        assert torch.equal(out[b].double(), v[j].unsqueeze(1).expand_as(out[b]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("which", ["keys", "values", "low keys", "low values"])
def test_ends_of_the_type_with_ordinary_scores(dtype, D, which):
    """K or V at the largest or smallest scales with queries that keep the scores
    ordinary: fp4_ref's bound is tight (checked), outputs near the type's maximum."""
    lo, hi = (-23, 13) if dtype == torch.float16 else (-100, 120)
    e = lo if "low" in which else hi
    c = Case([100, 1033], 4, 2, D, 0, dtype, 16, 28)
    codes, scales = c.caches["values" in which]
    scales[scales != 255] = 127 + e
    if "keys" in which:
        # (queries of 2^-13 are fp16's small normal numbers, of 2^13 its large ones)
        shift = -e - 2 if dtype == torch.bfloat16 else max(min(-e - 2, 12), -12)
        c.q = (c.q.double() * 2.0 ** shift).to(dtype)
    out = c.call().cpu().unsqueeze(2)
    for b in range(2):
        want, tol = R.attention(c.q[b], *c.values(b), False)
        # The bound is h |o| (2^-8) and a share of A = sum p |v|: 4 (D + 4) u of the largest
        # score, here under 2^4, so 2^-10 at D = 256.  A is up to sqrt(1033) |o| and more
        # where signs cancel: 2^-5 in all.  (fp16 at the smallest values: half the type's
        # least number is all of it.)
        if which != "low values":
            assert (tol / want.abs()).median() < 0.1
        R.within(out[b], want, tol)


@pytest.mark.parametrize("D,QH,KVH,M,lens", [
    (128, 8, 1, 0, [100001]),                    # one context, longer than 2^16 keys
    (64, 4, 2, 3, [70000, 40000]),
    (128, 32, 32, 0, [1500, 33, 700]),           # more than 8 heads of K and V
    (64, 20, 20, 4, [900, 1]),
])
def test_longer_contexts_and_more_heads(D, QH, KVH, M, lens):
    c = Case(lens, QH, KVH, D, M, torch.bfloat16, 16, 29, causal=bool(M))
    c.check(c.call())


@pytest.mark.parametrize("drafts", [False, True])
@pytest.mark.parametrize("bad,kind,text", [
    ("dims", ValueError, "q must be [B, QH"), ("dtype", TypeError, "unsupported dtype"),
    ("head_dim", ValueError, "head_dim"), ("heads", ValueError, "multiple of kv_heads"),
    ("lens", ValueError, "need 2 rows"), ("rows", ValueError, "need 2 rows"),
    ("v", ValueError, "v_cache is missing"), ("codes", TypeError, "must be uint8"),
    ("pages", ValueError, "equal shapes"), ("scales", ValueError, "contiguous"),
    ("device", AssertionError, "same device"), ("aligned", RuntimeError, "status 7"),
])
def test_refusals_name_the_cause(drafts, bad, kind, text):
    """One exception and one message for each cause, with and without the extension."""
    import kernels.decode_fp4 as m
    c = Case([40, 3], 4, 2, 128, 3 if drafts else 0, torch.float16, 16, 25)
    d = c.dev()
    q, k, v = d.pop("q"), d.pop("k_cache"), d.pop("v_cache")
    if bad == "dims":
        q = q[0]
    elif bad == "dtype":
        q = q.float()
    elif bad == "head_dim":
        q = q[..., :64]
    elif bad == "heads":
        q = q[:, :3]
    elif bad == "lens":
        d["kv_indptr"] = d["kv_indptr"][:1]
    elif bad == "rows":
        d["v_block_table"] = d["v_block_table"][:1]
    elif bad == "v":
        v = None
    elif bad == "codes":
        v = (v[0].char(), v[1])
    elif bad == "pages":
        v = (v[0][1:], v[1][1:])
    elif bad == "scales":
        k = (k[0], k[1][..., :3])
    elif bad == "device":
        d["kv_indptr"] = d["kv_indptr"].cpu()
    else:  # codes off a 16-byte boundary
        n = k[0].numel()
        k = (torch.zeros(n + 8, dtype=torch.uint8, device="cuda")[8:].view(k[0].shape), k[1])
    name = "speculative_decode_attention_fp4" if drafts else "decode_attention_fp4"
    said = []
    for use in (True, False):
        m.USE_EXT = use
        try:
            with pytest.raises(kind) as e:
                getattr(m, name)(q, k, v, **d)
        finally:
            m.USE_EXT = True
        assert text in str(e.value)
        assert kind is AssertionError or str(e.value).startswith(name)
        said.append((type(e.value), str(e.value)))
    assert said[0] == said[1]
    torch.cuda.synchronize()


@pytest.mark.parametrize("use_ext", [True, False])
def test_int64_lengths_past_32_bits(use_ext):
    """A length of 2^32 and more is past the table and counts as its keys; entries
    that 32 bits do not hold are clamped into the pool from their own side."""
    import kernels.decode_fp4 as m
    c = Case([48, 32], 4, 2, 64, 0, torch.float16, 16, 37)
    m.USE_EXT = use_ext
    try:
        want = c.call()
        got = c.call(kv_indptr=torch.tensor([2 ** 32 + 5, 32], device="cuda"))
        assert torch.equal(got, want)
        last = c.caches[0][0].shape[0] - 1
        for codes, scales in c.caches:
            scales[scales == 255] = 126
        tables = []
        for t in c.tables:
            t[1] = torch.tensor([0, last, -1])
            t64 = t.long()
            t64[1] = torch.tensor([-2 ** 32 + 3, 2 ** 32 + 1, -1])
            tables.append(t64.cuda())
        want = c.call()
        got = c.call(k_block_table=tables[0], v_block_table=tables[1])
        assert torch.equal(got[1], want[1])
    finally:
        m.USE_EXT = True
