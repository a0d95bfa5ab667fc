"""paged_kv_append_fp4 and paged_kv_gather_fp4: exact, against the quantiser in
64 bits (fp4_ref)."""

import math

import pytest
import torch

import fp4_ref as R

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need an MI355X")


def tables(lens, page, seed, spare=2):
    """Two shuffled block tables over one pool, padding -1."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages, width = sum(need) + spare, max(need + [1])
    out = []
    for _ in range(2):
        perm, t, at = torch.randperm(pages, generator=g), torch.full((len(lens), width), -1), 0
        for b, n in enumerate(need):
            t[b, :n] = perm[at:at + n]
            at += n
        out.append(t.to(torch.int32))
    return out[0], out[1], pages


def place(table, b, n, page):
    return table[b, n // page].item(), n % page


def rows_of(T, H, D, dtype, seed):
    """Blocks of many sizes, with ties, signed zeros and blocks of zeros."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, D, generator=g)
    x = x * torch.exp2(torch.randint(-9, 9, (T, H, D // 32), generator=g).float()
                       ).repeat_interleave(32, -1)
    x[0] = 0.0
    x[0, 0, 1] = -0.0
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4)
    x[-1, :, :32] = ties
    x[-1, :, 32:64] = -ties * 2.0 ** -7
    x[T // 2, 0, :32] = torch.linspace(-7, 7, 32)         # the step's border is 7
    x[T // 2, 0, 32:64] = torch.linspace(-6.999, 6.999, 32)
    return x.to(dtype)


def indptr(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,H,page", [(64, 1, 16), (64, 3, 5), (128, 8, 16), (128, 2, 1),
                                      (128, 5, 64), (256, 2, 16), (256, 1, 7)])
def test_append_then_gather(dtype, D, H, page):
    from kernels import allocate_fp4_cache, paged_kv_append_fp4, paged_kv_gather_fp4
    lens, start = [1, 0, 37, 70, 5], [0, 9, 3, 130, 15]
    T = sum(lens)
    k, v = rows_of(T, H, D, dtype, 1), rows_of(T, H, D, dtype, 2)
    kt, vt, pages = tables([a + b for a, b in zip(lens, start)], page, 3)
    kc, vc = (allocate_fp4_cache(pages, page, H, D) for _ in range(2))
    ip, sp = indptr(lens).cuda(), torch.tensor(start, dtype=torch.int32).cuda()
    paged_kv_append_fp4(kc, vc, kt.cuda(), vt.cuda(), k.cuda(), v.cuda(), ip, start_pos=sp)
    for x, cache, table in ((k, kc, kt), (v, vc, vt)):
        val, nib, scale = R.quantize(x)
        codes, scales = torch.zeros_like(cache.codes.cpu()), torch.zeros_like(cache.scales.cpu())
        t = 0
        for b, n in enumerate(lens):
            for j in range(n):
                pg, off = place(table, b, start[b] + j, page)
                codes[pg, :, off], scales[pg, :, off] = R.pack(nib[t]), scale[t]
                t += 1
        assert torch.equal(cache.codes.cpu(), codes)
        assert torch.equal(cache.scales.cpu(), scales)
    for to in DTYPES:
        if dtype != to and to == torch.float16:
            continue  # (values of other types need not be exact in fp16)
        gk, gv = paged_kv_gather_fp4(kc, vc, kt.cuda(), vt.cuda(), ip, T, sp, dtype=to)
        assert gk.dtype == to
        assert torch.equal(gk.cpu().double(), R.quantize(k)[0])
        assert torch.equal(gv.cpu().double(), R.quantize(v)[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_extreme_values(dtype):
    """The largest, the smallest, infinities and NaN; error within 1/7 of the
    block's largest inside the type's range of powers."""
    from kernels import allocate_fp4_cache, paged_kv_append_fp4, paged_kv_gather_fp4
    f = torch.finfo(dtype)
    x = torch.zeros(12, 1, 64)
    x = x.to(torch.float64)
    x[0, 0, :] = f.max
    x[1, 0, :] = torch.linspace(-1, 1, 64, dtype=torch.float64) * f.max
    x[2, 0, :] = f.smallest_normal
    x[3, 0, 5] = f.smallest_normal * f.eps                # the smallest number
    x[4, 0, 3] = math.inf
    x[5, 0, 40] = -math.inf
    x[6, 0, 63] = math.nan
    x[7, 0, :32] = 2.0 ** -14
    x[8, 0, :] = torch.linspace(-1, 1, 64, dtype=torch.float64) * 2.0 ** -100 if dtype != torch.float16 else 0
    x[9, 0, :] = 49152.0
    x[10, 0, :] = torch.randn(64, generator=torch.Generator().manual_seed(0), dtype=torch.float64)
    x[11, 0, ::2] = -f.max
    x = x.to(dtype)
    kt = torch.zeros(1, 1, dtype=torch.int32).cuda()
    kc = allocate_fp4_cache(1, 12, 1, 64)
    ip = indptr([12]).cuda()
    paged_kv_append_fp4(kc, None, kt, None, x.cuda(), None, ip)
    val, nib, scale = R.quantize(x)
    assert torch.equal(kc.codes[0, 0].cpu(), R.pack(nib)[:, 0])
    assert torch.equal(kc.scales[0, 0].cpu(), scale[:, 0])
    got, none = paged_kv_gather_fp4(kc, None, kt, None, ip, 12, dtype=dtype)
    assert none is None
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(val))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(val))
    assert torch.isnan(got[4, 0, :32]).all() and (got[4, 0, 32:] == 0).all()
    a = x[10].double().unflatten(-1, (-1, 32))
    err = (got[10].unflatten(-1, (-1, 32)) - a).abs().amax(-1)
    assert (err <= a.abs().amax(-1) / 7).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_without_a_place(dtype):
    """Pages past the table or outside the pool are skipped by the writer and
    zeros to the reader; rows that no sequence holds stay as they are."""
    from kernels import allocate_fp4_cache, paged_kv_append_fp4, paged_kv_gather_fp4
    H, D, page = 2, 64, 4
    x = rows_of(20, H, D, dtype, 4)
    kt = torch.tensor([[2, -1, 7], [0, 3, 1]], dtype=torch.int32)  # pages 0..3
    kc = allocate_fp4_cache(4, page, H, D)
    ip = torch.tensor([2, 12, 18], dtype=torch.int32)  # rows 0, 1, 18, 19: nobody's
    sp = torch.tensor([0, 8], dtype=torch.int32)
    args = (kc, None, kt.cuda(), None)
    paged_kv_append_fp4(*args, x.cuda(), None, ip.cuda(), start_pos=sp.cuda())
    want = torch.zeros(4, H, page, D // 2, dtype=torch.uint8)
    nib = R.pack(R.quantize(x)[1])
    for j in range(4):
        want[2, :, j] = nib[2 + j]       # sequence 0: page 2, then none
        want[1, :, j] = nib[12 + j]      # sequence 1: page 1, then past the table
    assert torch.equal(kc.codes.cpu(), want)
    out = torch.full((20, H, D), 7.0, dtype=dtype, device="cuda")
    got, _ = paged_kv_gather_fp4(*args, ip.cuda(), 20, sp.cuda(), out=(out, None))
    assert got is out
    got, val = got.cpu().double(), R.quantize(x)[0]
    for t in range(20):
        exp = (torch.full((H, D), 7.0, dtype=torch.float64) if t < 2 or t >= 18
               else val[t] if 2 <= t < 6 or 12 <= t < 16 else torch.zeros(H, D).double())
        assert torch.equal(got[t], exp), t


def test_strides_and_index_types():
    """K and V views of one projection with strides of their own, unaligned rows,
    int64 indices, tables that are slices."""
    from kernels import allocate_fp4_cache, paged_kv_append_fp4
    H, D, page, lens = 4, 128, 16, [3, 40]
    T = sum(lens)
    kt, vt, pages = tables(lens, page, 5)
    wide = torch.cat([kt, kt + 100], 1).cuda()
    qkv = rows_of(T, 3 * H, D, torch.bfloat16, 6).cuda()
    k, v = qkv[:, H:2 * H], qkv[:, 2 * H:]
    ip = indptr(lens).cuda()
    want = [allocate_fp4_cache(pages, page, H, D) for _ in range(2)]
    paged_kv_append_fp4(*want, kt.cuda(), vt.cuda(), k.contiguous(), v.contiguous(), ip)
    off = torch.empty(T * H * D + 1, dtype=k.dtype, device="cuda")[1:].view(T, H, D).copy_(v)
    for kk, vv in ((k, v), (k.contiguous(), v), (k, off),
                   (k.transpose(0, 2).contiguous().transpose(0, 2), v)):
        got = [allocate_fp4_cache(pages, page, H, D) for _ in range(2)]
        paged_kv_append_fp4(*got, wide[:, :kt.shape[1]], vt.long().cuda(), kk, vv, ip.long())
        for a, b in zip(got, want):
            assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


def test_many_sequences():
    """More sequences than the writer keeps in LDS, one row each."""
    from kernels import allocate_fp4_cache, paged_kv_append_fp4, paged_kv_gather_fp4
    n, H, D = 1500, 1, 64
    x = rows_of(n, H, D, torch.float16, 8).cuda()
    kt = torch.randperm(n, generator=torch.Generator().manual_seed(1)).to(torch.int32)[:, None].cuda()
    kc = allocate_fp4_cache(n, 2, H, D)
    ip = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    sp = torch.ones(n, dtype=torch.int32, device="cuda")
    paged_kv_append_fp4(kc, None, kt, None, x, None, ip, start_pos=sp)
    got, _ = paged_kv_gather_fp4(kc, None, kt, None, ip, n, sp, dtype=torch.float16)
    assert torch.equal(got.cpu().double(), R.quantize(x.cpu())[0])
    assert (kc.codes[:, :, 0] == 0).all()


def test_no_rows():
    from kernels import allocate_fp4_cache, paged_kv_append_fp4, paged_kv_gather_fp4
    kc = allocate_fp4_cache(2, 16, 2, 64)
    kt = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    ip = torch.zeros(4, dtype=torch.int32, device="cuda")
    none = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    paged_kv_append_fp4(kc, None, kt, None, none, None, ip)
    got, _ = paged_kv_gather_fp4(kc, None, kt, None, ip, 0)
    assert got.shape == (0, 2, 64) and (kc.codes == 0).all()


def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes of codes."""
    from kernels import allocate_fp4_cache, paged_kv_append_fp4, paged_kv_gather_fp4
    H, D, page, pages = 8, 256, 64, 70000
    kc = allocate_fp4_cache(pages, page, H, D)
    x = rows_of(100, H, D, torch.bfloat16, 9).cuda()
    kt = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device="cuda")
    ip = indptr([100]).cuda()
    paged_kv_append_fp4(kc, None, kt, None, x, None, ip)
    got, _ = paged_kv_gather_fp4(kc, None, kt, None, ip, 100)
    assert torch.equal(got.cpu().double(), R.quantize(x.cpu())[0])
    assert not kc.codes[:pages - 2].any()


def test_ctypes_path_stream_and_graph():
    import kernels.fp4_cache as m
    H, D, page, lens = 4, 128, 16, [3, 40]
    T = sum(lens)
    kt, vt, pages = tables(lens, page, 5)
    k, v = (rows_of(T, H, D, torch.bfloat16, s).cuda() for s in (6, 7))
    ip, kt, vt = indptr(lens).cuda(), kt.cuda(), vt.cuda()
    want = [m.allocate_fp4_cache(pages, page, H, D) for _ in range(2)]
    m.paged_kv_append_fp4(*want, kt, vt, k, v, ip)
    rows = m.paged_kv_gather_fp4(*want, kt, vt, ip, T)
    m.USE_EXT = False
    try:
        got = [m.allocate_fp4_cache(pages, page, H, D) for _ in range(2)]
        m.paged_kv_append_fp4(*got, kt, vt, k, v, ip)
        rows2 = m.paged_kv_gather_fp4(*got, kt, vt, ip, T)
    finally:
        m.USE_EXT = True
    for a, b in zip(got, want):
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    assert torch.equal(rows[0], rows2[0]) and torch.equal(rows[1], rows2[1])
    got = [m.allocate_fp4_cache(pages, page, H, D) for _ in range(2)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.paged_kv_append_fp4(*got, kt, vt, k, v, ip)
        held = m.paged_kv_gather_fp4(*got, kt, vt, ip, T)
    for i in range(3):
        k.copy_(rows_of(T, H, D, torch.bfloat16, 20 + i))
        graph.replay()
        m.paged_kv_append_fp4(*want, kt, vt, k, v, ip)
        rows = m.paged_kv_gather_fp4(*want, kt, vt, ip, T)
        torch.cuda.synchronize()
        assert torch.equal(held[0], rows[0]) and torch.equal(held[1], rows[1])


@pytest.mark.parametrize("bad", ["codes", "scales", "ctype", "contiguous", "v", "v_table", "v_rows",
                                 "tables", "start", "rtype", "rows", "mixed", "device", "count"])
def test_refusals(bad):
    """The same error with and without the extension, before any launch."""
    import kernels.fp4_cache as m
    H, D, page, lens = 2, 64, 16, [3, 20]
    T = sum(lens)
    kt, vt, pages = tables(lens, page, 5)
    kt, vt, ip = kt.cuda(), vt.cuda(), indptr(lens).cuda()
    k, v = (rows_of(T, H, D, torch.bfloat16, s).cuda() for s in (6, 7))
    kc, vc = (m.allocate_fp4_cache(pages, page, H, D) for _ in range(2))
    sp, count, gather = torch.zeros(2, dtype=torch.int32, device="cuda"), T, True
    if bad == "codes":
        vc = m.allocate_fp4_cache(pages, page, H, 128)
    elif bad == "scales":
        kc = (kc.codes, kc.scales[..., :1].contiguous())
    elif bad == "ctype":
        kc = (kc.codes.char(), kc.scales)
    elif bad == "contiguous":
        kc = (kc.codes.transpose(1, 2), kc.scales.transpose(1, 2))
    elif bad == "v":
        vc = None
    elif bad == "v_table":
        vt = None
    elif bad == "v_rows":
        v, gather = None, False
    elif bad == "tables":
        kt = kt[:1]
    elif bad == "start":
        sp = sp[:1]
    elif bad == "rtype":
        k, v, gather = k.double(), v.double(), False
    elif bad == "rows":
        k, v, gather = k[:, :1], v[:, :1], False
    elif bad == "mixed":
        v, gather = v.float(), False
    elif bad == "device":
        ip = ip.cpu()
    else:
        count = -1
    calls = [lambda: m.paged_kv_gather_fp4(kc, vc, kt, vt, ip, count, sp)] if gather else []
    if bad != "count":
        calls.append(lambda: m.paged_kv_append_fp4(kc, vc, kt, vt, k, v, ip, sp))
    for call in calls:
        seen = []
        for use in (True, False):
            m.USE_EXT = use
            try:
                with pytest.raises((ValueError, TypeError, AssertionError)) as e:
                    call()
                seen.append((e.type, str(e.value)))
            finally:
                m.USE_EXT = True
        assert seen[0] == seen[1]
    torch.cuda.synchronize()


def test_gather_into_tensors():
    """Into given tensors; rows that no sequence holds stay as they were, and tensors
    that do not fit are refused."""
    import kernels.fp4_cache as m
    H, D, page, lens = 3, 64, 16, [5, 0, 33]
    T, ahead, behind = sum(lens), 2, 3
    kt, vt, pages = tables(lens, page, 5)
    kt, vt, ip = kt.cuda(), vt.cuda(), indptr(lens).cuda()
    k, v = (rows_of(T, H, D, torch.float16, s).cuda() for s in (6, 7))
    kc, vc = (m.allocate_fp4_cache(pages, page, H, D) for _ in range(2))
    m.paged_kv_append_fp4(kc, vc, kt, vt, k, v, ip)
    n = ahead + T + behind
    for use in (True, False):
        m.USE_EXT = use
        try:
            out = tuple(torch.full((n, H, D), 7.0, dtype=torch.float16, device="cuda")
                        for _ in range(2))
            got = m.paged_kv_gather_fp4(kc, vc, kt, vt, ip + ahead, n, out=out)
            assert got[0] is out[0] and got[1] is out[1]
            for x, rows in zip(got, (k, v)):
                assert (x[:ahead] == 7).all() and (x[ahead + T:] == 7).all()
                assert torch.equal(x[ahead:ahead + T].cpu().double(), R.quantize(rows.cpu())[0])
            for bad in ((out[0][:-1], out[1]), (out[0], out[1].float()), (out[0], None),
                        (out[0].transpose(0, 1).contiguous().transpose(0, 1), out[1]),
                        (out[0].int(), out[1].int()), (out[0].cpu(), out[1])):
                with pytest.raises((ValueError, TypeError, AssertionError)):
                    m.paged_kv_gather_fp4(kc, vc, kt, vt, ip + ahead, n, out=bad)
        finally:
            m.USE_EXT = True


@pytest.mark.parametrize("dtype", DTYPES)
def test_gather_past_the_caches(dtype):
    """More than 2^28 bytes of rows (sequences that share their pages)."""
    from kernels import allocate_fp4_cache, paged_kv_append_fp4, paged_kv_gather_fp4
    H, D, page, n = 8, 128, 16, 1001
    seqs = (1 << 28) // (n * H * D * 2 * dtype.itemsize) + 2
    kt, vt, pages = tables([n], page, 5)
    kt, vt = kt.cuda(), vt.cuda()
    k, v = (rows_of(n, H, D, dtype, s).cuda() for s in (6, 7))
    kc, vc = (allocate_fp4_cache(pages, page, H, D) for _ in range(2))
    paged_kv_append_fp4(kc, vc, kt, vt, k, v, indptr([n]).cuda())
    want = paged_kv_gather_fp4(kc, vc, kt, vt, indptr([n]).cuda(), n, dtype=dtype)
    assert torch.equal(want[0].cpu().double(), R.quantize(k.cpu())[0])
    got = paged_kv_gather_fp4(kc, vc, kt.expand(seqs, -1), vt.expand(seqs, -1).contiguous(),
                              indptr([n] * seqs).cuda(), n * seqs, dtype=dtype)
    for x, w in zip(got, want):
        assert torch.equal(x.view(seqs, n, H, D), w.expand(seqs, -1, -1, -1))


@pytest.mark.parametrize("dtype", DTYPES)
def test_error_bound_of_a_block(dtype):
    """The error of a block is at most 1/5 of its largest value a, which the step keeps
    within 3.5 <= a < 7 steps: values from 4 steps up are off by at most one step, which is
    a / 5 at a = 5 (midway between 4 and 6, it becomes 4) and less elsewhere (a - 4 below 5,
    1 above); the others by half a step at most, a / 7."""
    from kernels import allocate_fp4_cache, paged_kv_append_fp4, paged_kv_gather_fp4
    tops = [3.5, 3.75, 4.0, 4.5, 4.75, 5.0, 5.25, 5.5, 5.75, 6.0, 6.5, 6.75, 6.9375]
    x = torch.empty(16 * len(tops), 1, 64, dtype=torch.float64)
    g = torch.Generator().manual_seed(30)
    for i, a in enumerate(tops):
        for j in range(16):
            row = (torch.rand(64, generator=g, dtype=torch.float64) * 2 - 1) * a
            row[[j, 32 + j]] = torch.tensor([a, -a], dtype=torch.float64)
            x[16 * i + j, 0] = row * 2.0 ** (j - 8)
    x = x.to(dtype)
    n = x.shape[0]
    kt = torch.arange(-(-n // 16), dtype=torch.int32).cuda()[None]
    kc, ip = allocate_fp4_cache(kt.shape[1], 16, 1, 64), indptr([n]).cuda()
    paged_kv_append_fp4(kc, None, kt, None, x.cuda(), None, ip)
    got, _ = paged_kv_gather_fp4(kc, None, kt, None, ip, n, dtype=dtype)
    blocks = x.double().unflatten(-1, (-1, 32))
    err = (got.cpu().double().unflatten(-1, (-1, 32)) - blocks).abs().amax(-1)
    share = (err / blocks.abs().amax(-1)).view(len(tops), -1)
    assert (share <= 0.2).all()
    assert (share[tops.index(5.0)] == 0.2).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,D", [(32, 128), (20, 128), (9, 256), (33, 64), (17, 64), (64, 256)])
@pytest.mark.parametrize("only_k", [False, True])
def test_wide_rows(dtype, H, D, only_k):
    """More code words in a row than the workgroup has threads, and row lengths that
    leave threads idle; rows that the last workgroup does not fill."""
    from kernels import allocate_fp4_cache, paged_kv_append_fp4, paged_kv_gather_fp4
    lens, start, page = [1, 0, 18, 6], [3, 0, 15, 0], 16
    T = sum(lens) + 1                                       # and a row that is nobody's
    k, v = rows_of(T, H, D, dtype, 31), rows_of(T, H, D, dtype, 32)
    kt, vt, pages = tables([a + b for a, b in zip(lens, start)], page, 33)
    kc, vc = (allocate_fp4_cache(pages, page, H, D) for _ in range(2))
    ip, sp = indptr(lens).cuda(), torch.tensor(start, dtype=torch.int32).cuda()
    sides = [(k, kc, kt)] + ([] if only_k else [(v, vc, vt)])
    args = (kc, None if only_k else vc, kt.cuda(), None if only_k else vt.cuda())
    paged_kv_append_fp4(*args, k.cuda(), None if only_k else v.cuda(), ip, start_pos=sp)
    out = [torch.full((T, H, D), 7.0, dtype=dtype, device="cuda") for _ in sides]
    paged_kv_gather_fp4(*args, ip, T, sp, out=(out[0], None if only_k else out[1]))
    for (x, cache, table), got in zip(sides, out):
        val, nib, scale = R.quantize(x)
        codes, scales = torch.zeros_like(cache.codes.cpu()), torch.zeros_like(cache.scales.cpu())
        t = 0
        for b, n in enumerate(lens):
            for j in range(n):
                pg, off = place(table, b, start[b] + j, page)
                codes[pg, :, off], scales[pg, :, off] = R.pack(nib[t]), scale[t]
                t += 1
        assert torch.equal(cache.codes.cpu(), codes)
        assert torch.equal(cache.scales.cpu(), scales)
        assert torch.equal(got[:-1].cpu().double(), val[:-1])
        assert (got[-1] == 7.0).all()


@pytest.mark.parametrize("n", [255, 256, 257, 300, 512, 513])
def test_batches_around_the_staged_ones(n):
    """As many sequences as a workgroup has threads, as its LDS holds, and one more."""
    from kernels import allocate_fp4_cache, paged_kv_append_fp4, paged_kv_gather_fp4
    H, D, page = 2, 64, 4
    g = torch.Generator().manual_seed(n)
    lens = torch.randint(0, 4, (n,), generator=g).tolist()
    lens[-1], start = 2, torch.randint(0, 6, (n,), generator=g)
    T = sum(lens)
    x = rows_of(T, H, D, torch.bfloat16, 34)
    kt, _, pages = tables([a + b for a, b in zip(lens, start.tolist())], page, 35)
    kc = allocate_fp4_cache(pages, page, H, D)
    ip, sp = indptr(lens).cuda(), start.to(torch.int32).cuda()
    paged_kv_append_fp4(kc, None, kt.cuda(), None, x.cuda(), None, ip, start_pos=sp)
    got, _ = paged_kv_gather_fp4(kc, None, kt.cuda(), None, ip, T, sp)
    val, nib, _ = R.quantize(x)
    assert torch.equal(got.cpu().double(), val)
    t, codes = 0, torch.zeros_like(kc.codes.cpu())
    for b, m in enumerate(lens):
        for j in range(m):
            pg, off = place(kt, b, start[b].item() + j, page)
            codes[pg, :, off] = R.pack(nib[t])
            t += 1
    assert torch.equal(kc.codes.cpu(), codes)


@pytest.mark.parametrize("use_ext", [True, False])
def test_int64_indices_past_32_bits(use_ext):
    """Entries and positions that 32 bits do not hold are outside, not another page."""
    import kernels.fp4_cache as m
    H, D, page = 1, 64, 4
    x = rows_of(16, H, D, torch.bfloat16, 36).cuda()
    far = 2 ** 32
    kt = torch.tensor([[far, 1], [-2 ** 63, 2], [0, -far], [3, far + 3]], device="cuda")
    sp = torch.tensor([0, 0, 0, far], device="cuda")
    ip = torch.arange(0, 17, 4, device="cuda")
    kc = m.allocate_fp4_cache(4, page, H, D)
    m.USE_EXT = use_ext
    try:
        m.paged_kv_append_fp4(kc, None, kt, None, x, None, ip, start_pos=sp)
        got, _ = m.paged_kv_gather_fp4(kc, None, kt, None, ip, 16, sp)
    finally:
        m.USE_EXT = True
    val, nib, _ = R.quantize(x.cpu())
    want = torch.zeros_like(kc.codes.cpu())
    want[0] = R.pack(nib)[8:12].transpose(0, 1)  # sequence 2 alone has a page
    assert torch.equal(kc.codes.cpu(), want)
    assert torch.equal(got[8:12].cpu().double(), val[8:12])
    assert not got[:8].any() and not got[12:].any()


@pytest.mark.parametrize("written", [torch.bfloat16, torch.float32])
def test_gather_in_fp16_of_other_rows(written):
    """Every scale that bf16 and fp32 rows give, read in fp16: the values rounded to
    nearest, to fp16's small numbers and zero below its range and infinity past it."""
    from kernels import allocate_fp4_cache, paged_kv_append_fp4, paged_kv_gather_fp4
    e = torch.arange(-101, 120, dtype=torch.float64)
    x = torch.empty(len(e), 1, 64, dtype=torch.float64)
    x[:, 0] = torch.tensor([0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.5] * 8, dtype=torch.float64)
    x = (x * torch.exp2(e)[:, None, None]).to(written)
    n = len(e)
    kt = torch.arange(-(-n // 16), dtype=torch.int32).cuda()[None]
    kc, ip = allocate_fp4_cache(kt.shape[1], 16, 1, 64), indptr([n]).cuda()
    paged_kv_append_fp4(kc, None, kt, None, x.cuda(), None, ip)
    val = R.quantize(x)[0]
    for to in DTYPES:
        got, _ = paged_kv_gather_fp4(kc, None, kt, None, ip, n, dtype=to)
        assert torch.equal(got.cpu(), val.to(to)), to
        out = torch.empty(n, 1, 64, dtype=to, device="cuda")
        paged_kv_gather_fp4(kc, None, kt, None, ip, n, out=(out, None))  # (out's type)
        assert torch.equal(out, got)


@pytest.mark.parametrize("use_ext", [True, False])
@pytest.mark.parametrize("only_k", [False, True])
def test_tables_without_columns(use_ext, only_k):
    """No row has a place: nothing is written, rows are zeros, outputs NaN."""
    import kernels.decode_fp4 as d
    import kernels.fp4_cache as m
    H, D = 2, 64
    kc, vc = (m.allocate_fp4_cache(2, 16, H, D) for _ in range(2))
    none = torch.empty(3, 0, dtype=torch.int32, device="cuda")
    x = rows_of(9, H, D, torch.float16, 38).cuda()
    ip = indptr([4, 0, 5]).cuda()
    m.USE_EXT = d.USE_EXT = use_ext
    args = (kc, None, none, None) if only_k else (kc, vc, none, none)
    try:
        m.paged_kv_append_fp4(*args, x, None if only_k else x, ip)
        got = m.paged_kv_gather_fp4(*args, ip, 9, dtype=torch.float16)
        out = d.decode_attention_fp4(x[:3], kc, vc, kv_indptr=ip[1:], k_block_table=none,
                                     v_block_table=none)
    finally:
        m.USE_EXT = d.USE_EXT = True
    for c in (kc, vc):
        assert not c.codes.any() and not c.scales.any()
    assert not got[0].any() and (only_k or not got[1].any())
    assert torch.isnan(out).all()
