"""qk_norm_rope against its formula in 64 bits (bounds: fp4_ref)."""

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


def data(T, HQ, HK, D, dtype, seed, wtype=None):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(T, HQ, D, generator=g) * 3).to(dtype)
    k = (torch.randn(T, HK, D, generator=g) * torch.rand(D, generator=g) * 20).to(dtype)
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(wtype or dtype) for _ in range(2)]
    return q, k, w[0], w[1], g


def check(out, x, w, table, pos, inter, eps=1e-6):
    want, tol = R.norm_rope(x.cpu(), w.cpu(), table.cpu(), pos.cpu(), inter, eps)
    R.within(out, want, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,rot", [(16, 16), (32, 16), (64, 64), (64, 32), (128, 128), (128, 48),
                                   (256, 256), (256, 64), (128, 0)])
@pytest.mark.parametrize("inter", [False, True])
def test_shapes(dtype, D, rot, inter):
    from kernels import build_rope_table, qk_norm_rope
    for T, HQ, HK in ((1, 1, 1), (7, 6, 2), (65, 5, 3)):
        q, k, qw, kw, g = data(T, HQ, HK, D, dtype, T + D)
        table = (build_rope_table(5000, rot, device="cuda") if rot
                 else torch.empty(5000, 0, device="cuda"))
        pos = torch.randint(0, 5000, (T,), generator=g, dtype=torch.int32)
        qo, ko = qk_norm_rope(q.cuda(), k.cuda(), qw.cuda(), kw.cuda(), table, pos.cuda(),
                              interleaved=inter)
        assert qo.dtype == dtype and qo.is_contiguous() and ko.is_contiguous()
        check(qo, q, qw, table, pos, inter)
        check(ko, k, kw, table, pos, inter)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_tokens(dtype):
    """Enough rows for the four-head variant, head counts that do not divide."""
    from kernels import build_rope_table, qk_norm_rope
    q, k, qw, kw, g = data(3001, 13, 3, 128, dtype, 1, torch.float32)
    table = build_rope_table(40000, 128, base=500000.0, device="cuda")
    pos = torch.randint(0, 40000, (3001,), generator=g)
    qo, ko = qk_norm_rope(q.cuda(), k.cuda(), qw.cuda(), kw.cuda(), table, pos.cuda(), eps=1e-5)
    check(qo, q, qw, table, pos, False, 1e-5)
    check(ko, k, kw, table, pos, False, 1e-5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts_and_strides(dtype):
    """Views of a fused projection; drafts [B, H, M, D]; other orders, unaligned rows."""
    from kernels import build_rope_table, qk_norm_rope
    B, M, HQ, HK, D = 5, 3, 8, 2, 64
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(B * M, HQ + 2 * HK, D, generator=g).to(dtype)
    w = torch.rand(2, D, generator=g).to(dtype)
    table = build_rope_table(300, D, device="cuda")
    pos = torch.randint(0, 300, (B, M), generator=g)
    dev, wd, pd = qkv.cuda(), w.cuda(), pos.cuda()
    q, k = dev[:, :HQ], dev[:, HQ:HQ + HK]
    q4 = q.unflatten(0, (B, M)).transpose(1, 2)
    qo, ko = qk_norm_rope(q4, k, wd[0], wd[1], table, pd)
    assert qo.shape == (B, HQ, M, D) and ko.shape == (B * M, HK, D)
    check(qo.transpose(1, 2).flatten(0, 1), qkv[:, :HQ], w[0], table, pos, False)
    check(ko, qkv[:, HQ:HQ + HK], w[1], table, pos, False)
    k4 = k.unflatten(0, (B, M)).transpose(1, 2).contiguous()
    qo3, ko4 = qk_norm_rope(q, k4, wd[0], wd[1], table, pd)
    assert torch.equal(qo3.unflatten(0, (B, M)).transpose(1, 2), qo)
    assert torch.equal(ko4.transpose(1, 2).flatten(0, 1), ko)
    # rows that start off a 16-byte boundary, a transposed head dim, one key head
    # for all (stride 0): the same values
    off = torch.empty(q.numel() + 1, dtype=dtype, device="cuda")[1:].view(q.shape).copy_(q)
    tr = k.transpose(1, 2).contiguous().transpose(1, 2)
    a, b = qk_norm_rope(off, tr, wd[0], wd[1], table, pd)
    assert torch.equal(a, qo3) and torch.equal(b, ko)
    one = k[:, :1].expand(B * M, 4, D)
    _, c = qk_norm_rope(q, one, wd[0], wd[1], table, pd)
    assert torch.equal(c, ko[:, :1].expand(-1, 4, -1))


def test_positions_and_rows_of_zeros():
    """Positions past the table give NaN in their rows only; both integer types;
    a row of zeros is zeros."""
    from kernels import build_rope_table, qk_norm_rope
    q, k, qw, kw, g = data(6, 4, 2, 64, torch.bfloat16, 5)
    q[2] = 0
    table = build_rope_table(100, 64, device="cuda")
    pos = torch.tensor([0, 99, 5, 100, -1, 2 ** 32 + 1])
    qo, ko = qk_norm_rope(q.cuda(), k.cuda(), qw.cuda(), kw.cuda(), table, pos.cuda())
    check(qo, q, qw, table, pos, False)
    check(ko, k, kw, table, pos, False)
    assert (qo[2] == 0).all() and torch.isnan(qo[3:]).all() and torch.isnan(ko[3:]).all()
    p32 = torch.tensor([0, 99, 5, 7, 8, 9], dtype=torch.int32)
    a = qk_norm_rope(q.cuda(), k.cuda(), qw.cuda(), kw.cuda(), table, p32.cuda())
    b = qk_norm_rope(q.cuda(), k.cuda(), qw.cuda(), kw.cuda(), table, p32.long().cuda())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_no_tokens_and_one_side_without_heads():
    from kernels import build_rope_table, qk_norm_rope
    q, k, qw, kw, _ = data(4, 4, 2, 64, torch.float16, 6)
    table = build_rope_table(10, 64, device="cuda")
    qo, ko = qk_norm_rope(q[:0].cuda(), k[:0].cuda(), qw.cuda(), kw.cuda(), table,
                          torch.empty(0, dtype=torch.int32, device="cuda"))
    assert qo.shape == (0, 4, 64) and ko.shape == (0, 2, 64)
    pos = torch.arange(4, dtype=torch.int32)
    qo, ko = qk_norm_rope(q.cuda(), k[:, :0].cuda(), qw.cuda(), kw.cuda(), table, pos.cuda())
    assert ko.shape == (4, 0, 64)
    check(qo, q, qw, table, pos, False)


def test_ctypes_path_and_stream_and_graph():
    """The launch without the extension, another stream, and a replayed graph
    give the same bits."""
    import kernels.norm_rope as m
    q, k, qw, kw, _ = data(50, 8, 2, 128, torch.bfloat16, 7)
    table = m.build_rope_table(64, 128, device="cuda")
    args = [t.cuda() for t in (q, k, qw, kw)] + [table, torch.arange(50, device="cuda") % 64]
    want = m.qk_norm_rope(*args)
    m.USE_EXT = False
    try:
        got = m.qk_norm_rope(*args)
    finally:
        m.USE_EXT = True
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = m.qk_norm_rope(*args)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got[0], want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = m.qk_norm_rope(*args)
    for i in range(3):
        args[0].copy_(torch.randn_like(args[0]))
        graph.replay()
        eager = m.qk_norm_rope(*args)
        torch.cuda.synchronize()
        assert torch.equal(held[0], eager[0]) and torch.equal(held[1], eager[1])


def test_table_of_far_positions():
    """The table's angles are those of 64 bits."""
    from kernels import build_rope_table
    t = build_rope_table(200001, 64, base=10000.0, device="cuda").cpu()
    for p, i in ((200000, 0), (199999, 1), (131072, 31)):
        a = p * 10000.0 ** (-2 * i / 64)
        assert abs(t[p, i].item() - math.cos(a)) <= 2 ** -24 + 1e-9
        assert abs(t[p, 32 + i].item() - math.sin(a)) <= 2 ** -24 + 1e-9


@pytest.mark.parametrize("bad", ["dtype", "mixed", "dim", "dims", "tokens", "weight", "wtype",
                                 "wmixed", "positions", "ptype", "table", "ttype", "wide", "odd",
                                 "eps", "device"])
def test_refusals(bad):
    """The same error with and without the extension, before any launch."""
    import kernels.norm_rope as m
    q, k, qw, kw, _ = data(6, 4, 2, 64, torch.float16, 31)
    q, k, qw, kw = (t.cuda() for t in (q, k, qw, kw))
    table = m.build_rope_table(16, 64, device="cuda")
    pos = torch.arange(6, device="cuda")
    kwargs = {}
    if bad == "dtype":
        q, k = q.double(), k.double()
    elif bad == "mixed":
        k = k.float()
    elif bad == "dim":
        q, k, qw, kw = (t[..., :48] for t in (q, k, qw, kw))
    elif bad == "dims":
        q = q[0]
    elif bad == "tokens":
        k = k[:5]
    elif bad == "weight":
        kw = kw[:32]
    elif bad == "wtype":
        qw, kw = qw.bfloat16(), kw.bfloat16()
    elif bad == "wmixed":
        kw = kw.float()
    elif bad == "positions":
        pos = pos[:5]
    elif bad == "ptype":
        pos = pos.short()
    elif bad == "table":
        table = table[0]
    elif bad == "ttype":
        table = table.half()
    elif bad == "wide":
        table = m.build_rope_table(16, 128, device="cuda")
    elif bad == "odd":
        table = table[:, :24]
    elif bad == "eps":
        kwargs["eps"] = -1e-6
    else:
        pos = pos.cpu()
    seen = []
    for use in (True, False):
        m.USE_EXT = use
        try:
            with pytest.raises((ValueError, TypeError, AssertionError)) as e:
                m.qk_norm_rope(q, k, qw, kw, table, pos, **kwargs)
            seen.append((e.type, str(e.value)))
        finally:
            m.USE_EXT = True
    assert seen[0] == seen[1]
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,rot", [(64, 32), (128, 48), (128, 0), (256, 64), (32, 16)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T", [3, 3001])  # (one and four heads per lane group)
def test_infinities_stay_in_their_place(dtype, D, rot, inter, T):
    """An infinity makes its own value NaN and the rest of its row zeros; in a rotated
    pair both are NaN by the formula, in the dims behind them only itself.  A weight
    that is infinite or NaN touches its own dim alone there."""
    from kernels import build_rope_table, qk_norm_rope
    q, k, qw, kw, g = data(T, 5, 2, D, dtype, 7)
    table = (build_rope_table(5000, rot, device="cuda") if rot
             else torch.empty(5000, 0, device="cuda"))
    pos = torch.randint(0, 5000, (T,), generator=g, dtype=torch.int32)
    q[0, 0, D - 1] = math.inf
    q[1, 4, rot] = -math.inf
    q[T - 1, 2, rot + (D - rot) // 2] = math.inf
    q[2, 1, 0] = math.inf                               # (rotated, where rot > 0)
    k[T - 1, 1, D - 2] = math.nan                       # all of its row
    kw[rot + 1], kw[D - 1] = math.inf, math.nan
    qo, ko = qk_norm_rope(q.cuda(), k.cuda(), qw.cuda(), kw.cuda(), table, pos.cuda(),
                          interleaved=inter)
    check(qo, q, qw, table, pos, inter)
    want, tol = R.norm_rope(k, kw, table.cpu(), pos, inter, 1e-6)
    # (a value times the infinite weight is infinite in both)
    ko, inf = ko.cpu().double(), torch.isinf(want)
    assert torch.equal(ko[inf], want[inf])
    R.within(torch.where(inf, 0.0, ko), torch.where(inf, 0.0, want), torch.where(inf, 0.0, tol))
