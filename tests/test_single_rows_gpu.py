"""One token or one sequence out of a wider buffer: a dim of size one keeps any
stride, and torch calls such a tensor contiguous.  Results are those of a plain copy,
with and without the launch extension."""

import pytest
import torch

from kernels import _launch


def odd_row(*shape, dtype=torch.bfloat16, device="cpu", seed=0):
    """A ``[1, ...]`` view at an aligned address in a buffer whose rows are 4 values
    longer than a multiple of 8."""
    n = 1
    for s in shape[1:]:
        n *= s
    g = torch.Generator().manual_seed(seed)
    buf = torch.randn(3, -(-n // 8) * 8 + 4, generator=g).to(dtype).to(device)
    # (row 2 starts at a multiple of 8 values)
    return buf[:, :n].unflatten(1, shape[1:])[2:3]


@pytest.mark.parametrize("shape", [(1, 8, 128), (1, 4, 3, 64), (1, 1, 64), (1, 1, 1, 16)])
def test_strides_are_the_layouts(shape):
    t = odd_row(*shape)
    assert t.is_contiguous() and t.stride(0) % 8 and _launch.rows_ok(t)
    want = torch.empty(shape)
    assert _launch.strides(t) == _launch.strides(want)
    assert [_launch.stride_of(t, d) for d in range(len(shape))] == list(want.stride())


def plain(*ts):
    """Copies in the layout's own strides."""
    return [t.clone(memory_format=torch.contiguous_format) for t in ts]


def test_strides_of_other_tensors_are_their_own():
    t = torch.empty(4, 9, 128)[:, :3].transpose(0, 1)
    assert _launch.strides(t) == (0, t.stride(1), t.stride(0))
    empty = torch.empty(0, 4, 128)
    assert _launch.strides(empty) == (0, 128, 512)


@pytest.fixture(params=[True, False], ids=["extension", "ctypes"])
def launch(request):
    import kernels.attention as a
    import kernels.decode as d
    import kernels.decode_fp4 as d4
    import kernels.fp4_cache as f4
    import kernels.norm_rope as n
    import kernels.paged_cache as pc
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need an MI355X")
    mods = (a, d, d4, f4, n, pc)
    for m in mods:
        m.USE_EXT = request.param
    yield request.param
    for m in mods:
        m.USE_EXT = True


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_norms(launch, dtype):
    from kernels import build_rope_table, qk_norm_rope
    table, pos = build_rope_table(100, 128, device="cuda"), torch.tensor([37], device="cuda")
    w = torch.ones(128, dtype=dtype, device="cuda")
    for shape in ((1, 8, 128), (1, 8, 1, 128)):
        q = odd_row(*shape, dtype=dtype, device="cuda", seed=1)
        k = odd_row(1, 2, 128, dtype=dtype, device="cuda", seed=2)
        got = qk_norm_rope(q, k, w, w, table, pos)
        want = qk_norm_rope(*plain(q, k), w, w, table, pos)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_cache_in_4_bits(launch):
    from kernels import (allocate_fp4_cache, decode_attention_fp4, paged_kv_append_fp4,
                         speculative_decode_attention_fp4)
    H, D, page = 2, 128, 16
    k, v = (odd_row(1, H, D, device="cuda", seed=s) for s in (3, 4))
    ip = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    t = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    got, want = ([allocate_fp4_cache(3, page, H, D) for _ in range(2)] for _ in range(2))
    paged_kv_append_fp4(*got, t, t, k, v, ip)
    paged_kv_append_fp4(*want, t, t, *plain(k, v), ip)
    for a, b in zip(got, want):
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
        assert a.codes.any()
    kw = dict(kv_indptr=torch.tensor([1], dtype=torch.int32, device="cuda"), k_block_table=t,
              v_block_table=t)
    q = odd_row(1, 8, D, device="cuda", seed=5)
    assert torch.equal(decode_attention_fp4(q, *want, **kw),
                       decode_attention_fp4(*plain(q), *want, **kw))
    q = odd_row(1, 8, 3, D, device="cuda", seed=6)
    assert torch.equal(speculative_decode_attention_fp4(q, *want, **kw),
                       speculative_decode_attention_fp4(*plain(q), *want, **kw))


@pytest.mark.gpu
def test_cache_in_16_bits_and_prefill(launch):
    from kernels import decode_attention, flash_attention_v2, speculative_decode_attention
    from kernels.paged_cache import paged_kv_append
    H, D, page = 2, 128, 16
    k, v = (odd_row(1, H, D, device="cuda", seed=s) for s in (7, 8))
    ip = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    t = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    got, want = ([torch.zeros(3 * page, H, D, dtype=k.dtype, device="cuda") for _ in range(2)]
                 for _ in range(2))
    paged_kv_append(*got, t, t, k, v, ip, page)
    paged_kv_append(*want, t, t, *plain(k, v), ip, page)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[0].any()
    kw = dict(kv_indptr=ip[1:], k_block_table=t, v_block_table=t, kv_page_size=page)
    q = odd_row(1, 8, D, device="cuda", seed=9)
    assert torch.equal(decode_attention(q, *want, **kw), decode_attention(*plain(q), *want, **kw))
    q = odd_row(1, 8, 3, D, device="cuda", seed=10)
    assert torch.equal(speculative_decode_attention(q, *want, **kw),
                       speculative_decode_attention(*plain(q), *want, **kw))
    q = odd_row(1, 8, 5, D, device="cuda", seed=11)      # dense, one sequence
    kd, vd = (odd_row(1, H, 9, D, device="cuda", seed=s) for s in (12, 13))
    assert torch.equal(flash_attention_v2(q, kd, vd),
                       flash_attention_v2(*plain(q, kd, vd)))
