"""include/fa2_ops.h without a GPU: exports, struct layouts, and the refusals of
the C entry points and of the Python wrappers, all before any device work."""

import ctypes
import os
import re

import pytest
import torch

from kernels import _fa2, _ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_exports_and_sizes():
    text = open(os.path.join(ROOT, "include", "fa2_ops.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = set(re.findall(r"^[A-Za-z_][\w\s\*]*?\b(fa2_\w+)\s*\(", text, flags=re.M))
    assert names == set(_ops.EXPORTS)
    lib = ctypes.CDLL(_fa2.LIB_PATH)
    for n in names:
        assert hasattr(lib, n), n
    for i, p in enumerate((_ops.NormRopeParams, _ops.Fp4RowsParams, _ops.Fp4DecodeParams)):
        assert _ops.lib().fa2_ops_params_size(i) == ctypes.sizeof(p)
    assert _ops.lib().fa2_ops_params_size(3) == _ops.lib().fa2_ops_params_size(-1) == 0


def norm_rope(**kw):
    p = _ops.NormRopeParams()
    p.dtype = p.weight_dtype = 1
    p.eps = 1e-6
    p.tokens, p.q_heads, p.kv_heads, p.head_dim, p.rotary_dim = 10, 8, 2, 128, 128
    p.positions, p.rope_stride, p.q_rows, p.k_rows = 100, 128, 10, 10
    p.q_sh = p.k_sh = p.qo_sh = p.ko_sh = 128
    p.q_ss = p.qo_ss = 1024
    p.k_ss = p.ko_ss = 256
    for n in "q k q_out k_out q_weight k_weight rope position".split():
        setattr(p, n, 0x1000)
    for n, v in kw.items():
        setattr(p, n, v)
    return _ops.lib().fa2_norm_rope(ctypes.byref(p), None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=3), 3), (dict(weight_dtype=0), 3), (dict(head_dim=96), 6), (dict(head_dim=0), 6),
    (dict(rotary_dim=8), 5), (dict(rotary_dim=144), 5), (dict(rotary_dim=-16), 5),
    (dict(tokens=-1), 5), (dict(q_heads=-1), 5), (dict(eps=-1.0), 5), (dict(eps=float("nan")), 5),
    (dict(q_rows=0), 5), (dict(tokens=2 ** 31), 13), (dict(q_heads=70000), 13),
    (dict(q_ss=4), 7), (dict(ko_sh=129), 7), (dict(rope_stride=130), 7), (dict(q=0x1008), 7),
    (dict(k_weight=0x1004), 7), (dict(rope=0x1008), 7), (dict(q=None), 1), (dict(k_out=None), 1),
    (dict(position=None), 1), (dict(rope=None), 1), (dict(tokens=2 ** 29, q_rows=2 ** 29,
                                                          k_rows=2 ** 29, q_heads=65536), 13),
])
def test_norm_rope_refusals(kw, code):
    assert norm_rope(**kw) == code


def test_norm_rope_nothing_to_do():
    assert norm_rope(tokens=0, q_rows=0, k_rows=0) == 0
    assert norm_rope(q_heads=0, kv_heads=0, q=None, k=None) == 0
    assert _ops.lib().fa2_norm_rope(None, None) == 1


def rows(entry="fa2_fp4_append", **kw):
    p = _ops.Fp4RowsParams()
    p.dtype, p.batch, p.kv_heads, p.head_dim, p.num_rows = 1, 2, 4, 128, 30
    p.page_size, p.num_pages, p.table_width = 16, 10, 4
    p.k_table_stride = p.v_table_stride = 4
    p.k_ts = p.v_ts = 512
    p.k_hs = p.v_hs = 128
    for n in "k v k_codes k_scales v_codes v_scales indptr k_block_table v_block_table".split():
        setattr(p, n, 0x1000)
    for n, v in kw.items():
        setattr(p, n, v)
    return getattr(_ops.lib(), entry)(ctypes.byref(p), None)


@pytest.mark.parametrize("entry", ["fa2_fp4_append", "fa2_fp4_gather"])
@pytest.mark.parametrize("kw,code", [
    (dict(dtype=-1), 3), (dict(head_dim=32), 6), (dict(head_dim=192), 6), (dict(kv_heads=0), 5),
    (dict(batch=-1), 5), (dict(page_size=0), 5), (dict(num_pages=-1), 5), (dict(num_rows=-1), 5),
    (dict(k_table_stride=-1), 5), (dict(num_rows=2 ** 30), 13), (dict(page_size=2 ** 31), 13),
    (dict(k_ts=516), 7), (dict(v_hs=4), 7), (dict(k=0x1008), 7), (dict(v_codes=0x1001), 7),
    (dict(k=None), 1), (dict(indptr=None), 1), (dict(k_scales=None), 1), (dict(v=None), 1),
    (dict(v_scales=None), 1),
])
def test_rows_refusals(entry, kw, code):
    assert rows(entry, **kw) == code


@pytest.mark.parametrize("entry", ["fa2_fp4_append", "fa2_fp4_gather"])
@pytest.mark.parametrize("kw", [dict(page_size=2 ** 23), dict(kv_heads=2 ** 25),
                                dict(kv_heads=2 ** 62), dict(kv_heads=2 ** 14, page_size=2 ** 11)])
def test_rows_pages_past_31_bits(entry, kw):
    """Offsets inside a page are 32-bit: larger pages are refused."""
    assert rows(entry, **kw) == 13


def test_rows_nothing_to_do():
    assert rows(batch=0) == 0 and rows(num_rows=0) == 0
    assert _ops.lib().fa2_fp4_append(None, None) == 1


def decode_params(**kw):
    p = _ops.Fp4DecodeParams()
    p.dtype, p.mask = 1, 2
    p.batch, p.q_heads, p.kv_heads, p.head_dim, p.q_len = 3, 8, 2, 128, 2
    p.page_size, p.num_pages, p.table_width = 16, 10, 4
    p.k_table_stride = p.v_table_stride = 4
    p.q_sb = p.o_sb = 2048
    p.q_sh = p.o_sh = 256
    p.q_ss = p.o_ss = 128
    for n in ("q o k_codes k_scales v_codes v_scales kv_lens k_block_table v_block_table "
              "workspace").split():
        setattr(p, n, 0x1000)
    p.softmax_scale = 128 ** -0.5
    for n, v in kw.items():
        setattr(p, n, v)
    return p


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), 3), (dict(mask=1), 4), (dict(mask=3), 4), (dict(head_dim=32), 6),
    (dict(q_heads=7), 5), (dict(q_heads=0), 5), (dict(batch=-1), 5), (dict(page_size=0), 8),
    (dict(num_pages=-1), 8), (dict(batch=65537), 13), (dict(q_heads=131072), 13),
    (dict(page_size=2 ** 24), 13), (dict(table_width=2 ** 27), 13), (dict(q_sh=128), 14),
    (dict(o_ss=256), 14), (dict(q_ss=132), 7), (dict(batch=60000, table_width=2 ** 21,
                                                     page_size=256, kv_heads=1, q_heads=4), 13),
])
def test_decode_refusals(kw, code):
    p = decode_params(**kw)
    n = ctypes.c_size_t(1)
    assert _ops.lib().fa2_fp4_decode_workspace_size(ctypes.byref(p), ctypes.byref(n)) == code
    assert _ops.lib().fa2_fp4_decode(ctypes.byref(p), None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), 1), (dict(v_scales=None), 1), (dict(kv_lens=None), 8), (dict(num_pages=0), 8),
    (dict(k_block_table=None), 8), (dict(o=0x1008), 7), (dict(v_codes=0x1004), 7), (dict(), 10),
    (dict(workspace=None), 10), (dict(head_dim=256, k_scales=0x1001, q_sb=4096, o_sb=4096,
                                      q_sh=512, o_sh=512, q_ss=256, o_ss=256), 7),
])
def test_decode_pointer_refusals(kw, code):
    p = decode_params(**kw)
    assert _ops.lib().fa2_fp4_decode(ctypes.byref(p), None) == code


def test_decode_workspace_off_16_bytes():
    p = decode_params(workspace=0x1008, workspace_bytes=1 << 30)
    assert _ops.lib().fa2_fp4_decode(ctypes.byref(p), None) == 7


def test_decode_workspace_and_nothing_to_do():
    n = ctypes.c_size_t(0)
    size = lambda p: (_ops.lib().fa2_fp4_decode_workspace_size(ctypes.byref(p), ctypes.byref(n)),
                      n.value)  # noqa: E731
    rc, small = size(decode_params())
    assert rc == 0 and small > 0
    assert size(decode_params(batch=0)) == (0, 0)
    assert size(decode_params(q_len=0, q_sh=0, o_sh=0)) == (0, 0)
    assert _ops.lib().fa2_fp4_decode(ctypes.byref(decode_params(batch=0)), None) == 0
    assert _ops.lib().fa2_fp4_decode_workspace_size(ctypes.byref(decode_params()), None) == 1
    assert _ops.lib().fa2_fp4_decode(None, None) == 1


def test_error_text_names_the_operator():
    e = _ops.OpsError("decode_attention_fp4", 6)
    assert "decode_attention_fp4" in str(e) and e.code == 6 and isinstance(e, RuntimeError)


# ---- the Python wrappers: checks that come before the device is needed ---------

def test_wrappers_need_the_gpu():
    import kernels as K
    q, k = torch.zeros(4, 8, 128).half(), torch.zeros(4, 2, 128).half()
    w, table, pos = torch.ones(128).half(), torch.zeros(10, 128), torch.arange(4)
    with pytest.raises(AssertionError, match="CUDA"):
        K.qk_norm_rope(q, k, w, w, table, pos)
    with pytest.raises(AssertionError, match="dtype"):
        K.qk_norm_rope(q, k.float(), w, w, table, pos)
    c = K.allocate_fp4_cache(3, 16, 2, 128, device="cpu")
    assert c.codes.shape == (3, 2, 16, 64) and c.scales.shape == (3, 2, 16, 4)
    kt = torch.zeros(1, 3, dtype=torch.int32)
    ip = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(AssertionError, match="CUDA"):
        K.paged_kv_append_fp4(c, c, kt, kt, k, k, ip)
    with pytest.raises(AssertionError, match="CUDA"):
        K.paged_kv_gather_fp4(c, c, kt, kt, ip, 4)
    with pytest.raises(AssertionError, match="CUDA"):
        K.decode_attention_fp4(q, c, c, kv_indptr=ip, k_block_table=kt, v_block_table=kt)
    with pytest.raises(AssertionError, match="M <= 16"):
        K.speculative_decode_attention_fp4(torch.zeros(1, 8, 17, 128).half(), c, c, kv_indptr=ip,
                                           k_block_table=kt, v_block_table=kt)
    with pytest.raises(ValueError, match=r"\[B, QH, D\]"):
        K.decode_attention_fp4(q[None], c, c, kv_indptr=ip, k_block_table=kt, v_block_table=kt)


@pytest.mark.parametrize("args", [(3, 16, 2, 96), (3, 16, 2, 32), (0, 16, 2, 64), (3, 0, 2, 64)])
def test_allocate_refusals(args):
    from kernels import allocate_fp4_cache
    with pytest.raises(ValueError):
        allocate_fp4_cache(*args, device="cpu")


def test_cache_refusals():
    from kernels.fp4_cache import check_cache
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    good = (u8(3, 2, 16, 64), u8(3, 2, 16, 4))
    with pytest.raises(TypeError):
        check_cache("x", (good[0].int(), good[1]), None)
    with pytest.raises(ValueError, match="contiguous"):
        check_cache("x", (u8(3, 2, 16, 128)[..., :64], good[1]), None)
    with pytest.raises(ValueError, match="4-D"):
        check_cache("x", (u8(48, 2, 64), good[1]), None)


def test_rope_table():
    from kernels import build_rope_table
    t = build_rope_table(1000, 64, base=1e6, device="cpu")
    assert t.shape == (1000, 64) and t.dtype == torch.float32
    a = 777 * 1e6 ** (-2 * 3 / 64)
    assert t[777, 3].item() == pytest.approx(torch.tensor(a, dtype=torch.float64).cos().item(),
                                             abs=2 ** -24)
    for r in (0, 8, -16):
        with pytest.raises(ValueError):
            build_rope_table(10, r, device="cpu")


@pytest.mark.parametrize("scale", [0.0, -0.0, -0.1, float("nan"), float("inf"), -float("inf")])
def test_decode_scale_refusals(scale):
    """Refused before any launch; the workspace's size does not ask for one."""
    n = ctypes.c_size_t(0)
    p = decode_params(softmax_scale=scale)
    assert _ops.lib().fa2_fp4_decode_workspace_size(ctypes.byref(p), ctypes.byref(n)) == 0
    p.workspace_bytes = n.value
    assert _ops.lib().fa2_fp4_decode(ctypes.byref(p), None) == 5
