"""include/fa2_latent.h without a GPU: exports, struct layouts, and the refusals of
the C entry points and of the Python wrappers, all before any device work."""

import ctypes
import os
import re

import pytest
import torch

import kernels
from kernels import _fa2, _latent

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NULL, LAYOUT, DTYPE, MASK, SHAPE, DIM, ALIGN, PAGED, RAGGED, WORKSPACE = range(1, 11)
LARGE, QLAYOUT = 13, 14


def test_exports_and_sizes():
    text = open(os.path.join(ROOT, "include", "fa2_latent.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = set(re.findall(r"^[A-Za-z_][\w\s\*]*?\b(fa2_\w+)\s*\(", text, flags=re.M))
    assert names == set(_latent.EXPORTS)
    lib = ctypes.CDLL(_fa2.LIB_PATH)
    for n in names:
        assert hasattr(lib, n), n
    L = _latent.lib()
    for i, p in enumerate(_latent._PARAMS):
        assert L.fa2_latent_params_size(i) == ctypes.sizeof(p)
    assert L.fa2_latent_params_size(len(_latent._PARAMS)) == L.fa2_latent_params_size(-1) == 0


def fill(p, kw, pointers):
    for n in pointers.split():
        setattr(p, n, 0x1000)
    for n, v in kw.items():
        setattr(p, n, v)
    return p


def append(**kw):
    p = _latent.LatentAppendParams()
    p.dtype = p.weight_dtype = 1
    p.eps = 1e-6
    p.batch, p.num_rows, p.latent_dim, p.rope_dim = 2, 10, 512, 64
    p.page_size, p.num_pages, p.table_width, p.table_stride = 16, 10, 4, 4
    p.positions, p.rope_stride, p.x_ts = 100, 64, 576
    fill(p, kw, "x cache weight rope indptr block_table")
    return _latent.lib().fa2_latent_append(ctypes.byref(p), None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), DTYPE), (dict(dtype=-1), DTYPE), (dict(weight_dtype=0), DTYPE),
    (dict(latent_dim=128), DIM), (dict(latent_dim=0), DIM), (dict(rope_dim=32), DIM),
    (dict(batch=-1), SHAPE), (dict(num_rows=-1), SHAPE), (dict(page_size=0), SHAPE),
    (dict(num_pages=-1), SHAPE), (dict(table_width=-1), SHAPE), (dict(table_stride=-1), SHAPE),
    (dict(positions=-1), SHAPE), (dict(rope_stride=-64), SHAPE), (dict(x_ts=-576), SHAPE),
    (dict(eps=-1.0), SHAPE), (dict(eps=float("nan")), SHAPE), (dict(num_rows=2 ** 31), LARGE),
    (dict(page_size=2 ** 31), LARGE), (dict(positions=2 ** 31), LARGE), (dict(x_ts=577), ALIGN),
    (dict(rope_stride=66), ALIGN), (dict(x=0x1008), ALIGN), (dict(cache=0x1008), ALIGN),
    (dict(rows_out=0x1008), ALIGN), (dict(weight=0x1004), ALIGN), (dict(rope=0x1008), ALIGN),
    (dict(x=None), NULL), (dict(cache=None), NULL), (dict(weight=None), NULL),
    (dict(indptr=None), NULL), (dict(rope=None), NULL), (dict(block_table=None), NULL),
    (dict(num_rows=2 ** 26), LARGE), (dict(num_rows=2 ** 27, latent_dim=256), LARGE),  # the grid
])
def test_append_refusals(kw, code):
    assert append(**kw) == code


def test_append_nothing_to_do():
    assert append(num_rows=0, x=None) == append(batch=0, x=None) == 0
    assert _latent.lib().fa2_latent_append(None, None) == NULL


def latent(ws=True, **kw):
    p = _latent.LatentDecodeParams()
    p.dtype, p.batch, p.q_heads, p.q_len, p.latent_dim, p.rope_dim = 1, 2, 16, 3, 512, 64
    p.page_size, p.num_pages, p.table_width, p.table_stride = 16, 10, 4, 4
    p.q_sb, p.q_sh, p.q_ss = 16 * 3 * 576, 3 * 576, 576
    p.o_sb, p.o_sh, p.o_ss = 16 * 3 * 512, 3 * 512, 512
    p.softmax_scale = 0.07
    fill(p, kw, "q o cache kv_lens block_table")
    n = ctypes.c_size_t(0)
    rc = _latent.lib().fa2_latent_decode_workspace_size(ctypes.byref(p), ctypes.byref(n))
    if rc:
        return rc
    if ws:
        p.workspace, p.workspace_bytes = 0x1000, 2 ** 40
        for k, v in kw.items():
            setattr(p, k, v)
    return _latent.lib().fa2_latent_decode(ctypes.byref(p), None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), DTYPE), (dict(mask=1), MASK), (dict(mask=4), MASK), (dict(latent_dim=64), DIM),
    (dict(rope_dim=0), DIM), (dict(q_heads=0), SHAPE), (dict(batch=-1), SHAPE),
    (dict(q_len=-1), SHAPE), (dict(mask=3, q_len=65, o_sh=65 * 512), SHAPE),
    (dict(page_size=0), PAGED), (dict(num_pages=-1), PAGED), (dict(table_width=-1), PAGED),
    (dict(table_stride=-1), PAGED), (dict(num_pages=0), PAGED), (dict(kv_lens=None), PAGED),
    (dict(block_table=None), PAGED), (dict(q_heads=70000), LARGE), (dict(batch=2 ** 20), LARGE),
    (dict(table_width=2 ** 28, page_size=2 ** 10), LARGE), (dict(q_ss=577), ALIGN),
    (dict(o_sb=4), ALIGN), (dict(o_sh=512), QLAYOUT), (dict(q=0x1008), ALIGN),
    (dict(cache=0x1008), ALIGN), (dict(q=None), NULL), (dict(o=None), NULL),
    (dict(cache=None), NULL), (dict(mask=3), NULL), (dict(softmax_scale=0.0), SHAPE),
    (dict(softmax_scale=-1.0), SHAPE), (dict(softmax_scale=float("inf")), SHAPE),
    (dict(softmax_scale=float("nan")), SHAPE), (dict(workspace=0x1008), ALIGN),
    (dict(workspace_bytes=16), WORKSPACE), (dict(ws=False), WORKSPACE),
])
def test_latent_decode_refusals(kw, code):
    assert latent(**kw) == code


def test_latent_decode_nothing_to_do():
    assert latent(ws=False, batch=0, q=None) == latent(ws=False, q_len=0, o_sh=0, q=None) == 0
    assert _latent.lib().fa2_latent_decode(None, None) == NULL
    assert _latent.lib().fa2_latent_decode_workspace_size(None, None) == NULL


def tree(ws=True, **kw):
    p = _latent.TreeDecodeParams()
    p.layout, p.dtype, p.batch, p.q_heads, p.kv_heads, p.head_dim, p.q_len = 0, 1, 2, 8, 2, 128, 5
    p.kv_len = 160
    p.q_sb, p.q_sh, p.q_ss = 8 * 5 * 128, 5 * 128, 128
    p.o_sb, p.o_sh, p.o_ss = p.q_sb, p.q_sh, p.q_ss
    p.k_sb, p.k_sh, p.k_ss = 2 * 160 * 128, 160 * 128, 128
    p.v_sb, p.v_sh, p.v_ss = p.k_sb, p.k_sh, p.k_ss
    p.page_size, p.table_width, p.k_table_stride, p.v_table_stride = 16, 4, 4, 4
    p.softmax_scale = 0.07
    fill(p, kw, "q k v o kv_indptr k_block_table v_block_table tree")
    for n, v in kw.items():
        if n != "ws":
            setattr(p, n, v)
    n = ctypes.c_size_t(0)
    rc = _latent.lib().fa2_tree_decode_workspace_size(ctypes.byref(p), ctypes.byref(n))
    if rc:
        return rc
    if ws:
        p.workspace, p.workspace_bytes = 0x1000, 2 ** 40
        for k, v in kw.items():
            setattr(p, k, v)
    return _latent.lib().fa2_tree_decode(ctypes.byref(p), None)


@pytest.mark.parametrize("kw,code", [
    (dict(layout=3), LAYOUT), (dict(layout=-1), LAYOUT), (dict(dtype=2), DTYPE),
    (dict(head_dim=32), DIM), (dict(head_dim=96), DIM), (dict(q_heads=7), SHAPE),
    (dict(kv_heads=0), SHAPE), (dict(kv_len=-1), SHAPE), (dict(q_len=65, o_sh=65 * 128), SHAPE),
    (dict(layout=2, page_size=0), PAGED), (dict(layout=2, table_width=-1), PAGED),
    (dict(layout=2, k_table_stride=-1), PAGED), (dict(layout=2, kv_indptr=None), PAGED),
    (dict(layout=2, kv_len=15), PAGED), (dict(layout=2, v_block_table=None), PAGED),
    (dict(layout=1, kv_indptr=None), RAGGED), (dict(k_ss=2 ** 25), LARGE), (dict(v_ss=-8), LARGE),
    (dict(batch=2 ** 20), LARGE), (dict(layout=2, table_width=2 ** 28, page_size=2 ** 10), LARGE),
    (dict(k_sh=4), ALIGN), (dict(o_sh=128), QLAYOUT), (dict(v=0x1008), ALIGN),
    (dict(q=None), NULL), (dict(k=None), NULL), (dict(tree=None), NULL),
    (dict(softmax_scale=0.0), SHAPE), (dict(workspace=0x1008), ALIGN),
    (dict(workspace_bytes=16), WORKSPACE), (dict(ws=False), WORKSPACE),
])
def test_tree_decode_refusals(kw, code):
    assert tree(**kw) == code


def prefill(**kw):
    p = _latent.LatentPrefillParams()
    p.layout, p.dtype, p.mask, p.batch, p.heads, p.head_dim, p.rope_dim = 0, 1, 2, 2, 8, 128, 64
    p.q_len = p.kv_len = 100
    p.q_sb, p.q_sh, p.q_ss = 8 * 100 * 192, 100 * 192, 192
    p.k_sb, p.k_sh, p.k_ss = 8 * 100 * 128, 100 * 128, 128
    p.v_sb, p.v_sh, p.v_ss = p.k_sb, p.k_sh, p.k_ss
    p.o_sb, p.o_sh, p.o_ss = p.k_sb, p.k_sh, p.k_ss
    p.kr_sb, p.kr_ss = 6400, 64
    p.softmax_scale = 0.07
    fill(p, kw, "q k kr v o q_indptr kv_indptr")
    for n, v in kw.items():
        setattr(p, n, v)
    return _latent.lib().fa2_latent_prefill(ctypes.byref(p), None)


@pytest.mark.parametrize("kw,code", [
    (dict(layout=2), LAYOUT), (dict(dtype=2), DTYPE), (dict(mask=3), MASK),
    (dict(head_dim=256), DIM), (dict(rope_dim=32), DIM), (dict(heads=0), SHAPE),
    (dict(q_len=-1), SHAPE), (dict(kv_len=-1), SHAPE), (dict(layout=1, q_indptr=None), RAGGED),
    (dict(layout=1, kv_indptr=None), RAGGED), (dict(q_ss=194), ALIGN), (dict(kr_ss=2), ALIGN),
    (dict(heads=70000), LARGE), (dict(k_ss=2 ** 25), LARGE), (dict(kr_ss=-64), LARGE),
    (dict(batch=2 ** 29), LARGE), (dict(batch=2 ** 21), LARGE), (dict(q=None), NULL), (dict(kr=None), NULL), (dict(o=None), NULL),
    (dict(kr=0x1008), ALIGN), (dict(softmax_scale=0.0), SHAPE),
    (dict(kv_len=4096, batch=1), WORKSPACE),  # splits: partials
])
def test_prefill_refusals(kw, code):
    assert prefill(**kw) == code


def test_prefill_nothing_to_do():
    assert prefill(batch=0, q=None) == prefill(q_len=0, q=None) == 0


# ---- the Python wrappers, without a device -------------------------------------------

def test_allocate_refusals():
    with pytest.raises(ValueError):
        kernels.allocate_latent_cache(2, 16, 128, device="cpu")
    with pytest.raises(ValueError):
        kernels.allocate_latent_cache(0, 16, 512, device="cpu")
    with pytest.raises(TypeError):
        kernels.allocate_latent_cache(2, 16, 512, torch.float32, device="cpu")
    assert kernels.allocate_latent_cache(2, 16, 256, device="cpu").shape == (2, 16, 320)


def test_wrappers_want_the_gpu():
    c = torch.zeros(2, 16, 576, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    t = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(AssertionError):
        kernels.paged_latent_append(c, t, c[0], i, torch.ones(512), torch.ones(4, 64))
    with pytest.raises(AssertionError):
        kernels.latent_decode_attention(c[:1], c, latent_dim=512, softmax_scale=1.0, kv_indptr=i,
                                        block_table=t)
    q = torch.zeros(1, 2, 3, 64, dtype=torch.float16)
    with pytest.raises(AssertionError):
        kernels.tree_decode_attention(q, q, q, torch.ones(3, 3, dtype=torch.bool))
    q = torch.zeros(1, 2, 3, 128, dtype=torch.float16)
    with pytest.raises(AssertionError):
        kernels.latent_attention(q, q[..., :64], q[0, :1, :, :64], q[..., :64])
    with pytest.raises(ValueError):
        kernels.latent_attention(q, q, q, q, True, causal_alignment="middle")
