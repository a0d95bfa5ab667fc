"""Query/key norms with rotation and the 4-bit paged cache: the measured cases.

Four operators that stand next to paged attention in a serving program:

* ``qk_norm_rope``: RMS norm of every query and key head and the position
  rotation, in one pass;
* ``paged_kv_append_fp4``: new K/V rows into a paged cache held in 4 bits;
* ``paged_kv_gather_fp4``: rows of that cache back in 16 or 32 bits, packed
  token by token for a prefill chunk;
* ``decode_attention_fp4`` / ``speculative_decode_attention_fp4``: attention of
  one or a few query tokens per sequence over that cache.

The cache: codes uint8 ``[pages, KVH, page, D/2]`` (value 2i of a row in byte
i's low nibble, 2i+1 in the high one; E2M1 with the sign in bit 3) and scales
uint8 ``[pages, KVH, page, D/32]`` (a value is ``e2m1 * 2**(scale - 127)``, 255
is NaN).  A block of 32 with largest magnitude a takes the least power of two
whose 6 is not passed by a after rounding (a < 7 steps).

Each case is a dict of plain values; lengths follow from (``n``, ``lo``,
``hi``, ``lens_seed``).
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False  # the framework's kernels (True) or the plain forms below

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "triton-kernels_amd")
_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EPS = 1e-6
MAX_POSITIONS = 32768


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # The projections of one decode step of a full batch: latency.
        dict(name="norm_rope_step", kind="norm_rope", dtype="bf16", t=64, m=0, hq=32, hkv=8,
             d=128, rot=128, inter=False),
        # ... of a prefill of 8192 packed tokens: the largest, bound by memory.
        dict(name="norm_rope_prefill", kind="norm_rope", dtype="bf16", t=8192, m=0, hq=32, hkv=8,
             d=128, rot=128, inter=False),
        # A speculative step's drafts, rotated in part and in neighbouring
        # pairs, the queries leaving head by head as the attention takes them.
        dict(name="norm_rope_drafts", kind="norm_rope", dtype="f16", t=77 * 5, m=5, hq=16, hkv=4,
             d=64, rot=32, inter=True),
        # A decode step's new token of each sequence into the 4-bit cache, and
        # the rows read back: latency.
        dict(name="append_step", kind="append", dtype="bf16", n=64, lo=1, hi=1, lens_seed=1,
             start=4000, hkv=8, d=128, page=16),
        # A prefill chunk of sequences of unequal lengths (the range of the
        # 16-bit append's case), read back as the chunk's attention does.
        dict(name="append_chunk", kind="append", dtype="bf16", n=16, lo=64, hi=1024, lens_seed=5,
             start=300, hkv=8, d=128, page=16),
        # One short context of a small model back in fp16.
        dict(name="gather_small", kind="gather", dtype="f16", n=1, lo=501, hi=501, lens_seed=0,
             hkv=4, d=64, page=16),
        # A batch's contexts back in bf16 for a prefill chunk over them.
        dict(name="gather_batch", kind="gather", dtype="bf16", n=32, lo=512, hi=8192, lens_seed=0,
             hkv=8, d=128, page=16),
        # A decode step of an interactive session: few sequences, short cache.
        dict(name="decode_small", kind="decode", dtype="f16", n=4, lo=1023, hi=1023, lens_seed=0,
             m=0, hq=32, hkv=8, d=128, page=16),
        # A decode step of a full serving batch (the 16-bit benchmark's d2).
        dict(name="decode_batch", kind="decode", dtype="bf16", n=64, lo=512, hi=8192, lens_seed=2,
             m=0, hq=32, hkv=8, d=128, page=16),
        # Long contexts, what a 4-bit cache is for: most keys per sequence.
        dict(name="decode_long", kind="decode", dtype="bf16", n=16, lo=16000, hi=32768,
             lens_seed=6, m=0, hq=32, hkv=4, d=128, page=64),
        # A speculative step, 8 drafts, heads of 64 dims without grouping (the
        # 16-bit benchmark's s1).
        dict(name="spec_mha", kind="decode", dtype="f16", n=16, lo=8192, hi=8200, lens_seed=3, m=8,
             hq=8, hkv=8, d=64, page=16),
        # A speculative step of a serving batch with grouped heads, odd lengths
        # and drafts: 20 query rows for each K/V row.
        dict(name="spec_gqa", kind="decode", dtype="bf16", n=33, lo=100, hi=4096, lens_seed=4, m=5,
             hq=16, hkv=4, d=128, page=16),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm_rope", "append", "gather", "decode", "decode", "spec"])
    dtype = rng.choice(["bf16", "f16"])
    hq, hkv = rng.choice([(8, 8), (8, 2), (16, 4), (16, 16), (32, 8), (32, 4), (16, 1)])
    d = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 16, 16, 32, 64, 8])
    seed = rng.randrange(1 << 20)
    if kind == "norm_rope":
        m = rng.choice([0, 0, 0, rng.randint(2, 8)])
        t = max(1, _log_int(rng, 1, 4096) // max(m, 1)) * max(m, 1)
        return dict(kind=kind, dtype=dtype if d == 256 else rng.choice([dtype, dtype, "f32"]), t=t,
                    m=m, hq=hq, hkv=hkv, d=d, rot=rng.choice([d, d, d // 2]),
                    inter=rng.random() < 0.3)
    if kind == "append":
        n = _log_int(rng, 1, 64)
        return dict(kind=kind, dtype=rng.choice([dtype, dtype, "f32"]), n=n, lo=1,
                    hi=_log_int(rng, 1, min(512, 8192 // n)), lens_seed=seed,
                    start=_log_int(rng, 1, 4000), hkv=min(hkv, 8), d=d, page=page)
    n = _log_int(rng, 1, 64)
    hkv = min(hkv, 4 if d == 256 else 8)
    hi = _log_int(rng, 40, min(32768, (100000 if kind == "gather" else 250000) // n))
    lo = rng.randint(max(8, hi // 10), hi)
    if kind == "gather":
        return dict(kind=kind, dtype=rng.choice([dtype, dtype, "f32"]), n=n, lo=lo, hi=hi,
                    lens_seed=seed, hkv=hkv, d=min(d, 128), page=page)
    return dict(kind="decode", dtype=dtype, n=n, lo=lo, hi=hi, lens_seed=seed,
                m=0 if kind == "decode" else rng.randint(2, 8), hq=hq, hkv=hkv, d=d, page=page)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _lens(case):
    r = random.Random(case["lens_seed"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["n"])]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + 17)


def _heads_data(shape, gen, dtype):
    """Normal values under a spread of sizes per head dim, a few dims large, as
    keys and values of trained models have them."""
    x = torch.randn(shape, generator=gen, device="cuda")
    size = torch.exp(0.6 * torch.randn(shape[-1], generator=gen, device="cuda"))
    size[torch.randint(0, shape[-1], (2,), generator=gen, device="cuda")] *= 6.0
    return (x * size).to(dtype)


def _pow2(e):
    """2**e in fp32 for whole numbers e in [-126, 128), by its bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantize(x, dtype):
    """(codes, scales) of x [..., D], by comparisons with the code borders."""
    blocks = x.float().unflatten(-1, (-1, 32))
    a = blocks.abs().amax(-1)
    mant, exp = torch.frexp(a)  # a = mant 2^exp, mant in [1/2, 1)
    e = exp - 3 + (mant >= 0.875).to(exp.dtype)
    lo, hi = (-23, 13) if dtype == torch.float16 else (-100, 125)
    e = torch.where(a == 0, lo, e).clamp(lo, hi)
    y = blocks * _pow2(-e).unsqueeze(-1)
    mag = y.abs()
    # ties go to the even code: above 1/4, from 3/4, above 5/4, from 7/4, ...
    code = ((mag > 0.25).to(torch.uint8) + (mag >= 0.75) + (mag > 1.25) + (mag >= 1.75)
            + (mag > 2.5) + (mag >= 3.5) + (mag > 5.0))
    code = code + 8 * torch.signbit(y).to(torch.uint8)
    finite = torch.isfinite(a)
    code = torch.where(finite.unsqueeze(-1), code, 0).flatten(-2)
    scale = torch.where(finite, e + 127, 255).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def _pool(case, pages, gen, dtype):
    shape = (pages, case["hkv"], case["page"], case["d"])
    return tuple(t.contiguous() for t in _quantize(_heads_data(shape, gen, dtype), dtype))


def _tables(lens, page, gen, count):
    """``count`` block tables over one pool's pages, shuffled."""
    need = [(n + page - 1) // page for n in lens]
    pages, width = sum(need) + 3, max(need)
    starts = torch.tensor([0] + need, device="cuda").cumsum(0)[:-1]
    cols = torch.arange(width, device="cuda")
    held = cols < torch.tensor(need, device="cuda")[:, None]
    at = torch.where(held, starts[:, None] + cols, 0)
    tables = [torch.where(held, torch.randperm(pages, generator=gen, device="cuda")[at], -1)
              .to(torch.int32) for _ in range(count)]
    return tables, pages


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _rope_table(rot):
    """[positions, rot]: cos then sin of position * 10000^(-2i/rot)."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = torch.arange(MAX_POSITIONS, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def prepare(case, seed):
    gen = _generator(seed)
    dtype = _DTYPES[case["dtype"]]
    kind, d, hkv = case["kind"], case["d"], case["hkv"]
    s = dict(case=case, dtype=dtype)
    if kind == "norm_rope":
        t, hq, m = case["t"], case["hq"], case["m"]
        # queries and keys are views of the fused projection's output
        qkv = _heads_data((t, hq + 2 * hkv, d), gen, dtype)
        q, k = qkv[:, :hq], qkv[:, hq:hq + hkv]
        if m:
            q = q.unflatten(0, (t // m, m)).transpose(1, 2)  # [B, Hq, M, D]
        w = 1 + 0.1 * torch.randn((2, d), generator=gen, device="cuda")
        step = m if m else (t if t > 256 else 1)  # tokens in a row of one sequence
        first = torch.randint(0, MAX_POSITIONS - step + 1, (t // step,), generator=gen, device="cuda")
        pos = (first[:, None] + torch.arange(step, device="cuda")).flatten().to(torch.int32)
        s.update(q=q, k=k, qw=w[0].to(dtype), kw=w[1].to(dtype), pos=pos,
                 rope=_rope_table(case["rot"]))
        return s
    lens = _lens(case)
    page = case["page"]
    if kind == "append":
        start = random.Random(case["lens_seed"] + 1).choices(range(case["start"] + 1), k=len(lens))
        (kt, vt), pages = _tables([a + b for a, b in zip(start, lens)], page, gen, 2)
        t = sum(lens)
        # keys leave the norm, values are a view of the fused projection's output
        kv = _heads_data((t, 2 * hkv, d), gen, dtype)
        s.update(k=kv[:, :hkv].contiguous(), v=kv[:, hkv:], kt=kt, vt=vt,
                 kc=tuple(torch.zeros((pages, hkv, page, x), dtype=torch.uint8, device="cuda")
                          for x in (d // 2, d // 32)),
                 vc=tuple(torch.zeros((pages, hkv, page, x), dtype=torch.uint8, device="cuda")
                          for x in (d // 2, d // 32)),
                 indptr=torch.nn.functional.pad(_int32(lens).cumsum(0), (1, 0)).to(torch.int32),
                 start=_int32(start), rows=t)
        return s
    (kt, vt), pages = _tables(lens, page, gen, 2)
    s.update(kc=_pool(case, pages, gen, dtype), vc=_pool(case, pages, gen, dtype), kt=kt, vt=vt)
    if kind == "gather":
        s.update(indptr=torch.nn.functional.pad(_int32(lens).cumsum(0), (1, 0)).to(torch.int32),
                 rows=sum(lens))
        return s
    m = case["m"]
    shape = (len(lens), case["hq"], m, d) if m else (len(lens), case["hq"], d)
    s.update(q=torch.randn(shape, generator=gen, device="cuda").to(dtype), lens=_int32(lens))
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

_calls = {}


def _framework():
    if not _calls:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        import kernels
        _calls.update(vars(kernels))
    return _calls


def run(s):
    if own:
        return _run_own(s)
    kind = s["case"]["kind"]
    if kind == "norm_rope":
        return _plain_norm_rope(s)
    if kind == "append":
        return _plain_append(s)
    if kind == "gather":
        return _plain_gather(s, s["indptr"], None)
    return _plain_decode(s)


def _run_own(s):
    f = _framework()
    case = s["case"]
    kind = case["kind"]
    if kind == "norm_rope":
        return f["qk_norm_rope"](s["q"], s["k"], s["qw"], s["kw"], s["rope"], s["pos"], eps=EPS,
                                 interleaved=case["inter"])
    if kind == "append":
        f["paged_kv_append_fp4"](s["kc"], s["vc"], s["kt"], s["vt"], s["k"], s["v"], s["indptr"],
                                 start_pos=s["start"])
        return f["paged_kv_gather_fp4"](s["kc"], s["vc"], s["kt"], s["vt"], s["indptr"], s["rows"],
                                        start_pos=s["start"], dtype=s["dtype"])
    if kind == "gather":
        return f["paged_kv_gather_fp4"](s["kc"], s["vc"], s["kt"], s["vt"], s["indptr"], s["rows"],
                                        dtype=s["dtype"])
    if case["m"]:
        return f["speculative_decode_attention_fp4"](s["q"], s["kc"], s["vc"], causal=True,
                                                     kv_indptr=s["lens"], k_block_table=s["kt"],
                                                     v_block_table=s["vt"])
    return f["decode_attention_fp4"](s["q"], s["kc"], s["vc"], kv_indptr=s["lens"],
                                     k_block_table=s["kt"], v_block_table=s["vt"])


def _plain_norm_rope(s):
    return (_plain_norm_rope_of(s["q"], s["qw"], s), _plain_norm_rope_of(s["k"], s["kw"], s))


def _plain_norm_rope_of(x, w, s):
    rot, m = s["case"]["rot"], s["case"]["m"]
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w.float()
    cs = s["rope"][s["pos"].long()]
    if x.dim() == 4:  # [B, H, M, D]
        cs = cs.unflatten(0, (-1, m)).unsqueeze(1)
    else:
        cs = cs.unsqueeze(1)
    c, sn = cs[..., :rot // 2], cs[..., rot // 2:]
    head, tail = y[..., :rot], y[..., rot:]
    if s["case"]["inter"]:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack([a * c - b * sn, b * c + a * sn], -1).flatten(-2)
    else:
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        head = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    return torch.cat([head, tail], -1).to(x.dtype)


def _plain_rows(indptr, start, rows, table, page):
    """(page, row in it) of each packed row."""
    t = torch.arange(rows, device="cuda")
    b = torch.searchsorted(indptr[1:].long(), t, right=True)
    n = t - indptr.long()[b] + (start.long()[b] if start is not None else 0)
    return table[b, n // page].long(), n % page


def _plain_append(s):
    page = s["case"]["page"]
    pk, ok = _plain_rows(s["indptr"], s["start"], s["rows"], s["kt"], page)
    pv, ov = _plain_rows(s["indptr"], s["start"], s["rows"], s["vt"], page)
    s["kc"][0][pk, :, ok], s["kc"][1][pk, :, ok] = _quantize(s["k"], s["dtype"])
    s["vc"][0][pv, :, ov], s["vc"][1][pv, :, ov] = _quantize(s["v"], s["dtype"])
    return _plain_gather(s, s["indptr"], s["start"])


def _plain_values(codes, scales):
    """The fp32 values that codes [..., D/2] and scales [..., D/32] stand for."""
    lut = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=codes.device)
    nib = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    x = lut[nib.int()].unflatten(-1, (-1, 32))
    f = torch.where(scales == 255, math.nan, _pow2(scales.int() - 127))
    return (x * f.unsqueeze(-1)).flatten(-2)


def _plain_gather(s, indptr, start):
    page = s["case"]["page"]
    pk, ok = _plain_rows(indptr, start, s["rows"], s["kt"], page)
    pv, ov = _plain_rows(indptr, start, s["rows"], s["vt"], page)
    return (_plain_values(s["kc"][0][pk, :, ok], s["kc"][1][pk, :, ok]).to(s["dtype"]),
            _plain_values(s["vc"][0][pv, :, ov], s["vc"][1][pv, :, ov]).to(s["dtype"]))


def _plain_decode(s):
    case = s["case"]
    m, hkv, d = max(case["m"], 1), case["hkv"], case["d"]
    q = s["q"].float().reshape(case["n"], hkv, -1, d)  # rows: (head in group, draft)
    k = _plain_values(s["kc"][0][s["kt"].long()], s["kc"][1][s["kt"].long()])  # [B, W, H, P, D]
    k = k.transpose(1, 2).flatten(2, 3).contiguous()
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()) * d ** -0.5
    key = torch.arange(k.shape[2], device="cuda")
    draft = torch.arange(q.shape[2], device="cuda") % m
    last = s["lens"].long()[:, None] - m + draft if case["m"] else s["lens"].long()[:, None] - 1
    seen = key <= last[:, :, None] if case["m"] else (key <= last[:, :, None]).expand(-1, q.shape[2], -1)
    scores = torch.where(seen[:, None], scores, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    v = _plain_values(s["vc"][0][s["vt"].long()], s["vc"][1][s["vt"].long()])
    o = torch.matmul(p, v.transpose(1, 2).flatten(2, 3).contiguous()) / p.sum(-1, keepdim=True)
    return o.reshape(s["q"].shape).to(s["dtype"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    eb, d, hkv = _BYTES[case["dtype"]], case["d"], case["hkv"]
    if case["kind"] == "norm_rope":
        values = case["t"] * (case["hq"] + hkv) * d
        return dict(bytes=2 * values * eb + case["t"] * (4 + case["rot"] * 4) + 2 * d * eb,
                    flops=8 * values)
    lens = _lens(case)
    rows = sum(lens)
    held = d // 2 + d // 32  # bytes of a cached row of one head
    pages = sum((n + case["page"] - 1) // case["page"] for n in lens)
    if case["kind"] == "append":  # rows in, cache out; cache in, rows out
        return dict(bytes=2 * rows * hkv * 2 * (d * eb + held), flops=6 * rows * hkv * d)
    if case["kind"] == "gather":
        return dict(bytes=2 * rows * hkv * (d * eb + held) + 8 * pages, flops=2 * rows * hkv * d)
    q = case["n"] * max(case["m"], 1) * case["hq"] * d
    return dict(bytes=2 * rows * hkv * held + 2 * q * eb + 8 * pages,
                flops=4 * rows * max(case["m"], 1) * case["hq"] * d)


# ---------------------------------------------------------------------------
# in 64 bits
# ---------------------------------------------------------------------------

def _power(e):
    return ((e + 1023) << 52).view(torch.float64)


def _exact_values(codes, scales):
    """E2M1 by its fields: s eem -> (-1)^s 2^(ee-1) (1 + m/2), 0 and 1/2 below."""
    nib = torch.empty(codes.shape[:-1] + (2 * codes.shape[-1],), dtype=torch.float64, device="cuda")
    for i, n in ((0, codes & 15), (1, codes >> 4)):
        ee, mm = ((n >> 1) & 3).double(), (n & 1).double()
        mag = torch.where(ee == 0, 0.5 * mm, 2.0 ** (ee - 1) * (1 + 0.5 * mm))
        nib[..., i::2] = torch.where(n >= 8, -mag, mag)
    f = torch.where(scales == 255, math.nan, _power(scales.long() - 127))
    return nib * f.repeat_interleave(32, -1)


def _exact_round(x, dtype):
    """What the cache keeps of rows x [T, H, D]: the nearest of the 15 values at
    the block's scale, the even code where two are as near."""
    y = x.double().unflatten(-1, (-1, 32))
    a = y.abs().amax(-1, keepdim=True)
    fl = (a.view(torch.int64) >> 52) - 1023  # floor(log2 a)
    e = fl - 2 + (a >= 1.75 * _power(fl)).long()
    lo, hi = (-23, 13) if dtype == torch.float16 else (-100, 125)
    e = torch.where(a > 0, e, lo).clamp(lo, hi)
    r = (y * _power(-e)).abs().clamp(max=6.0)
    # the grid's step: 1/2 below 2, 1 below 4, 2 above; round() ties to even
    step = torch.where(r < 2, 0.5, torch.where(r < 4, 1.0, 2.0))
    r = torch.round(r / step) * step
    return (torch.sign(y) * r * _power(e)).flatten(-2)


def _exact_of_rows(s, cache, table, lens, start):
    page, got = s["case"]["page"], []
    for b, n in enumerate(lens):
        at = torch.arange(start[b], start[b] + n, device="cuda")
        pages = table[b].long()[at // page]
        got.append(_exact_values(cache[0][pages, :, at % page], cache[1][pages, :, at % page]))
    return got


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm_rope":
        rot, m, outs = case["rot"], case["m"], []
        half = rot // 2
        cs = s["rope"].double()[s["pos"].long()]
        for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
            y = x.double()
            y = w.double() * y / torch.sqrt(y.square().mean(-1, keepdim=True) + EPS)
            c = cs.reshape(-1, m, rot)[:, None] if x.dim() == 4 else cs[:, None]
            z = y.clone()
            for i in range(half):
                p, q = (2 * i, 2 * i + 1) if case["inter"] else (i, i + half)
                z[..., p] = y[..., p] * c[..., i] - y[..., q] * c[..., half + i]
                z[..., q] = y[..., q] * c[..., i] + y[..., p] * c[..., half + i]
            outs.append(z)
        return tuple(outs)
    if case["kind"] == "append":
        return _exact_round(s["k"], s["dtype"]), _exact_round(s["v"], s["dtype"])
    lens = _lens(case)
    ks = _exact_of_rows(s, s["kc"], s["kt"], lens, [0] * len(lens))
    vs = _exact_of_rows(s, s["vc"], s["vt"], lens, [0] * len(lens))
    if case["kind"] == "gather":
        return torch.cat(ks), torch.cat(vs)
    q = s["q"].double()
    out = torch.empty_like(q)
    group = case["hq"] // case["hkv"]
    for b, n in enumerate(lens):
        for h in range(case["hq"]):
            k, v = ks[b][:, h // group], vs[b][:, h // group]
            x = q[b, h].reshape(-1, case["d"])  # the drafts of this head
            logits = x @ k.T / math.sqrt(case["d"])
            for i in range(x.shape[0]):
                logits[i, n - x.shape[0] + 1 + i:] = -math.inf
            out[b, h] = (torch.softmax(logits, -1) @ v).reshape(out[b, h].shape)
    return out
