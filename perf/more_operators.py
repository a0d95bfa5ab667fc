"""Latent attention and attention for trees of drafts: the measured cases.

Four operators of a serving program, next to paged attention:

* ``paged_latent_append``: new rows of a latent cache.  A row is a latent vector
  (normalised with a weight) and a key part shared by all heads (rotated to the
  row's position); the cache is ``[pages, page, latent + rope]``;
* ``latent_decode_attention``: attention of one or a few query tokens per
  sequence over that cache in the absorbed form: a key is a whole row, its value
  the latent, for every head;
* ``latent_attention``: the expanded form, for prefill: keys of each head
  followed by the shared rotated part, values of each head;
* ``tree_decode_attention``: query tokens that form a tree of drafts, the last
  keys of each sequence, over 16-bit K/V caches.

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
_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6
ROPE = 64  # values of the shared key part
MAX_POSITIONS = 32768


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # The new token of each sequence of a decode step: latency.
        dict(name="append_step", kind="append", dtype="bf16", n=64, lo=1, hi=1, lens_seed=1,
             start=500, latent=512, page=16, rows=False, inter=False),
        # A prefill chunk of sequences of unequal lengths, whose finished rows go
        # on to the up-projection.
        dict(name="append_chunk", kind="append", dtype="bf16", n=16, lo=64, hi=1024, lens_seed=5,
             start=300, latent=512, page=16, rows=True, inter=False),
        # A decode step of an interactive session: few sequences and heads.
        dict(name="latent_small", kind="latent", dtype="f16", n=4, lo=700, hi=1100, lens_seed=0,
             m=0, tree=False, hq=16, latent=512, page=16),
        # A decode step of a full serving batch with every head on one card.
        dict(name="latent_batch", kind="latent", dtype="bf16", n=64, lo=512, hi=8192, lens_seed=2,
             m=0, tree=False, hq=128, latent=512, page=16),
        # Long contexts with a share of the heads: bound by the cache's bytes.
        dict(name="latent_long", kind="latent", dtype="bf16", n=16, lo=16000, hi=32768,
             lens_seed=6, m=0, tree=False, hq=16, latent=512, page=64),
        # A speculative step over the latent cache: a tree of drafts, odd lengths.
        dict(name="latent_drafts", kind="latent", dtype="f16", n=17, lo=1000, hi=8192, lens_seed=3,
             m=7, tree=True, hq=32, latent=256, page=32),
        # A tree of drafts in an interactive session.
        dict(name="tree_small", kind="tree", dtype="f16", n=2, lo=500, hi=1500, lens_seed=4, m=13,
             hq=8, hkv=8, d=64, page=16),
        # A tree of drafts for each sequence of a serving batch.
        dict(name="tree_batch", kind="tree", dtype="bf16", n=64, lo=512, hi=8192, lens_seed=7, m=16,
             hq=32, hkv=8, d=128, page=16),
        # The widest trees: many more query rows for each key.
        dict(name="tree_wide", kind="tree", dtype="bf16", n=16, lo=2000, hi=8192, lens_seed=8, m=61,
             hq=32, hkv=8, d=128, page=16),
        # A short prompt.
        dict(name="prefill_small", kind="prefill", dtype="f16", n=1, lo=333, hi=333, lens_seed=0,
             past=0, hq=16, nope=128),
        # A prefill of prompts of unequal lengths: bound by the matrix rate.
        dict(name="prefill_ragged", kind="prefill", dtype="bf16", n=16, lo=128, hi=4096,
             lens_seed=9, past=0, hq=32, nope=128),
        # A chunk of a longer prompt over what is cached already.
        dict(name="prefill_chunk", kind="prefill", dtype="bf16", n=8, lo=100, hi=512, lens_seed=10,
             past=4000, hq=16, nope=128),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "latent", "latent", "tree", "tree", "prefill"])
    case = dict(kind=kind, dtype=rng.choice(["bf16", "f16"]), lens_seed=rng.randrange(1 << 20))
    page = rng.choice([16, 16, 16, 32, 64, 8, 5])
    if kind == "append":
        n = _log_int(rng, 1, 64)
        return dict(case, n=n, lo=1, hi=_log_int(rng, 1, min(512, 8192 // n)),
                    start=_log_int(rng, 1, 500), latent=rng.choice([512, 512, 256]), page=page,
                    rows=rng.random() < 0.5, inter=rng.random() < 0.3)
    if kind == "prefill":
        n = _log_int(rng, 1, 16)
        hi = _log_int(rng, 2, min(4096, 16384 // n))
        return dict(case, n=n, lo=rng.randint(max(1, hi // 10), hi), hi=hi,
                    past=rng.choice([0, 0, _log_int(rng, 1, 2000)]),
                    hq=rng.choice([4, 8, 16, 32]), nope=rng.choice([128, 128, 64]))
    m = rng.choice([0, 0, rng.randint(2, 16)]) if kind == "latent" else _log_int(rng, 2, 64)
    n = _log_int(rng, 1, 64)
    hi = _log_int(rng, 80, min(32768, 200000 // n))
    case.update(n=n, lo=rng.randint(max(m, hi // 10), hi), hi=hi, m=m, page=page)
    if kind == "latent":
        hq = rng.choice([8, 16, 16, 32, 64, 128])
        while hq * max(m, 1) > 256:
            hq //= 2
        return dict(case, tree=m > 0 and rng.random() < 0.5, hq=hq,
                    latent=rng.choice([512, 512, 256]))
    hq, hkv, d = rng.choice([(8, 8, 64), (8, 2, 128), (16, 4, 128), (32, 8, 128), (16, 16, 64),
                             (16, 1, 128), (8, 2, 256)])
    return dict(case, hq=hq, hkv=hkv, d=d)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _lens(case):
    r = random.Random(case["lens_seed"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["n"])]


def _starts(case):
    """The rows that each sequence holds already (append, prefill)."""
    r = random.Random(case["lens_seed"] + 1)
    return [r.randint(0, case["start" if case["kind"] == "append" else "past"])
            for _ in range(case["n"])]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + 29)


def _randn(shape, gen, dtype):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _spread(shape, gen, dtype):
    """Normal values under a spread of sizes per dim, as trained models have them."""
    x = torch.randn(shape, generator=gen, device="cuda")
    return (x * torch.exp(0.4 * torch.randn(shape[-1], generator=gen, device="cuda"))).to(dtype)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _indptr(lens):
    return torch.nn.functional.pad(_int32(lens).cumsum(0), (1, 0)).to(torch.int32)


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


def _rope_table():
    """[positions, ROPE]: cos then sin of position * 10000^(-2i/ROPE)."""
    inv = 10000.0 ** (-torch.arange(0, ROPE, 2, dtype=torch.float64, device="cuda") / ROPE)
    angle = torch.arange(MAX_POSITIONS, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _trees(n, m, seed):
    """[n, m, m]: draft i of a tree of m sees itself and its ancestors."""
    r = random.Random(seed)
    sees = torch.zeros((n, m, m), dtype=torch.bool)
    for b in range(n):
        for i in range(m):
            parent = r.randint(-1, i - 1)
            if parent >= 0:
                sees[b, i] = sees[b, parent]
            sees[b, i, i] = True
    return sees.cuda()


def prepare(case, seed):
    gen = _generator(seed)
    dtype = _DTYPES[case["dtype"]]
    kind = case["kind"]
    lens = _lens(case)
    s = dict(case=case, dtype=dtype)
    if kind == "append":
        start, width = _starts(case), case["latent"] + ROPE
        (table,), pages = _tables([a + b for a, b in zip(start, lens)], case["page"], gen, 1)
        # rows are a view of the fused down-projection's output, behind the queries' part
        down = _spread((sum(lens), 512 + width), gen, dtype)
        weight = 1 + 0.1 * torch.randn(case["latent"], generator=gen, device="cuda")
        s.update(x=down[:, 512:], weight=weight.to(dtype), rope=_rope_table(), table=table,
                 cache=_spread((pages, case["page"], width), gen, dtype), indptr=_indptr(lens),
                 start=_int32(start))
        return s
    if kind == "prefill":
        hq, nope = case["hq"], case["nope"]
        past = _starts(case)
        kv_lens = [a + b for a, b in zip(past, lens)]
        # keys and values of the heads are views of the up-projection's output, the
        # shared part one of the cached rows
        up = _spread((sum(kv_lens), hq, 2 * nope), gen, dtype)
        rows = _spread((sum(kv_lens), 512 + ROPE), gen, dtype)
        s.update(q=_randn((sum(lens), hq, nope + ROPE), gen, dtype), k=up[..., :nope],
                 v=up[..., nope:], k_rope=rows[:, 512:], q_indptr=_indptr(lens),
                 kv_indptr=_indptr(kv_lens), kv_lens=kv_lens)
        return s
    m, hq = case["m"], case["hq"]
    if kind == "latent":
        width = case["latent"] + ROPE
        (table,), pages = _tables(lens, case["page"], gen, 1)
        shape = (len(lens), hq, m, width) if m else (len(lens), hq, width)
        s.update(cache=_spread((pages, case["page"], width), gen, dtype), table=table,
                 q=_randn(shape, gen, dtype), scale=(128 + ROPE) ** -0.5)
    else:
        (kt, vt), pages = _tables(lens, case["page"], gen, 2)
        pool = (pages, case["page"], case["hkv"], case["d"])
        s.update(k=_spread(pool, gen, dtype), v=_spread(pool, gen, dtype), kt=kt, vt=vt,
                 q=_randn((len(lens), hq, m, case["d"]), gen, dtype), scale=case["d"] ** -0.5)
    s.update(lens=_int32(lens),
             tree=_trees(len(lens), m, seed) if kind == "tree" or case["tree"] else None)
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
    kind = s["case"]["kind"]
    if own:
        return _run_own(s, kind)
    if kind == "append":
        return _plain_append(s)
    if kind == "prefill":
        return _plain_prefill(s)
    return _plain_decode(s)


def _run_own(s, kind):
    f = _framework()
    case = s["case"]
    if kind == "append":
        rows = f["paged_latent_append"](s["cache"], s["table"], s["x"], s["indptr"], s["weight"],
                                        s["rope"], s["start"], eps=EPS,
                                        interleaved=case["inter"], return_rows=case["rows"])
        return (s["cache"], rows) if case["rows"] else s["cache"]
    if kind == "prefill":
        return f["latent_attention"](s["q"], s["k"], s["k_rope"], s["v"], is_causal=True,
                                     q_indptr=s["q_indptr"], kv_indptr=s["kv_indptr"],
                                     causal_alignment="bottom_right")
    if kind == "latent":
        return f["latent_decode_attention"](s["q"], s["cache"], latent_dim=case["latent"],
                                            softmax_scale=s["scale"], kv_indptr=s["lens"],
                                            block_table=s["table"], causal=case["m"] > 0,
                                            tree_mask=s["tree"])
    return f["tree_decode_attention"](s["q"], s["k"], s["v"], s["tree"], kv_indptr=s["lens"],
                                      k_block_table=s["kt"], v_block_table=s["vt"],
                                      kv_page_size=case["page"])


def _plain_append(s):
    case = s["case"]
    page, latent, half = case["page"], case["latent"], ROPE // 2
    t = torch.arange(s["x"].shape[0], device="cuda")
    b = torch.searchsorted(s["indptr"][1:].long(), t, right=True)
    pos = t - s["indptr"].long()[b] + s["start"].long()[b]
    x = s["x"].float()
    c, r = x[:, :latent], x[:, latent:]
    c = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS) * s["weight"].float()
    cos, sin = s["rope"][pos][:, :half], s["rope"][pos][:, half:]
    if case["inter"]:
        u, w = r[:, 0::2], r[:, 1::2]
        r = torch.stack([u * cos - w * sin, w * cos + u * sin], -1).flatten(-2)
    else:
        u, w = r[:, :half], r[:, half:]
        r = torch.cat([u * cos - w * sin, w * cos + u * sin], -1)
    rows = torch.cat([c, r], -1).to(s["dtype"])
    s["cache"][s["table"][b, pos // page].long(), pos % page] = rows
    return (s["cache"], rows) if case["rows"] else s["cache"]


def _plain_seen(s, keys):
    """[B, M, keys]: what draft m of each sequence sees."""
    m = max(s["case"]["m"], 1)
    key = torch.arange(keys, device="cuda")
    draft = key - (s["lens"].long()[:, None, None] - m)  # the key's place among the drafts
    row = torch.arange(m, device="cuda")[:, None]
    if s["tree"] is None:
        return draft <= row
    at = draft.clamp(0, m - 1).expand(-1, m, -1)
    return (draft < 0) | ((draft < m) & s["tree"].gather(2, at))


def _plain_decode(s):
    case = s["case"]
    m = max(case["m"], 1)
    if case["kind"] == "latent":  # one K/V head: whole rows, and their latents
        k = s["cache"][s["table"].long()].flatten(1, 2).float().unsqueeze(1)
        v = k[..., :case["latent"]]
    else:
        k, v = (x[t.long()].flatten(1, 2).float().transpose(1, 2)
                for x, t in ((s["k"], s["kt"]), (s["v"], s["vt"])))
    hkv = k.shape[1]
    q = s["q"].float().reshape(case["n"], hkv, -1, k.shape[-1])  # rows: (head in group, draft)
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()) * s["scale"]
    seen = _plain_seen(s, k.shape[2]).repeat(1, case["hq"] // hkv, 1)
    scores = torch.where(seen[:, None], scores, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    # (what lies behind a sequence's end has no weight and need not be finite)
    o = torch.matmul(p, v.contiguous()) / p.sum(-1, keepdim=True)
    return o.reshape(s["q"].shape[:-1] + (v.shape[-1],)).to(s["dtype"])


def _plain_prefill(s):
    q, k, v, r = s["q"], s["k"], s["v"], s["k_rope"]
    out = torch.empty(q.shape[:2] + v.shape[2:], dtype=s["dtype"], device="cuda")
    q0 = k0 = 0
    for nq, nk in zip(_lens(s["case"]), s["kv_lens"]):
        qb = q[q0:q0 + nq].float().transpose(0, 1).contiguous()
        kb = k[k0:k0 + nk].float().permute(1, 2, 0)
        rb = r[k0:k0 + nk].float().t().expand(q.shape[1], -1, -1)
        scores = torch.matmul(qb, torch.cat([kb, rb], 1)) * q.shape[-1] ** -0.5
        last = torch.arange(nk - nq, nk, device="cuda")
        scores.masked_fill_(torch.arange(nk, device="cuda") > last[:, None], -math.inf)
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        del scores
        o = torch.matmul(p, v[k0:k0 + nk].float().transpose(0, 1).contiguous())
        out[q0:q0 + nq] = (o / p.sum(-1, keepdim=True)).transpose(0, 1).to(s["dtype"])
        q0, k0 = q0 + nq, k0 + nk
    return out


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    lens, hq = _lens(case), case["hq"] if "hq" in case else 0
    rows = sum(lens)
    if case["kind"] == "append":  # rows in, rows out (twice where they are returned)
        values = rows * (case["latent"] + ROPE)
        return dict(bytes=2 * values * (3 if case["rows"] else 2) + rows * ROPE * 4,
                    flops=6 * values)
    if case["kind"] == "prefill":
        kv = [a + b for a, b in zip(_starts(case), lens)]
        pairs = sum(n * (k - n) + n * (n + 1) // 2 for n, k in zip(lens, kv))
        nope = case["nope"]
        return dict(bytes=2 * (rows * hq * (2 * nope + ROPE) + sum(kv) * (hq * 2 * nope + ROPE)),
                    flops=2 * (2 * nope + ROPE) * hq * pairs)
    m = max(case["m"], 1)
    pages = sum((n + case["page"] - 1) // case["page"] for n in lens)
    if case["kind"] == "latent":
        dk, dv = case["latent"] + ROPE, case["latent"]
        held, tables = rows * dk, 1
    else:
        dk = dv = case["d"]
        held, tables = rows * 2 * case["hkv"] * dk, 2
    return dict(bytes=2 * held + 2 * case["n"] * m * hq * (dk + dv) + 4 * tables * pages,
                flops=2 * (dk + dv) * hq * m * rows)


# ---------------------------------------------------------------------------
# in 64 bits
# ---------------------------------------------------------------------------

def _exact_append(s, case):
    lens, start, latent = _lens(case), _starts(case), case["latent"]
    half = ROPE // 2
    cache, t0 = s["cache"].double(), 0
    done = torch.empty(s["x"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        at = torch.arange(start[b], start[b] + n, device="cuda")
        x, y = s["x"][t0:t0 + n].double(), done[t0:t0 + n]
        c = x[:, :latent]
        y[:, :latent] = s["weight"].double() * c / torch.sqrt(c.square().mean(-1, keepdim=True) + EPS)
        cs = s["rope"].double()[at]
        for i in range(half):
            p, q = (2 * i, 2 * i + 1) if case["inter"] else (i, i + half)
            u, w = x[:, latent + p], x[:, latent + q]
            y[:, latent + p] = u * cs[:, i] - w * cs[:, half + i]
            y[:, latent + q] = w * cs[:, i] + u * cs[:, half + i]
        cache[s["table"][b].long()[at // case["page"]], at % case["page"]] = y
        t0 += n
    return (cache, done) if case["rows"] else cache


def _exact_prefill(s, case):
    q, out, q0, k0 = s["q"], [], 0, 0
    for nq, nk in zip(_lens(case), s["kv_lens"]):
        heads = torch.empty((nq, q.shape[1], case["nope"]), dtype=torch.float64, device="cuda")
        hidden = torch.ones((nq, nk), dtype=torch.bool, device="cuda").triu(nk - nq + 1)
        for h in range(q.shape[1]):
            x, k = q[q0:q0 + nq, h].double(), s["k"][k0:k0 + nk, h].double()
            logits = x[:, :case["nope"]] @ k.T
            logits += x[:, case["nope"]:] @ s["k_rope"][k0:k0 + nk].double().T
            logits /= math.sqrt(q.shape[-1])
            logits[hidden] = -math.inf
            heads[:, h] = torch.softmax(logits, -1) @ s["v"][k0:k0 + nk, h].double()
        out.append(heads)
        q0, k0 = q0 + nq, k0 + nk
    return torch.cat(out)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(s, case)
    if case["kind"] == "prefill":
        return _exact_prefill(s, case)
    latent, page, m = case["kind"] == "latent", case["page"], max(case["m"], 1)
    q = s["q"].double()
    out = torch.empty(q.shape[:-1] + (case["latent"] if latent else case["d"],),
                      dtype=torch.float64, device="cuda")
    group = case["hq"] // (1 if latent else case["hkv"])
    for b, n in enumerate(_lens(case)):
        at = torch.arange(n, device="cuda")
        sees = torch.ones((m, n), dtype=torch.bool, device="cuda")
        sees[:, n - m:] = (s["tree"][b] if s["tree"] is not None
                           else torch.ones((m, m), dtype=torch.bool, device="cuda").tril())
        if latent:
            rows = s["cache"][s["table"][b].long()[at // page], at % page].double()
            ks, vs = rows[:, None], rows[:, None, :case["latent"]]
        else:
            ks = s["k"][s["kt"][b].long()[at // page], at % page].double()
            vs = s["v"][s["vt"][b].long()[at // page], at % page].double()
        for g in range(ks.shape[1]):
            heads = slice(g * group, (g + 1) * group)
            x = q[b, heads].reshape(group, m, -1)
            logits = torch.matmul(x, ks[:, g].T) * s["scale"]
            logits = logits.masked_fill(~sees, -math.inf)
            out[b, heads] = (torch.softmax(logits, -1) @ vs[:, g]).reshape(out[b, heads].shape)
    return out
