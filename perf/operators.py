"""Performance cases of the paged K/V cache: appending to it with the position rotation, and the
attention of a batch of sequences that share a prefix.

A cache is a pool of pages [n_pages, page_len, n_kv_head * d_head] for K and one for V.  A batch is
`b` sequences with `n_s` new tokens each (rows tok_off[s] .. tok_off[s+1] of q, k, v), `own_len[s]`
own tokens in the cache, the new ones among them, and a prefix of `prefix` tokens that all share.
New token i of a sequence has the own index own_len - n_s + i and stands at position prefix + index.

Each case runs in two ways: `own` false, in elementary torch operations in 32 bits; `own` true,
through `aurora_amd.gpu`.
"""
import math

import numpy as np
import torch

own = False

_CTX = None


def _ctx():
    """The program's one context (one device, one stream)."""
    global _CTX
    if _CTX is None:
        from aurora_amd.gpu import GpuContext
        _CTX = GpuContext.new(0)
    return _CTX


# ------------------------------------------------------------------ the cases


def listed():
    return [
        # one decode step of the tiny model (d 128): the smallest call, where latency counts
        {"name": "append_tiny", "op": "append", "type": "f32", "b": 4, "tok": 1, "h": 4, "kv": 4, "dh": 32,
         "prefix": 32, "own": 32, "page": 16, "rot": 32, "pairs": False},
        # one decode step of 32 sequences of the d 1024 model, 512 shared tokens, pages in bf16
        {"name": "append_step", "op": "append", "type": "bf16", "b": 32, "tok": 1, "h": 16, "kv": 16, "dh": 64,
         "prefix": 512, "own": 256, "page": 64, "rot": 64, "pairs": False},
        # prompts of up to 1024 tokens enter the cache: the largest append
        {"name": "append_prompts", "op": "append", "type": "f32", "b": 16, "tok": 1024, "h": 16, "kv": 16, "dh": 64,
         "prefix": 0, "own": 1024, "page": 64, "rot": 64, "pairs": False},
        # ragged prompts, heads of 48 columns of which 16 rotate in neighbouring pairs, shared kv heads
        {"name": "append_odd", "op": "append", "type": "bf16", "b": 7, "tok": 333, "h": 6, "kv": 3, "dh": 48,
         "prefix": 77, "own": 411, "page": 8, "rot": 16, "pairs": True},
        # the tiny model's attention in that step
        {"name": "attn_tiny", "op": "attn", "type": "f32", "b": 4, "tok": 1, "h": 4, "kv": 4, "dh": 32,
         "prefix": 32, "own": 32, "page": 16},
        # a decode step of the d 1024 model: 32 continuations of one prompt of 512 tokens
        {"name": "attn_step", "op": "attn", "type": "f32", "b": 32, "tok": 1, "h": 16, "kv": 16, "dh": 64,
         "prefix": 512, "own": 256, "page": 64},
        # 64 continuations of a long document, pages in bf16
        {"name": "attn_step_long", "op": "attn", "type": "bf16", "b": 64, "tok": 1, "h": 16, "kv": 16, "dh": 64,
         "prefix": 32768, "own": 1024, "page": 64},
        # a single sequence far into a long document: few rows, one long axis
        {"name": "attn_one", "op": "attn", "type": "f32", "b": 1, "tok": 1, "h": 16, "kv": 16, "dh": 64,
         "prefix": 16384, "own": 500, "page": 32},
        # heads that share kv heads, a prefix that ends inside a page, 48 sequences
        {"name": "attn_step_grouped", "op": "attn", "type": "f32", "b": 48, "tok": 1, "h": 16, "kv": 4, "dh": 128,
         "prefix": 4999, "own": 700, "page": 32},
        # short questions about a shared text: prompt tails of up to 128 tokens
        {"name": "attn_questions", "op": "attn", "type": "f32", "b": 16, "tok": 128, "h": 16, "kv": 16, "dh": 64,
         "prefix": 2048, "own": 160, "page": 64},
        # ragged tails of odd sizes, bf16
        {"name": "attn_odd", "op": "attn", "type": "bf16", "b": 5, "tok": 37, "h": 6, "kv": 3, "dh": 48,
         "prefix": 333, "own": 101, "page": 8},
        # long tails on a long prefix: the largest call, bound by the products
        {"name": "attn_prompts", "op": "attn", "type": "f32", "b": 16, "tok": 512, "h": 16, "kv": 16, "dh": 64,
         "prefix": 4096, "own": 512, "page": 64},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the same ranges: one token a sequence or many, sizes over their logarithm, any ending."""
    while True:
        dh = rng.choice([16, 32, 40, 48, 64, 64, 64, 96, 128])
        kv = rng.randint(1, 16)
        group = rng.choice([1, 1, 1, 2, 4, 6])
        c = {"op": rng.choice(["append", "attn", "attn"]), "type": rng.choice(["f32", "f32", "bf16"]),
             "b": _log(rng, 1, 64), "tok": 1 if rng.random() < 0.5 else _log(rng, 2, 512), "h": kv * group, "kv": kv,
             "dh": dh, "prefix": 0 if rng.random() < 0.1 else _log(rng, 1, 16384), "own": 0,
             "page": rng.choice([8, 16, 32, 64, 128])}
        c["own"] = c["tok"] + _log(rng, 1, 1024)
        if c["op"] == "append":
            c["rot"] = rng.choice([0, dh // 2 // 8 * 8, dh, dh])
            c["pairs"] = rng.random() < 0.3
        w = work(c)
        # the plain form holds padded scores and copies of them: keep those small beside the memory
        if (w["flops"] < 1.4e11 and c["b"] * c["tok"] * c["h"] * (c["prefix"] + c["own"]) < 6e8
                and w["bytes"] < 6e8 and c["h"] <= 32):
            return c


# ------------------------------------------------------------------ inputs


_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _lengths(c):
    """New tokens and own lengths of the case's sequences: the same for every seed, so that outputs
    keep their shapes."""
    rng = np.random.default_rng([c[x] for x in ("b", "tok", "own", "prefix", "h", "dh")])
    b, tok, past = c["b"], c["tok"], c["own"] - c["tok"]
    n = np.ones(b, np.int64) if tok == 1 else rng.integers((tok + 1) // 2, tok + 1, b)
    return n, n + rng.integers(past // 2, past + 1, b)


def _plan(c, seed):
    """Lengths and page tables: (tok_off [b+1], own_len [b], pages [b, m], prefix_pages, pool size)."""
    n, length = _lengths(c)
    used = -(-length // c["page"])
    first = -(-c["prefix"] // c["page"])
    total = first + int(used.sum()) + 3  # a few pages stay free
    order = np.random.default_rng(seed).permutation(total).astype(np.int32)
    pages = np.full((c["b"], -(-c["own"] // c["page"])), -1, np.int32)
    at = first
    for s in range(c["b"]):
        pages[s, :used[s]] = order[at:at + used[s]]
        at += used[s]
    off = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    return off, length.astype(np.int32), pages, order[:first].copy(), total


def _normal(g, shape, dtype=torch.float32):
    x = torch.empty(shape, device="cuda", dtype=torch.float32)
    return x.normal_(0.0, 1.0, generator=g).to(dtype)


def _tensors(c, seed):
    """The inputs' values: projections and cached rows as a LayerNorm before them leaves them, N(0, 1)."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    off, length, pages, prefix_pages, total = _plan(c, seed)
    n, row = int(off[-1]), c["kv"] * c["dh"]
    st = {"kp": _normal(g, (total, c["page"], row), _TYPES[c["type"]]),
          "vp": _normal(g, (total, c["page"], row), _TYPES[c["type"]]),
          "q": _normal(g, (n, c["h"] * c["dh"]))}
    if c["op"] == "append":
        st["k"], st["v"] = _normal(g, (n, row)), _normal(g, (n, row))
        # cos and sin of position * 10000^(-2i / rot), as the program made them once
        half = c["rot"] // 2
        f = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / max(1, half))
        a = torch.arange(c["prefix"] + c["own"], dtype=torch.float64, device="cuda")[:, None] * f
        st["table"] = torch.stack([a.cos(), a.sin()], -1).float().contiguous()
    for name, x in (("off", off), ("len", length), ("pages", pages), ("prefix_pages", prefix_pages)):
        st[name] = torch.from_numpy(x).cuda()
    return st, n


def prepare(case, seed):
    c = case
    st, n = _tensors(c, seed)
    st["case"], st["n"] = c, n
    st["out"] = torch.zeros_like(st["q"])
    if c["op"] == "attn":
        st["lse"] = torch.zeros((n, c["h"]), device="cuda")
    torch.cuda.synchronize()
    return st


# ------------------------------------------------------------------ one pass


def _rows(st):
    """Of each new token: its sequence, its number there, its own index."""
    off, t = st["off"].long(), torch.arange(st["n"], device="cuda")
    s = torch.searchsorted(off[1:].contiguous(), t, right=True)
    i = t - off[s]
    return s, i, (st["len"].long() - (off[1:] - off[:-1]))[s] + i


def _rotated(c, x, heads, table):
    """The first `rot` columns of every head by the angle of the row's position."""
    r = c["rot"]
    y = x.reshape(x.shape[0], heads, c["dh"]).clone()
    if r == 0:
        return y
    cos, sin = table[:, None, :, 0], table[:, None, :, 1]
    if c["pairs"]:
        a, b = y[..., 0:r:2].clone(), y[..., 1:r:2].clone()
        y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = y[..., :r // 2].clone(), y[..., r // 2:r].clone()
        y[..., :r // 2], y[..., r // 2:r] = a * cos - b * sin, b * cos + a * sin
    return y


def _append(st):
    c = st["case"]
    s, _, j = _rows(st)
    page, slot = st["pages"][s, j // c["page"]].long(), j % c["page"]
    table = st["table"][c["prefix"] + j]
    k = _rotated(c, st["k"], c["kv"], table).reshape(st["n"], -1)
    st["kp"][page, slot] = k.to(st["kp"].dtype)
    st["vp"][page, slot] = st["v"].to(st["vp"].dtype)
    return {"q": _rotated(c, st["q"], c["h"], table).reshape(st["n"], -1), "k": st["kp"], "v": st["vp"]}


def _attend(st):
    c = st["case"]
    b, tok, h, kv, dh, P, L = (c[x] for x in ("b", "tok", "h", "kv", "dh", "prefix", "own"))
    group = h // kv
    s, i, j = _rows(st)
    # queries padded to [b, kv, tok * group, dh]
    q = torch.zeros((b, tok, h, dh), device="cuda")
    q[s, i] = st["q"].reshape(-1, h, dh) / math.sqrt(dh)
    q = q.reshape(b, tok, kv, group, dh).permute(0, 2, 1, 3, 4).reshape(b, kv, tok * group, dh)
    last = torch.full((b, tok), -1, device="cuda", dtype=torch.long)
    last[s, i] = j
    at = torch.arange(L, device="cuda")
    page = st["pages"].long().clamp(min=0)[:, at // c["page"]]
    there = (at[None] < st["len"][:, None])[:, :, None, None]
    ko = torch.where(there, st["kp"][page, at % c["page"]].reshape(b, L, kv, dh).float(), 0.0)
    vo = torch.where(there, st["vp"][page, at % c["page"]].reshape(b, L, kv, dh).float(), 0.0)
    so = torch.matmul(q, ko.permute(0, 2, 3, 1).contiguous())
    hidden = at[None, None] > last[:, :, None]  # [b, tok, L]
    so = so.reshape(b, kv, tok, group, L).masked_fill(hidden[:, None, :, None], -math.inf)
    so = so.reshape(b, kv, tok * group, L)
    # the prefix: all rows of a kv head against one copy of it
    at = torch.arange(P, device="cuda")
    page = st["prefix_pages"].long()[at // c["page"]]
    kp = st["kp"][page, at % c["page"]].reshape(P, kv, dh).float()
    vp = st["vp"][page, at % c["page"]].reshape(P, kv, dh).float()
    rows = q.permute(1, 0, 2, 3).reshape(kv, b * tok * group, dh)
    sp = torch.matmul(rows, kp.permute(1, 2, 0).contiguous())
    sp = sp.reshape(kv, b, tok * group, P).permute(1, 0, 2, 3)
    m = so.amax(-1, keepdim=True)
    if P:
        m = torch.maximum(m, sp.amax(-1, keepdim=True))
    m = m.clamp(min=-3e38)  # a row without any key (padding) gives zeros
    eo, ep = torch.exp(so - m), torch.exp(sp - m)
    l = eo.sum(-1, keepdim=True) + ep.sum(-1, keepdim=True)
    o = torch.matmul(eo, vo.permute(0, 2, 1, 3).contiguous())
    ep = ep.permute(1, 0, 2, 3).reshape(kv, b * tok * group, P)
    o = o + torch.matmul(ep, vp.permute(1, 0, 2).contiguous()).reshape(kv, b, tok * group, dh).permute(1, 0, 2, 3)
    o = torch.where(l > 0, o / l, 0.0).reshape(b, kv, tok, group, dh).permute(0, 2, 1, 3, 4)
    lse = (m + torch.log(l)).reshape(b, kv, tok, group).permute(0, 2, 1, 3)
    return {"out": o[s, i].reshape(st["n"], h * dh), "lse": lse[s, i].reshape(st["n"], h)}


def _handles(st):
    """What the program keeps for a cache and a batch: their descriptions, and the scratch."""
    from aurora_amd.gpu import PagedBatch, PagedKvAppendKernel, PagedKvCache, PagedMhaKernel

    c = st["case"]
    cache = PagedKvCache(st["kp"].data_ptr(), st["vp"].data_ptr(), st["kp"].shape[0], c["page"], c["kv"], c["dh"],
                         c["type"])
    batch = PagedBatch(st["off"].data_ptr(), st["len"].data_ptr(), st["pages"].data_ptr(), c["b"],
                       st["pages"].shape[1], st["n"], c["tok"], c["own"], st["prefix_pages"].data_ptr(),
                       st["prefix_pages"].shape[0], c["prefix"])
    if c["op"] == "append":
        return PagedKvAppendKernel.new(), cache, batch, None
    n = PagedMhaKernel.scratch_len(cache, batch, c["h"])
    scratch = torch.empty(max(1, n), device="cuda")
    torch.cuda.synchronize()
    return PagedMhaKernel.new(), cache, batch, scratch


def run(state):
    st = state
    c = st["case"]
    if not own:
        return _append(st) if c["op"] == "append" else _attend(st)
    if "handles" not in st:
        st["handles"] = _handles(st)
    kernel, cache, batch, scratch = st["handles"]
    ld, row = c["h"] * c["dh"], c["kv"] * c["dh"]
    if c["op"] == "append":
        kernel.dispatch_into(_ctx(), cache, batch, st["q"].data_ptr(), ld, st["k"].data_ptr(), st["v"].data_ptr(), row,
                             st["out"].data_ptr(), ld, st["table"].data_ptr(), st["table"].shape[0], c["rot"], c["h"],
                             pairs=c["pairs"])
        return {"q": st["out"], "k": st["kp"], "v": st["vp"]}
    kernel.dispatch_into(_ctx(), cache, batch, st["q"].data_ptr(), ld, st["out"].data_ptr(), ld, st["lse"].data_ptr(),
                         scratch.data_ptr(), scratch.numel(), c["h"])
    return {"out": st["out"], "lse": st["lse"]}


# ------------------------------------------------------------------ work


def work(case):
    c = case
    n, length = (x.astype(float) for x in _lengths(c))
    tokens, size = float(n.sum()), 4 if c["type"] == "f32" else 2
    q, row = c["h"] * c["dh"], c["kv"] * c["dh"]
    if c["op"] == "append":
        table = min(tokens, c["prefix"] + c["own"]) * c["rot"]
        rotate = 3.0 * tokens * (c["h"] + c["kv"]) * c["rot"]
        return {"bytes": 4.0 * (tokens * (2 * q + 2 * row) + table) + size * tokens * 2.0 * row, "flops": rotate}
    keys = float((n * (c["prefix"] + length - 0.5 * (n - 1))).sum())  # over all queries
    nbytes = size * 2.0 * row * (c["prefix"] + float(length.sum())) + 4.0 * tokens * (2 * q + c["h"])
    return {"bytes": nbytes, "flops": 4.0 * q * keys}


# ------------------------------------------------------------------ the same in 64 bits


def _f64_append(c, st, n):
    q, k, v = (st[x].double().cpu().numpy() for x in ("q", "k", "v"))
    off, length, pages, page = st["off"].cpu().numpy(), st["len"].cpu().numpy(), st["pages"].cpu().numpy(), c["page"]
    seq = np.repeat(np.arange(c["b"]), np.diff(off))
    index = np.concatenate([np.arange(length[s] - (off[s + 1] - off[s]), length[s]) for s in range(c["b"])])
    half = c["rot"] // 2
    angle = (c["prefix"] + index)[:, None] * 10000.0 ** (-np.arange(half) / max(1, half))
    turn = np.exp(1j * angle)[:, None, :]

    def rotated(x, heads):
        y = x.reshape(n, heads, c["dh"]).copy()
        if half:
            re, im = (slice(0, c["rot"], 2), slice(1, c["rot"], 2)) if c["pairs"] else (slice(0, half),
                                                                                       slice(half, c["rot"]))
            z = (y[..., re] + 1j * y[..., im]) * turn
            y[..., re], y[..., im] = z.real, z.imag
        return y.reshape(n, -1)

    out = {"q": torch.from_numpy(rotated(q, c["h"]))}
    where = torch.from_numpy(pages[seq, index // page].astype(np.int64) * page + index % page).cuda()
    for name, pool, x in (("k", "kp", rotated(k, c["kv"])), ("v", "vp", v)):
        p = st[pool].double().reshape(-1, x.shape[1])
        p[where] = torch.from_numpy(x).cuda()
        out[name] = p.reshape(st[pool].shape)
    return out


def _f64_attention(c, st, n):
    off, length, pages = st["off"].tolist(), st["len"].tolist(), st["pages"].long()
    h, kv, dh, row = c["h"], c["kv"], c["dh"], c["kv"] * c["dh"]
    out = torch.zeros((n, h * dh), dtype=torch.float64, device="cuda")
    lse = torch.zeros((n, h), dtype=torch.float64, device="cuda")
    for s in range(c["b"]):
        lo, hi, L = off[s], off[s + 1], length[s]
        m = -(-L // c["page"])

        def keys(pool):  # the prefix's rows, then the sequence's, every head of q its own copy
            head = st[pool][st["prefix_pages"].long()].reshape(-1, row)[:c["prefix"]]
            x = torch.cat([head, st[pool][pages[s, :m]].reshape(-1, row)[:L]]).double().reshape(-1, kv, dh)
            return x.transpose(0, 1).repeat_interleave(h // kv, 0).contiguous()

        q = st["q"][lo:hi].double().reshape(hi - lo, h, dh).transpose(0, 1).contiguous()
        sc = torch.matmul(q, keys("kp").transpose(1, 2).contiguous()) / math.sqrt(dh)
        seen = torch.arange(c["prefix"] + L, device="cuda")[None] <= (
            c["prefix"] + L - (hi - lo) + torch.arange(hi - lo, device="cuda"))[:, None]
        sc = sc.masked_fill(~seen, -math.inf)
        out[lo:hi] = torch.matmul(torch.softmax(sc, -1), keys("vp")).transpose(0, 1).reshape(hi - lo, -1)
        lse[lo:hi] = torch.logsumexp(sc, -1).transpose(0, 1)
    return {"out": out, "lse": lse}


def exact(case, seed):
    st, n = _tensors(case, seed)
    return (_f64_append if case["op"] == "append" else _f64_attention)(case, st, n)
