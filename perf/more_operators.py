"""Performance cases of serving from a paged K/V cache held in 8 bits, and of choosing the next token.

The cache: pools [n_pages, page, n_kv_head * d_head] of e4m3 numbers for K and V, and for each of them
scales [n_pages, n_kv_head, page / block] of powers of two (a byte e8m0 each), one for every `block`
tokens of a head.  A batch is `b` sequences with `n_s` new tokens each (rows tok_off[s] .. tok_off[s+1]
of q, k, v), `own_len[s]` own tokens in the cache, the new ones among them, and a prefix of `prefix`
tokens that all share.  New token i of a sequence has the own index own_len - n_s + i and stands at
position prefix + index.

  append  new k and v into the cache, k and q rotated by their positions, each block of tokens and head
          with the least scale that holds its values (a block that holds older tokens keeps its scale or
          takes a larger one, and then holds them rounded again)
  read    sequences out of the cache as dense rows in 32 bits
  attn    attention of the new tokens over prefix and own keys
  sample  the next token of each row of logits: temperature, top-k, top-p, min-p, from a random number

Each case runs in two ways: `own` false, in elementary torch operations in 32 bits (in 64 where
probabilities are summed and compared); `own` true, through `aurora_amd.gpu`.
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
        # one decode step of the tiny model (d 128) enters the cache: the smallest call, where latency counts
        {"name": "append_tiny", "op": "append", "b": 4, "tok": 1, "h": 4, "kv": 4, "dh": 32, "prefix": 32, "own": 32,
         "page": 16, "block": 16, "rot": 32, "pairs": False},
        # ragged prompts, heads of 48 columns of which 16 rotate in neighbouring pairs, shared kv heads
        {"name": "append_odd", "op": "append", "b": 7, "tok": 333, "h": 6, "kv": 3, "dh": 48, "prefix": 77, "own": 411,
         "page": 8, "block": 4, "rot": 16, "pairs": True},
        # prompts of up to 1024 tokens of the d 1024 model enter the cache: the largest append
        {"name": "append_prompts", "op": "append", "b": 16, "tok": 1024, "h": 16, "kv": 16, "dh": 64, "prefix": 0,
         "own": 1024, "page": 64, "block": 32, "rot": 64, "pairs": False},
        # 32 sequences with their prompt leave the cache (to be kept elsewhere, or for another program)
        {"name": "read_step", "op": "read", "b": 32, "h": 16, "kv": 16, "dh": 64, "prefix": 512, "own": 768,
         "page": 64, "block": 32},
        # a few short ones of odd sizes, a scale for each token
        {"name": "read_odd", "op": "read", "b": 5, "h": 6, "kv": 3, "dh": 48, "prefix": 77, "own": 411, "page": 8,
         "block": 1},
        # the tiny model's attention in a decode step
        {"name": "attn_tiny", "op": "attn", "b": 4, "tok": 1, "h": 4, "kv": 4, "dh": 32, "prefix": 32, "own": 32,
         "page": 16, "block": 16},
        # a decode step of 64 continuations of a long document
        {"name": "attn_step_long", "op": "attn", "b": 64, "tok": 1, "h": 16, "kv": 16, "dh": 64, "prefix": 32768,
         "own": 1024, "page": 64, "block": 32},
        # heads that share kv heads, a prefix that ends inside a page, 48 sequences, a scale for each token
        {"name": "attn_step_grouped", "op": "attn", "b": 48, "tok": 1, "h": 16, "kv": 4, "dh": 128, "prefix": 4999,
         "own": 700, "page": 32, "block": 1},
        # long prompt tails on a long prefix: the largest call, bound by the products
        {"name": "attn_prompts", "op": "attn", "b": 16, "tok": 512, "h": 16, "kv": 16, "dh": 64, "prefix": 4096,
         "own": 512, "page": 64, "block": 32},
        # the tiny vocabulary, four sequences: the smallest choice
        {"name": "sample_tiny", "op": "sample", "b": 4, "vocab": 256, "top_k": 0, "top_p": 0.9, "min_p": 0.0},
        # the vocabulary of the d 1024 model, 32 sequences, the usual filters
        {"name": "sample_step", "op": "sample", "b": 32, "vocab": 8192, "top_k": 50, "top_p": 0.95, "min_p": 0.0},
        # a large vocabulary without top-k: the probability mass of everything decides
        {"name": "sample_wide", "op": "sample", "b": 64, "vocab": 131072, "top_k": 0, "top_p": 0.95, "min_p": 0.01},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the same ranges: one token a sequence or many, sizes over their logarithm, any ending."""
    while True:
        op = rng.choice(["append", "append", "read", "attn", "attn", "attn", "sample", "sample"])
        if op == "sample":
            return {"op": op, "b": _log(rng, 1, 64), "vocab": _log(rng, 100, 131072),
                    "top_k": 0 if rng.random() < 0.5 else _log(rng, 1, 1000),
                    "top_p": 1.0 if rng.random() < 0.3 else round(rng.uniform(0.3, 0.999), 3),
                    "min_p": 0.0 if rng.random() < 0.6 else round(rng.uniform(0.001, 0.3), 3)}
        dh = rng.choice([16, 32, 40, 48, 64, 64, 64, 96, 128])
        kv = rng.randint(1, 16)
        page = rng.choice([8, 16, 32, 64, 128])
        c = {"op": op, "b": _log(rng, 1, 64), "tok": 1 if rng.random() < 0.5 else _log(rng, 2, 512),
             "h": kv * rng.choice([1, 1, 1, 2, 4, 6]), "kv": kv, "dh": dh,
             "prefix": 0 if rng.random() < 0.1 else _log(rng, 1, 16384), "own": 0, "page": page,
             "block": min(page, rng.choice([1, 4, 16, 32, 64]))}
        c["own"] = c["tok"] + _log(rng, 1, 1024)
        if op == "append":
            c["rot"] = rng.choice([0, dh // 2 // 8 * 8, dh, dh])
            c["pairs"] = rng.random() < 0.3
        if op == "read":
            del c["tok"]
        w = work(c)
        # the plain form holds padded scores and copies of them: keep those small beside the memory
        if (w["flops"] < 1.4e11 and c["b"] * c.get("tok", 1) * c["h"] * (c["prefix"] + c["own"]) < 6e8
                and w["bytes"] < 2e8 and c["h"] <= 32):
            return c


# ------------------------------------------------------------------ inputs


def _lengths(c):
    """New tokens and own lengths of the case's sequences: the same for every seed, so that outputs
    keep their shapes."""
    rng = np.random.default_rng([c.get(x, 0) for x in ("b", "tok", "own", "prefix", "h", "dh")])
    b, tok = c["b"], c.get("tok", 0)
    past = c["own"] - tok
    n = np.full(b, tok, np.int64) if tok <= 1 else rng.integers((tok + 1) // 2, tok + 1, b)
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


def _normal(g, shape):
    return torch.empty(shape, device="cuda", dtype=torch.float32).normal_(0.0, 1.0, generator=g)


def _exponent(amax):
    """The least e in [-117, 119] with amax <= 448 * 2^e."""
    m, x = torch.frexp(amax)
    return torch.where(amax > 0, x - torch.where(m > 0.875, 8, 9), -117).clamp(-117, 119)


def _pool(g, c, total):
    """Pages as earlier appends left them: N(0, 1) as a LayerNorm before the projections gives them."""
    x = _normal(g, (total, c["page"] // c["block"], c["block"], c["kv"], c["dh"]))
    e = _exponent(x.abs().amax((2, 4)))  # [page, block of it, head]
    x = torch.ldexp(x, -e[:, :, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    scale = (e + 127).to(torch.uint8).transpose(1, 2).contiguous()
    return x.reshape(total, c["page"], c["kv"] * c["dh"]).contiguous(), scale


def _tensors(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if c["op"] == "sample":
        b = c["b"]
        rng = np.random.default_rng(seed)
        # a few likely tokens over a broad rest, every request with a temperature of its own
        st = {"logits": 2.5 * _normal(g, (b, c["vocab"]))}
        for name, x in (("u", rng.random(b)), ("temperature", rng.uniform(0.6, 1.2, b)),
                        ("top_p", np.full(b, c["top_p"])), ("min_p", np.full(b, c["min_p"]))):
            st[name] = torch.from_numpy(x.astype(np.float32)).cuda().clamp(max=1.0 - 2.0**-24 if name == "u" else 2.0)
        st["top_k"] = torch.full((b,), c["top_k"], dtype=torch.int32, device="cuda")
        return st, b
    off, length, pages, prefix_pages, total = _plan(c, seed)
    n, row = int(off[-1]), c["kv"] * c["dh"]
    st = {}
    st["kp"], st["ks"] = _pool(g, c, total)
    st["vp"], st["vs"] = _pool(g, c, total)
    if c["op"] != "read":
        st["q"] = _normal(g, (n, c["h"] * c["dh"]))
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
    if c["op"] == "sample":
        st["tokens"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        st["logprob"] = torch.zeros(n, device="cuda")
    elif c["op"] == "read":
        shape = (c["b"], c["prefix"] + c["own"], c["kv"] * c["dh"])
        st["k_out"], st["v_out"] = torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda")
    else:
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


def _values(c, pool, scale, page, slot):
    """The cache's rows (page, slot) in 32 bits, [..., kv, dh]."""
    x = pool[page, slot].view(torch.float8_e4m3fn).float().unflatten(-1, (c["kv"], c["dh"]))
    e = scale[page, :, slot // c["block"]].int() - 127
    return torch.ldexp(x, e[..., None])


def _quantised(st, pool, scale, x):
    """Rows x [n, kv, dh] into the blocks of their tokens: [sequence, touched block, row of it]."""
    c = st["case"]
    S, kv, dh = c["block"], c["kv"], c["dh"]
    off, length = st["off"].long(), st["len"].long()
    past = length - (off[1:] - off[:-1])  # own tokens before the new ones
    touched = torch.arange((c["tok"] + S - 2) // S + 1, device="cuda")
    block = torch.minimum(past[:, None] // S + touched, (length[:, None] - 1) // S)
    # rows behind the sequence's last stand for that one again
    j = torch.minimum(block[..., None] * S + torch.arange(S, device="cuda"), (length - 1)[:, None, None])
    new = j >= past[:, None, None]
    page = st["pages"].long()[torch.arange(c["b"], device="cuda")[:, None, None], j // c["page"]]
    slot = j % c["page"]
    fresh = x[(off[:-1, None, None] + j - past[:, None, None]).clamp(min=0)]
    amax = torch.where(new[..., None, None] & fresh.isfinite(), fresh.abs(), 0.0).amax((2, 4))  # [b, touched, kv]
    held = scale[page[:, :, 0], :, slot[:, :, 0] // S].int() - 127
    e = _exponent(amax)
    e = torch.where(new[:, :, :1], e, torch.maximum(e, held))
    value = torch.where(new[..., None, None], fresh, _values(c, pool, scale, page, slot))
    y = torch.ldexp(value, -e[:, :, None, :, None])
    y = torch.where(y.isfinite(), y.clamp(-448.0, 448.0), math.nan).to(torch.float8_e4m3fn).view(torch.uint8)
    pool[page, slot] = y.reshape(*j.shape, kv * dh)
    scale[page[:, :, 0], :, slot[:, :, 0] // S] = (e + 127).to(torch.uint8)


def _append(st):
    c = st["case"]
    _, _, j = _rows(st)
    table = st["table"][c["prefix"] + j]
    _quantised(st, st["kp"], st["ks"], _rotated(c, st["k"], c["kv"], table))
    _quantised(st, st["vp"], st["vs"], st["v"].reshape(st["n"], c["kv"], c["dh"]))
    return _cache(st, _rotated(c, st["q"], c["h"], table).reshape(st["n"], -1))


def _cache(st, q):
    """The rotated queries and the whole cache: its elements and its scales as the numbers that they are."""
    e4m3, e8m0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    return {"q": q, "k": st["kp"].view(e4m3), "v": st["vp"].view(e4m3), "k_scale": st["ks"].view(e8m0),
            "v_scale": st["vs"].view(e8m0)}


def _read(st):
    c = st["case"]
    P, x = c["prefix"], torch.arange(c["prefix"] + c["own"], device="cuda")
    own_index = (x - P).clamp(min=0)
    page = st["pages"].long().clamp(min=0)[:, own_index // c["page"]]
    slot = own_index % c["page"]
    if P:
        at = x.clamp(max=P - 1)
        page = torch.where(x < P, st["prefix_pages"].long()[at // c["page"]], page)
        slot = torch.where(x < P, at % c["page"], slot)
    there = (x < P + st["len"].long()[:, None])[..., None, None]
    slot = slot.expand_as(page)
    k = torch.where(there, _values(c, st["kp"], st["ks"], page, slot), 0.0)
    v = torch.where(there, _values(c, st["vp"], st["vs"], page, slot), 0.0)
    return {"k": k.flatten(2), "v": v.flatten(2)}


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
    slot = (at % c["page"]).expand_as(page)
    there = (at[None] < st["len"][:, None])[:, :, None, None]
    ko = torch.where(there, _values(c, st["kp"], st["ks"], page, slot), 0.0)
    vo = torch.where(there, _values(c, st["vp"], st["vs"], page, slot), 0.0)
    so = torch.matmul(q, ko.permute(0, 2, 3, 1).contiguous())
    hidden = at[None, None] > last[:, :, None]  # [b, tok, L]
    so = so.reshape(b, kv, tok, group, L).masked_fill(hidden[:, None, :, None], -math.inf)
    so = so.reshape(b, kv, tok * group, L)
    # the prefix: all rows of a kv head against one copy of it
    at = torch.arange(P, device="cuda")
    page, slot = st["prefix_pages"].long()[at // c["page"]], at % c["page"]
    kp, vp = _values(c, st["kp"], st["ks"], page, slot), _values(c, st["vp"], st["vs"], page, slot)
    rows = q.permute(1, 0, 2, 3).reshape(kv, b * tok * group, dh)
    sp = torch.matmul(rows, kp.permute(1, 2, 0).contiguous())
    sp = sp.reshape(kv, b, tok * group, P).permute(1, 0, 2, 3)
    m = so.amax(-1, keepdim=True)
    if P:
        m = torch.maximum(m, sp.amax(-1, keepdim=True))
    m = m.clamp(min=-3e38)  # a row without any key (padding) gives zeros
    eo, ep = torch.exp(so - m), torch.exp(sp - m)
    total = eo.sum(-1, keepdim=True) + ep.sum(-1, keepdim=True)
    o = torch.matmul(eo, vo.permute(0, 2, 1, 3).contiguous())
    ep = ep.permute(1, 0, 2, 3).reshape(kv, b * tok * group, P)
    o = o + torch.matmul(ep, vp.permute(1, 0, 2).contiguous()).reshape(kv, b, tok * group, dh).permute(1, 0, 2, 3)
    o = torch.where(total > 0, o / total, 0.0).reshape(b, kv, tok, group, dh).permute(0, 2, 1, 3, 4)
    lse = (m + torch.log(total)).reshape(b, kv, tok, group).permute(0, 2, 1, 3)
    return {"out": o[s, i].reshape(st["n"], h * dh), "lse": lse[s, i].reshape(st["n"], h)}


def _sample(st):
    logits, V = st["logits"], st["case"]["vocab"]
    x = logits.double()
    x = (x - x.amax(-1, keepdim=True)) / st["temperature"].double()[:, None]
    w = torch.exp(x)
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices  # equal ones: the lower index first
    ranked = w.gather(-1, order)
    rank = torch.arange(V, device="cuda")
    k = torch.where(st["top_k"] > 0, st["top_k"], V)[:, None]
    ranked = torch.where(rank < k, ranked, 0.0)
    before = torch.cumsum(ranked, -1) - ranked
    keep = (rank < k) & (ranked >= st["min_p"].double()[:, None])
    keep &= (before < st["top_p"].double()[:, None] * ranked.sum(-1, keepdim=True)) | (st["top_p"] >= 1)[:, None]
    keep[:, 0] = True
    kept = torch.where(torch.zeros_like(keep).scatter(-1, order, keep), w, 0.0)
    cdf = torch.cumsum(kept, -1)
    total = cdf[:, -1:].contiguous()
    token = torch.searchsorted(cdf, st["u"].double()[:, None] * total, right=True).clamp(max=V - 1)
    logprob = x.gather(-1, token) - torch.log(total)
    return {"tokens": token[:, 0].int(), "logprob": logprob[:, 0].float()}


_PLAIN = {"append": _append, "read": _read, "attn": _attend, "sample": _sample}


def _handles(st):
    """What the program keeps for a cache and a batch: their descriptions, and the scratch."""
    from aurora_amd.gpu import (PagedBatch, PagedKvAppendKernel, PagedKvCache, PagedKvReadKernel, PagedMhaKernel,
                                SampleKernel)

    c = st["case"]
    if c["op"] == "sample":
        return SampleKernel.new(), None, None, None
    cache = PagedKvCache(st["kp"].data_ptr(), st["vp"].data_ptr(), st["kp"].shape[0], c["page"], c["kv"], c["dh"],
                         "e4m3", k_scale=st["ks"].data_ptr(), v_scale=st["vs"].data_ptr(), scale_len=c["block"])
    batch = PagedBatch(st["off"].data_ptr(), st["len"].data_ptr(), st["pages"].data_ptr(), c["b"],
                       st["pages"].shape[1], st["n"], c.get("tok", 0), c["own"], st["prefix_pages"].data_ptr(),
                       st["prefix_pages"].shape[0], c["prefix"])
    if c["op"] == "append":
        return PagedKvAppendKernel.new(), cache, batch, None
    if c["op"] == "read":
        return PagedKvReadKernel.new(), cache, batch, None
    n = PagedMhaKernel.scratch_len(cache, batch, c["h"])
    scratch = torch.empty(max(1, n), device="cuda")
    torch.cuda.synchronize()
    return PagedMhaKernel.new(), cache, batch, scratch


def run(state):
    st = state
    c = st["case"]
    if not own:
        return _PLAIN[c["op"]](st)
    if "handles" not in st:
        st["handles"] = _handles(st)
    kernel, cache, batch, scratch = st["handles"]
    if c["op"] == "sample":
        kernel.dispatch_into(_ctx(), st["logits"].data_ptr(), c["vocab"], st["u"].data_ptr(), st["tokens"].data_ptr(),
                             st["logprob"].data_ptr(), c["b"], c["vocab"], st["temperature"].data_ptr(),
                             st["top_k"].data_ptr(), st["top_p"].data_ptr(), st["min_p"].data_ptr())
        return {"tokens": st["tokens"], "logprob": st["logprob"]}
    ld, row = c["h"] * c["dh"], c["kv"] * c["dh"]
    if c["op"] == "append":
        kernel.dispatch_into(_ctx(), cache, batch, st["q"].data_ptr(), ld, st["k"].data_ptr(), st["v"].data_ptr(), row,
                             st["out"].data_ptr(), ld, st["table"].data_ptr(), st["table"].shape[0], c["rot"], c["h"],
                             pairs=c["pairs"])
        return _cache(st, st["out"])
    if c["op"] == "read":
        kernel.dispatch_into(_ctx(), cache, batch, st["k_out"].data_ptr(), st["v_out"].data_ptr(), row, 0,
                             c["prefix"] + c["own"])
        return {"k": st["k_out"], "v": st["v_out"]}
    kernel.dispatch_into(_ctx(), cache, batch, st["q"].data_ptr(), ld, st["out"].data_ptr(), ld, st["lse"].data_ptr(),
                         scratch.data_ptr(), scratch.numel(), c["h"])
    return {"out": st["out"], "lse": st["lse"]}


# ------------------------------------------------------------------ work


def work(case):
    c = case
    if c["op"] == "sample":
        n = float(c["b"]) * c["vocab"]
        return {"bytes": 4.0 * n, "flops": 3.0 * n}  # a difference, an exponential and a sum
    n, length = (x.astype(float) for x in _lengths(c))
    tokens, q, row = float(n.sum()), c["h"] * c["dh"], c["kv"] * c["dh"]
    held = row + c["kv"] / c["block"]  # bytes of a token's K or V and its share of the scales
    axis = c["prefix"] + float(length.sum())
    if c["op"] == "append":
        table = min(tokens, c["prefix"] + c["own"]) * c["rot"]
        rotate = 3.0 * tokens * (c["h"] + c["kv"]) * c["rot"]
        return {"bytes": 4.0 * (tokens * (2 * q + 2 * row) + table) + 2.0 * tokens * held,
                "flops": rotate + 2.0 * tokens * 2 * row}
    if c["op"] == "read":
        rows = float(c["b"] * (c["prefix"] + c["own"]))
        return {"bytes": 2.0 * held * axis + 8.0 * rows * row, "flops": 2.0 * rows * row}
    keys = float((n * (c["prefix"] + length - 0.5 * (n - 1))).sum())  # over all queries
    return {"bytes": 2.0 * held * axis + 4.0 * tokens * (2 * q + c["h"]), "flops": 4.0 * q * keys}


# ------------------------------------------------------------------ the same in 64 bits


def _f64_number(byte):
    """What the bytes of e4m3 numbers stand for: sign, 4 bits of exponent, 3 of significand; 127 is NaN."""
    e, m = (byte >> 3) & 15, byte & 7
    x = np.where(e > 0, (8 + m) * 2.0**(e - 10.0), m * 2.0**-9)
    return np.where(byte & 127 == 127, np.nan, np.where(byte & 128, -x, x))


_F64_NUMBERS = _f64_number(np.arange(256))


def _f64_round(x):
    """The nearest e4m3 number, ties to even."""
    size = np.abs(x)
    step = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(size, 1e-300))), -6) - 3)
    return np.clip(np.rint(x / step) * step, -448, 448)


def _f64_append(c, st, n):
    off, length, pages = (st[x].cpu().numpy() for x in ("off", "len", "pages"))
    page, S, kv, dh = c["page"], c["block"], c["kv"], c["dh"]
    index = np.concatenate([np.arange(length[s] - (off[s + 1] - off[s]), length[s]) for s in range(c["b"])])
    half = c["rot"] // 2
    angle = (c["prefix"] + index)[:, None] * 10000.0 ** (-np.arange(half) / max(1, half))
    turn = np.exp(1j * angle)[:, None, :]

    def rotated(x, heads):
        y = x.double().cpu().numpy().reshape(n, heads, dh).copy()
        if half:
            re, im = (slice(0, c["rot"], 2), slice(1, c["rot"], 2)) if c["pairs"] else (slice(0, half),
                                                                                       slice(half, c["rot"]))
            z = (y[..., re] + 1j * y[..., im]) * turn
            y[..., re], y[..., im] = z.real, z.imag
        return y

    out = {"q": torch.from_numpy(rotated(st["q"], c["h"]).reshape(n, -1))}
    for name, pool, scale, x in (("k", "kp", "ks", rotated(st["k"], kv)),
                                 ("v", "vp", "vs", st["v"].double().cpu().numpy().reshape(n, kv, dh))):
        number = _F64_NUMBERS[st[pool].cpu().numpy()].reshape(-1, page, kv, dh)
        power = st[scale].cpu().numpy().astype(np.int64) - 127
        for s in range(c["b"]):
            past = int(length[s] - (off[s + 1] - off[s]))
            for lo in range(past // S * S, int(length[s]), S):
                hi, p, at = min(lo + S, int(length[s])), pages[s, lo // page], lo % page
                new = x[off[s] + max(lo, past) - past:off[s] + hi - past]
                top = np.abs(new).max((0, 2))
                e = np.clip(np.ceil(np.log2(np.maximum(top, 1e-300) / 448.0)), -117, 119).astype(np.int64)
                old = number[p, at:at + max(past - lo, 0)] * 2.0 ** power[p, :, at // S][:, None]
                if past > lo:
                    e = np.maximum(e, power[p, :, at // S])
                both = np.concatenate([old, new]) * 2.0 ** -e.astype(float)[:, None]
                number[p, at:at + hi - lo] = _f64_round(both)
                power[p, :, at // S] = e
        out[name] = torch.from_numpy(number.reshape(st[pool].shape))
        out[name + "_scale"] = torch.from_numpy(2.0 ** power.astype(float))
    return out


def _f64_keys(c, st, s, pool, scale):
    """The keys (or values) of sequence s, prefix first, [keys, kv, dh]."""
    numbers = torch.from_numpy(_F64_NUMBERS).cuda()
    m = -(-int(st["len"][s]) // c["page"])
    got = []
    for pages, n in ((st["prefix_pages"].long(), c["prefix"]), (st["pages"].long()[s, :m], int(st["len"][s]))):
        x = numbers[st[pool][pages].int()].reshape(-1, c["page"], c["kv"], c["dh"])
        e = 2.0 ** (st[scale][pages].double() - 127.0)
        e = e.repeat_interleave(c["block"], 2).transpose(1, 2)
        got.append((x * e[..., None]).reshape(-1, c["kv"], c["dh"])[:n])
    return torch.cat(got)


def _f64_read(c, st, n):
    out = {}
    for name, pool, scale in (("k", "kp", "ks"), ("v", "vp", "vs")):
        x = torch.zeros((c["b"], c["prefix"] + c["own"], c["kv"] * c["dh"]), dtype=torch.float64, device="cuda")
        for s in range(c["b"]):
            rows = _f64_keys(c, st, s, pool, scale)
            x[s, :len(rows)] = rows.flatten(1)
        out[name] = x
    return out


def _f64_attention(c, st, n):
    off = st["off"].tolist()
    h, kv, dh = c["h"], c["kv"], c["dh"]
    out = torch.zeros((n, h * dh), dtype=torch.float64, device="cuda")
    lse = torch.zeros((n, h), dtype=torch.float64, device="cuda")
    for s in range(c["b"]):
        lo, hi = off[s], off[s + 1]
        k, v = (_f64_keys(c, st, s, *x).transpose(0, 1).repeat_interleave(h // kv, 0).contiguous()
                for x in (("kp", "ks"), ("vp", "vs")))
        q = st["q"][lo:hi].double().reshape(hi - lo, h, dh).transpose(0, 1).contiguous()
        sc = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(dh)
        seen = torch.arange(k.shape[1], device="cuda")[None] <= (
            k.shape[1] - (hi - lo) + torch.arange(hi - lo, device="cuda"))[:, None]
        sc = sc.masked_fill(~seen, -math.inf)
        out[lo:hi] = torch.matmul(torch.softmax(sc, -1), v).transpose(0, 1).reshape(hi - lo, -1)
        lse[lo:hi] = torch.logsumexp(sc, -1).transpose(0, 1)
    return {"out": out, "lse": lse}


def _f64_sample(c, st, b):
    x, u, t, p, m = (st[n].double().cpu().numpy() for n in ("logits", "u", "temperature", "top_p", "min_p"))
    tokens, logprob = np.zeros(b, np.int32), np.zeros(b)
    for r in range(b):
        w = np.exp((x[r] - x[r].max()) / t[r])
        order = np.argsort(-x[r], kind="stable")[:c["top_k"] or None]
        mass = np.cumsum(w[order])
        if p[r] < 1:
            order = order[:1 + int(np.searchsorted(mass, p[r] * mass[-1]))]
        order = np.sort(order[(w[order] >= m[r]) | (np.arange(len(order)) == 0)])
        mass = np.cumsum(w[order])
        tokens[r] = order[min(int(np.searchsorted(mass, u[r] * mass[-1], side="right")), len(order) - 1)]
        logprob[r] = np.log(w[tokens[r]] / mass[-1])
    return {"tokens": torch.from_numpy(tokens), "logprob": torch.from_numpy(logprob)}


_F64 = {"append": _f64_append, "read": _f64_read, "attn": _f64_attention, "sample": _f64_sample}


def exact(case, seed):
    st, n = _tensors(case, seed)
    return _F64[case["op"]](case, st, n)
