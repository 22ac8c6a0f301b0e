"""Operators of serving several continuations of one prompt, over caches in pages.

Four of them, in the order in which a step of beam search uses them:

* ``append``  -- new tokens' queries, keys and values: an RMS norm of each
  query and key head, the rotation, keys and values into pages of a pool held
  as fp16 or in 4 bits.
* ``share``   -- attention over such pages for groups of sequences whose first
  rows are the same ones (a prompt and its beams, a document and its
  questions): single tokens or prompts, with or without a sliding window.
* ``beam``    -- the best continuations of each group: log softmax of its
  beams' logits, their scores added, the highest over beams and vocabulary.
* ``reorder`` -- the page tables of the chosen continuations, and copies of the
  part-filled pages that two of them would share, in all layers.

A pool has pages of `page` rows.  Row j of sequence s lies in row j % page of
page table[s][j // page]; entries of -1 are no pages.  A page of an fp16 pool
is [page][n_kv_heads * head_dim]; in 4 bits it is [n_kv_heads][page][head_dim
/ 2] bytes of codes and behind them [n_kv_heads][page][head_dim / 32] pairs
(d, m) of fp16: code n of a group of 32 values stands for the fp16 number
nearest n d + m; a little-endian 32-bit word holds eight codes, value 2 j in
bits 4 j .. 4 j + 3, value 2 j + 1 in the same bits of the upper half.
"""
import math

import torch

own = False
DEV = "cuda"
EPS = 1e-6


# --------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------
def _append(name, heads, kv, hd, rope, half, norm, cache, page, nseq, ntok, ctx):
    return {"name": name, "kind": "append", "heads": heads, "kv": kv, "hd": hd, "rope": rope, "half": half, "norm": norm,
            "cache": cache, "page": page, "nseq": nseq, "ntok": ntok, "ctx": ctx}


def _share(name, heads, kv, hd, cache, page, groups, members, ntok, prefix, more, window, sinks, idle):
    return {"name": name, "kind": "share", "heads": heads, "kv": kv, "hd": hd, "cache": cache, "page": page, "groups": groups,
            "members": members, "ntok": ntok, "prefix": prefix, "more": more, "window": window, "sinks": sinks, "idle": idle}


def listed():
    return [
        # one token each of four beams of a chat: latency
        _append("append 4 beams f16", 32, 8, 128, 128, False, True, "f16", 16, 4, 1, 700),
        # one token each of 12 prompts' 8 beams, part of the head rotated, into 4 bits
        _append("append 96 seq 4-bit", 32, 8, 128, 64, True, False, "kv4", 32, 96, 1, 60),
        # the prompt itself, before its beams part
        _append("append prompt 5000 f16", 32, 8, 128, 128, True, True, "f16", 64, 1, 5000, 5000),
        # four beams some way into an answer: latency
        _share("share 4 beams 700", 32, 8, 128, "f16", 16, 1, 4, 1, 700, 50, 0, 0, 0),
        # one document, 48 questions about it, each with an answer of its own length, two slots idle
        _share("share 48 of 20000", 32, 8, 128, "f16", 64, 1, 48, 1, 20000, 600, 0, 0, 2),
        # nine prompts of several lengths with six beams each, held in 4 bits
        _share("share 9 x 6 ragged 4-bit", 32, 8, 128, "kv4", 32, 9, 6, 1, 5003, 250, 0, 0, 0),
        # ten questions of up to 160 tokens behind one set of instructions, small heads
        _share("share 10 prompts hd64", 32, 4, 64, "f16", 16, 1, 10, 160, 2900, 160, 0, 0, 1),
        # the first step of a short answer, four beams
        {"name": "beam 4 x 32000", "kind": "beam", "groups": 1, "beams": 4, "vocab": 32000, "top": 8, "done": False},
        # odd rows, some beams finished
        {"name": "beam 7 x 5 x 50257", "kind": "beam", "groups": 7, "beams": 5, "vocab": 50257, "top": 10, "done": True},
        # many prompts at once, a large vocabulary
        {"name": "beam 40 x 8 x 151936", "kind": "beam", "groups": 40, "beams": 8, "vocab": 151936, "top": 16, "done": True},
        # four beams of a chat over all layers of a model
        {"name": "reorder 4 beams", "kind": "reorder", "groups": 1, "beams": 4, "layers": 36, "kv": 8, "hd": 128, "page": 16,
         "prefix": 700, "more": 60},
        # 40 prompts' beams, pages of another size
        {"name": "reorder 40 x 8", "kind": "reorder", "groups": 40, "beams": 8, "layers": 24, "kv": 8, "hd": 128, "page": 32,
         "prefix": 90, "more": 70},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["append", "share", "share", "beam", "reorder"])
    if kind == "beam":
        vocab, groups = _log(rng, 1000, 160000), _log(rng, 1, 40)
        beams = rng.randint(1, max(1, min(16, 48000000 // (vocab * groups))))
        return {"kind": kind, "groups": groups, "beams": beams, "vocab": vocab, "top": rng.randint(1, 2 * beams),
                "done": rng.random() < 0.5}
    if kind == "reorder":
        beams = rng.randint(2, 12)
        groups = _log(rng, 1, 320 // beams)
        return {"kind": kind, "groups": groups, "beams": beams, "layers": rng.randint(1, 24), "kv": rng.choice([2, 8]),
                "hd": rng.choice([64, 128]), "page": rng.choice([16, 32]), "prefix": rng.randint(0, 100), "more": rng.randint(2, 70)}
    heads, kv, hd = rng.choice([(32, 8, 128), (32, 32, 128), (16, 2, 128), (32, 4, 64), (12, 12, 64), (16, 8, 256)])
    cache, page = rng.choice(["f16", "kv4"]), rng.choice([16, 32, 64, 128])
    if kind == "append":
        nseq = rng.choice([1, 3, 16, 96])
        ntok = _log(rng, 1, 2500 // nseq)
        return {"kind": kind, "heads": heads, "kv": kv, "hd": hd, "rope": rng.choice([hd, hd, hd // 2]), "half": rng.random() < 0.5,
                "norm": rng.random() < 0.5, "cache": cache, "page": page, "nseq": nseq, "ntok": ntok, "ctx": ntok + _log(rng, 1, 200)}
    groups, members = _log(rng, 1, 12), _log(rng, 1, 48)
    members = max(1, min(members, 60 // groups))
    ntok = 1 if rng.random() < 0.6 else _log(rng, 2, max(2, 400 // (groups * members)))
    # products and rows stay below those of the largest listed cases
    most = 4000000000 // (groups * members * ntok * heads * hd)
    more = ntok + _log(rng, 1, max(1, min(3000, most // 2, 20000000 // (groups * members * kv * hd))))
    prefix = _log(rng, 1, max(1, min(20000, most - more, 150000000 // (groups * kv * hd))))
    window = 0 if rng.random() < 0.7 else _log(rng, 16, 5000)
    return {"kind": kind, "heads": heads, "kv": kv, "hd": hd, "cache": cache, "page": page, "groups": groups, "members": members,
            "ntok": ntok, "prefix": prefix, "more": more, "window": window, "sinks": 0 if not window else rng.choice([0, 1, 4, 37]),
            "idle": 0 if members == 1 else rng.choice([0, 1])}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _shifts():
    return 4 * torch.arange(4, device=DEV, dtype=torch.int32).view(4, 1) + 16 * torch.arange(2, device=DEV, dtype=torch.int32)


def _pack(x):
    """fp32 [n, kv, rows, hd] -> codes as bytes [n, kv, rows, hd / 2] and pairs as bytes [n, kv, rows, hd / 8]."""
    n, kv, rows, hd = x.shape
    g = x.reshape(-1, 32).double()
    m = g.amin(1, True).clamp(-60000, 60000).float().half()
    d = ((g.amax(1, True).clamp(-60000, 60000) - m.double()) / 15).float().clamp(min=0).half()
    c = torch.where(d > 0, ((g - m.double()) / d.double()).round().clamp(0, 15), torch.zeros_like(g)).to(torch.int32)
    words = (c.view(-1, 4, 2) << _shifts()).sum((1, 2), dtype=torch.int64).to(torch.int32)     # sums of disjoint bits
    return words.view(torch.uint8).view(n, kv, rows, hd // 2), torch.cat([d, m], 1).view(torch.uint8).view(n, kv, rows, hd // 8)


def _pages4(x):
    """fp32 [n, kv, page, hd] -> pages in 4 bits, uint8 [n, bytes]."""
    return torch.cat([p.reshape(x.shape[0], -1) for p in _pack(x)], 1)


def _values4(pool, page, kv, hd, to):
    """What pages in 4 bits stand for: [n, page, kv, hd]."""
    n, nb = pool.shape[0], kv * page * hd // 2
    w = pool[:, :nb].contiguous().view(torch.int32).view(n, -1, 1, 1)
    c = ((w >> _shifts()) & 15).view(n, kv, page, hd // 32, 32)
    dm = pool[:, nb:].contiguous().view(torch.float16).view(n, kv, page, hd // 32, 2).double()
    v = (c.double() * dm[..., 0:1] + dm[..., 1:2]).to(torch.float16)
    return v.view(n, kv, page, hd).transpose(1, 2).to(to)


def _pool(g, cache, n, page, kv, hd):
    if cache == "f16":
        return torch.randn(n, page, kv * hd, generator=g, device=DEV, dtype=torch.float16)
    return torch.cat([_pages4(torch.randn(min(64, n - i), kv, page, hd, generator=g, device=DEV)) for i in range(0, n, 64)])


def _tables(g, groups, members, shared, total, page):
    """int32 [groups * members, pages] and the number of pages: the first shared[i] // page entries of group i are the same
    pages for its members (the first of whom holds all its rows), the others theirs; -1 behind row total[i]."""
    width = max(max(total) // page + 1, 1)
    t = torch.full((groups, members, width), -1, dtype=torch.int64)
    n = 0
    for i in range(groups):
        s, e = shared[i] // page, (total[i] + page - 1) // page
        t[i, :, :s] = torch.arange(n, n + s)
        n += s
        t[i, :, s:e] = torch.arange(n, n + members * (e - s)).view(members, e - s)
        n += members * (e - s)
    p = torch.cat([torch.randperm(max(n, 1), generator=g, device=DEV), torch.full((1,), -1, device=DEV)])
    return p[t.view(groups * members, width).to(DEV)].int(), max(n, 1)


def _prefixes(case):
    """Rows that each group shares: the first group the most, the last half as many."""
    n = case["groups"]
    return [case["prefix"] - case["prefix"] * i // (2 * n) for i in range(n)]


def _lengths(case):
    """Rows of each sequence beyond the shared ones (the last ntok are this pass's): from all of `more` downwards."""
    m = case["members"]
    return [case["more"] - (case["more"] - case["ntok"]) * i // m for i in range(m)] * case["groups"]


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    if kind == "beam":
        ng, nb, vocab = case["groups"], case["beams"], case["vocab"]
        x = torch.randn(ng, nb, vocab, generator=g, device=DEV) * 2.5
        # what a trained model says: a few tokens stand out
        at = torch.randint(0, vocab, (ng, nb, 6), generator=g, device=DEV)
        x.scatter_(2, at, 8.0 + 7.0 * torch.rand(ng, nb, 6, generator=g, device=DEV))
        st = {"case": case, "logits": x, "scores": -20.0 * torch.rand(ng, nb, generator=g, device=DEV).sort(1).values}
        st["done"] = (torch.rand(ng, nb, generator=g, device=DEV) < 0.2).to(torch.int32) if case["done"] else None
        return st
    if kind == "reorder":
        ng, nb, page = case["groups"], case["beams"], case["page"]
        total = [(case["prefix"] + case["more"]) // page * page + page] * ng
        st = {"case": case}
        st["table"], n = _tables(g, ng, nb, [case["prefix"]] * ng, total, page)
        for w in ("k", "v"):
            st[w] = torch.stack([_pool(g, "f16", n, page, case["kv"], case["hd"]) for _ in range(case["layers"])])
        st["parent"] = torch.randint(0, nb, (ng, nb), generator=g, device=DEV).int()
        st["length"] = (case["prefix"] + torch.randint(1, case["more"] + 1, (ng,), generator=g, device=DEV)).int()
        return st
    heads, kv, hd, page, ntok = (case[k] for k in ("heads", "kv", "hd", "page", "ntok"))
    if kind == "append":
        nseq, ctx = case["nseq"], case["ctx"]
        st = {"case": case}
        st["table"], n = _tables(g, nseq, 1, [0] * nseq, [ctx] * nseq, page)
        first = torch.randint(0, ctx - ntok + 1, (nseq, 1), generator=g, device=DEV)
        st["pos"] = (first + torch.arange(ntok, device=DEV)).int()
        # the output of a layer's fused q | k | v product
        st["qkv"] = torch.randn(nseq, ntok, (heads + 2 * kv) * hd, generator=g, device=DEV) * 1.5
        st["freq"] = (1e6 ** (-2.0 * torch.arange(case["rope"] // 2, device=DEV, dtype=torch.float64) / case["rope"])).float()
        st["qw"], st["kw"] = ((1 + 0.2 * torch.randn(hd, generator=g, device=DEV)) if case["norm"] else None for _ in range(2))
        if case["cache"] == "f16":
            st["k"], st["v"] = (torch.zeros(n, page, kv * hd, dtype=torch.float16, device=DEV) for _ in range(2))
        else:
            st["k"], st["v"] = (torch.zeros(n, kv * page * hd // 32 * 20, dtype=torch.uint8, device=DEV) for _ in range(2))
        return st
    groups, members = case["groups"], case["members"]
    pre, more = _prefixes(case), _lengths(case)
    st = {"case": case}
    st["table"], n = _tables(g, groups, members, pre, [p + case["more"] for p in pre], page)
    st["k"], st["v"] = (_pool(g, case["cache"], n, page, kv, hd) for _ in range(2))
    st["prefix"] = torch.tensor(pre, dtype=torch.int32, device=DEV)
    first = torch.tensor([pre[s // members] + more[s] - ntok for s in range(groups * members)], device=DEV)
    pos = first[:, None] + torch.arange(ntok, device=DEV)
    if case["idle"]:        # slots without a conversation; the ends of shorter prompts in a padded batch
        if ntok == 1:
            pos[groups * members - case["idle"]:] = -1
        else:
            pos[1::2, ntok - ntok // 3:] = -1
    st["pos"] = pos.int()
    st["q"] = torch.randn(groups * members, ntok, heads * hd, generator=g, device=DEV) * 1.5
    return st


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(st):
    case = st["case"]
    if own:
        return _run_own(case, st)
    return {"append": _plain_append, "share": _plain_share, "beam": _plain_beam, "reorder": _plain_reorder}[case["kind"]](case, st)


def _run_own(case, st):
    from ligguf_amd import ops
    kind = case["kind"]
    if kind == "beam":
        r = ops.beam_select(st["logits"], st["scores"], case["top"], done=st["done"], end=2)
        return r.score, r.parent, r.token
    kv, hd, page = case["kv"], case["hd"], case["page"]
    ctype = ops.KV4 if case.get("cache") == "kv4" else ops.F16
    if "cache" not in st:       # a program has the handle of its cache as long as the cache
        if kind == "reorder":
            st["cache"] = ops.PagedLayers([ops.PagedKvCache(k, v, st["table"], kv, hd, ctype, page) for k, v in zip(st["k"], st["v"])])
        else:
            st["cache"] = ops.PagedKvCache(st["k"], st["v"], st["table"], kv, hd, ctype, page)
    cache = st["cache"]
    if kind == "reorder":
        ops.beam_reorder(cache, st["parent"], st["length"])
        return st["table"], st["k"], st["v"]
    if kind == "append":
        q, k, v = st["qkv"].split([case["heads"] * hd, kv * hd, kv * hd], 2)
        q, _ = ops.qk_norm_rope_tokens(q, k, v, st["pos"], st["freq"], hd, rope_dim=case["rope"], half=case["half"], qw=st["qw"],
                                       kw=st["kw"], eps=EPS, cache=cache)
        return (q, st["k"], st["v"]) if ctype == ops.F16 else (q,) + ops.kv_values(cache.pool)
    return ops.attention_paged(st["q"], cache, st["pos"], window=case["window"], sinks=case["sinks"],
                               max_pos=case["prefix"] + case["more"] - 1, prefix=st["prefix"], max_prefix=case["prefix"])


def _plain_append(case, st):
    heads, kv, hd, nseq, ntok, page = (case[k] for k in ("heads", "kv", "hd", "nseq", "ntok", "page"))
    q, k, v = (x.reshape(nseq, ntok, -1, hd) for x in st["qkv"].split([heads * hd, kv * hd, kv * hd], 2))
    pos, r = st["pos"].long(), case["rope"] // 2
    ang = pos.double()[:, :, None, None] * st["freq"].double()
    cos, sin = ang.cos().float(), ang.sin().float()

    def turn(x, w):
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        if case["half"]:
            a, b = x[..., :r], x[..., r:2 * r]
            y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        else:
            a, b = x[..., 0:2 * r:2], x[..., 1:2 * r:2]
            y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        return torch.cat([y, x[..., 2 * r:]], -1)
    q, k = turn(q, st["qw"]).reshape(nseq, ntok, -1), turn(k, st["kw"])
    at, row = st["table"].long().gather(1, pos // page), pos % page
    if case["cache"] == "f16":
        st["k"][at, row] = k.reshape(nseq, ntok, -1).half()
        st["v"][at, row] = v.reshape(nseq, ntok, -1).half()
        return q, st["k"], st["v"]
    nb = kv * page * hd // 2
    for pool, x in ((st["k"], k), (st["v"], v)):
        codes, pairs = _pack(x.reshape(nseq * ntok, kv, 1, hd))
        pool[:, :nb].view(-1, kv, page, hd // 2)[at.flatten(), :, row.flatten()] = codes[:, :, 0]
        pool[:, nb:].view(-1, kv, page, hd // 8)[at.flatten(), :, row.flatten()] = pairs[:, :, 0]
    return (q,) + tuple(_values4(st[w], page, kv, hd, torch.float16).reshape(-1, page, kv * hd) for w in ("k", "v"))


def _plain_share(case, st):
    """Scores of the shared rows once for a group, those of the own rows by sequence; one softmax over both."""
    heads, kv, hd, page, G, M, ntok = (case[k] for k in ("heads", "kv", "hd", "page", "groups", "members", "ntok"))
    P, S, rep, nseq, cols = case["prefix"], case["more"], heads // kv, G * M, ntok * (heads // kv)
    if case["cache"] == "f16":
        K, V = (st[w].view(-1, kv, hd) for w in ("k", "v"))
    else:
        K, V = (_values4(st[w], page, kv, hd, torch.float16).reshape(-1, kv, hd) for w in ("k", "v"))
    table, pre = st["table"].long().clamp(min=0), st["prefix"].long()
    j = torch.arange(P, device=DEV).repeat(G, 1)
    jo = (pre.repeat_interleave(M)[:, None] + torch.arange(S, device=DEV))
    at = table[::M].gather(1, j // page) * page + j % page
    ato = table.gather(1, jo // page) * page + jo % page
    KP, VP = (x[at].float().transpose(1, 2).contiguous() for x in (K, V))       # [G, kv, P, hd]
    KO, VO = (x[ato].float().transpose(1, 2).contiguous() for x in (K, V))      # [nseq, kv, S, hd]
    q = st["q"].view(nseq, ntok, kv, rep, hd).permute(0, 2, 1, 3, 4).reshape(nseq, kv, cols, hd)
    qg = q.view(G, M, kv, cols, hd).transpose(1, 2).reshape(G, kv, M * cols, hd)
    sp = torch.matmul(qg, KP.transpose(2, 3).contiguous()).view(G, kv, M, cols, P).transpose(1, 2).reshape(nseq, kv, ntok, rep, P)
    so = torch.matmul(q, KO.transpose(2, 3).contiguous()).view(nseq, kv, ntok, rep, S)
    p = st["pos"].long()[:, :, None]
    key = torch.cat([torch.where(j < pre[:, None], j, 1 << 40).repeat_interleave(M, 0), jo], 1)[:, None]
    ok = key <= p
    if case["window"]:
        ok &= (key > p - case["window"]) | (key < case["sinks"])
    s = (torch.cat([sp, so], -1) / math.sqrt(hd)).masked_fill(~ok[:, None, :, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m)).view(nseq, kv, cols, P + S)
    l = w.sum(-1, keepdim=True)
    wp = w[..., :P].reshape(G, M, kv, cols, P).transpose(1, 2).reshape(G, kv, M * cols, P)
    o = torch.matmul(wp, VP).view(G, kv, M, cols, hd).transpose(1, 2).reshape(nseq, kv, cols, hd)
    o = (o + torch.matmul(w[..., P:].contiguous(), VO)) / torch.where(l == 0, torch.ones_like(l), l)
    return o.view(nseq, kv, ntok, rep, hd).permute(0, 2, 1, 3, 4).reshape(nseq, ntok, heads * hd)


def _plain_beam(case, st):
    """In 64 bits where scores of two beams may lie next to each other."""
    ng, nb, vocab, top = (case[k] for k in ("groups", "beams", "vocab", "top"))
    x, n = st["logits"], min(case["top"], case["vocab"])
    m = x.amax(-1, keepdim=True)
    z = m.double() + torch.exp((x - m).double()).sum(-1, keepdim=True).log()
    # the best of each beam: whole numbers that order (logit descending, lower token first)
    b = (x + 0.0).view(torch.int32).long()
    order = (torch.where(b < 0, -0x80000000 - b, b) << 32) | (0x7FFFFFFF - torch.arange(vocab, device=DEV))
    tok = 0x7FFFFFFF - (order.topk(n, -1).values & 0x7FFFFFFF)
    s = st["scores"].double()[..., None] + (x.gather(-1, tok).double() - z)
    if st["done"] is not None:      # a finished beam goes on as it is, with the token that ended it
        done, first = st["done"][..., None] != 0, torch.arange(n, device=DEV) == 0
        s = torch.where(done, torch.where(first, st["scores"].double()[..., None], -math.inf), s)
        tok = torch.where(done, 2, tok)
    s, at = s.view(ng, nb * n).sort(dim=-1, descending=True, stable=True)
    s, at = s[:, :top], at[:, :top]
    some = s > -math.inf
    return s.float(), torch.where(some, at // n, -1).int(), torch.where(some, tok.view(ng, nb * n).gather(1, at), -1).int()


def _plain_reorder(case, st):
    ng, nb, page = case["groups"], case["beams"], case["page"]
    parent, length = st["parent"].long(), st["length"].long()
    old = st["table"].long().view(ng, nb, -1)
    new = old.gather(1, parent[:, :, None].expand_as(old))
    at, rows = length // page, length % page
    slot = torch.arange(nb, device=DEV)
    same = parent[:, :, None] == parent[:, None, :]
    first = ~(same & (slot[None, :] < slot[:, None])).any(-1)                   # the first child of its parent
    none = ~(parent[:, None, :] == slot[:, None]).any(-1)                       # slots without a child
    page_of = old.gather(2, at[:, None, None].expand(ng, nb, 1))[..., 0]        # the part-filled pages
    spare = page_of.gather(1, (~none).int().sort(dim=1, stable=True).indices)       # those of slots without a child first
    src = page_of.gather(1, parent)
    dst = torch.where(first, src, spare.gather(1, ((~first).cumsum(1) - 1).clamp(min=0)))
    some = (rows > 0)[:, None]
    idx = torch.arange(old.shape[2], device=DEV)
    table = torch.where(idx < at[:, None, None], new, old)
    table = torch.where((idx == at[:, None, None]) & some[..., None], dst[..., None], table)
    st["table"].copy_(table.view(ng * nb, -1))
    # every destination once: copies onto themselves where there is nothing to copy
    put = some & ~first
    src, dst = torch.where(put, src, dst).flatten(), dst.flatten()
    live = torch.arange(page, device=DEV) < rows.repeat_interleave(nb)[:, None]
    for w in ("k", "v"):
        p = st[w]
        p[:, dst] = torch.where(live[None, :, :, None], p[:, src], p[:, dst])
    return st["table"], st["k"], st["v"]


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def _seen(p, window, sinks, lo, hi):
    """How many rows of [lo, hi) position p sees."""
    hi = min(hi, p + 1)
    if not window:
        return max(0, hi - lo)
    near = max(0, hi - max(lo, p - window + 1))
    return near + max(0, min(hi, sinks, max(0, p - window + 1)) - lo)


def work(case):
    held = {"f16": 2.0, "kv4": 0.625}
    kind = case["kind"]
    if kind == "beam":
        n = case["groups"] * case["beams"] * case["vocab"] * (0.8 if case["done"] else 1.0)
        return {"bytes": 4 * n + 12 * case["groups"] * case["top"], "flops": 4 * n}
    kv, hd = case["kv"], case["hd"]
    if kind == "reorder":
        nb, page = case["beams"], case["page"]
        copies = nb - nb * (1 - (1 - 1 / nb) ** nb)     # beams less the parents that random ones leave
        rows = case["groups"] * copies * case["layers"] * (page - 1) / 2
        return {"bytes": 2 * rows * 2 * kv * hd * 2 + 8 * case["groups"] * nb * (case["prefix"] + case["more"] / 2) / page,
                "flops": 0}
    heads = case["heads"]
    if kind == "append":
        T = case["nseq"] * case["ntok"]
        return {"bytes": 4 * T * hd * (2 * heads + 2 * kv) + T * 2 * kv * hd * held[case["cache"]] + 4 * T, "flops": T * (heads + kv) * hd * 6}
    G, M, ntok, w, sinks = (case[k] for k in ("groups", "members", "ntok", "window", "sinks"))
    pre, more = _prefixes(case), _lengths(case)
    keys = pairs = 0
    for i in range(G):
        tops = []
        for s in range(i * M, (i + 1) * M):
            n = ntok
            if case["idle"] and (s >= G * M - case["idle"] if ntok == 1 else s % 2 == 1):
                n = 0 if ntok == 1 else ntok - ntok // 3
            p0 = pre[i] + more[s] - ntok
            if n:
                tops += [p0, p0 + n - 1]
                # rows that the sequence's own tokens see: all from the first one's window on
                a, b = max(pre[i], p0 - w + 1) if w else pre[i], p0 + n
                keys += b - a + max(0, min(sinks, a) - pre[i])
                pairs += sum(_seen(p, w, sinks, 0, p + 1) for p in range(p0, p0 + n))
        if tops:
            a = max(0, min(tops) - w + 1) if w else 0
            keys += max(0, pre[i] - a) + min(sinks, a, pre[i])
    return {"bytes": 2 * keys * kv * hd * held[case["cache"]] + 8 * G * M * ntok * heads * hd, "flops": 4.0 * pairs * heads * hd}


# --------------------------------------------------------------------------
# the definitions, in 64 bits
# --------------------------------------------------------------------------
def _value(pool, page, kv, hd):
    """Pages in 4 bits read byte by byte: float64 [n, page, kv, hd]."""
    n, nb = pool.shape[0], kv * page * hd // 2
    b = pool[:, :nb].reshape(-1, 4)
    c = torch.stack([b & 15, b >> 4], 2).flatten(1)[:, [0, 4, 1, 5, 2, 6, 3, 7]].double().view(-1, 32)
    dm = pool[:, nb:].contiguous().view(torch.float16).double().view(-1, 2)
    return (c * dm[:, :1] + dm[:, 1:]).half().double().view(n, kv, page, hd).transpose(1, 2)


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "beam":
        out = []
        for x, score, done in zip(st["logits"], st["scores"].double(), st["done"] if st["done"] is not None else st["scores"] * 0):
            y = torch.log_softmax(x.double(), -1) + score[:, None]
            y[done != 0] = -math.inf
            rows = [r.topk(min(case["top"], case["vocab"])).values for r in y]
            out.append(torch.cat(rows + [score[done != 0]]).sort(descending=True).values)
            out[-1] = torch.cat([out[-1], out[-1].new_full((case["top"],), -math.inf)])[:case["top"]]
        return torch.stack(out), None, None
    if kind == "reorder":       # nothing is computed, all is moved: the pages as they have to lie, slot by slot
        nb, page, k, v = case["beams"], case["page"], st["k"].double(), st["v"].double()
        for g, (parents, n) in enumerate(zip(st["parent"].tolist(), st["length"].tolist())):
            at, rows = n // page, n % page
            held = st["table"][g * nb:(g + 1) * nb, at].tolist()
            spare = [held[i] for i in range(nb) if i not in parents]
            for i, p in enumerate(parents):
                if rows and p in parents[:i]:
                    to = spare.pop(0)
                    k[:, to, :rows], v[:, to, :rows] = st["k"][:, held[p], :rows].double(), st["v"][:, held[p], :rows].double()
        return None, k, v
    heads, kv, hd, page, ntok = (case[k] for k in ("heads", "kv", "hd", "page", "ntok"))
    table = st["table"].long()
    if kind == "append":
        r, nseq = case["rope"] // 2, case["nseq"]
        x = st["qkv"].double().view(nseq, ntok, heads + 2 * kv, hd)
        ang = st["pos"].double()[:, :, None, None] * st["freq"].double()
        spin = torch.polar(torch.ones_like(ang), ang)
        parts = []
        for y, w in ((x[:, :, :heads], st["qw"]), (x[:, :, heads:heads + kv], st["kw"])):
            y = y.clone() if w is None else y / (y.square().sum(-1, keepdim=True) / hd + EPS).sqrt() * w.double()
            a, b = (slice(0, r), slice(r, 2 * r)) if case["half"] else (slice(0, 2 * r, 2), slice(1, 2 * r, 2))
            z = torch.complex(y[..., a], y[..., b]) * spin
            y[..., a], y[..., b] = z.real, z.imag
            parts.append(y.reshape(nseq, ntok, -1))
        if case["cache"] == "kv4":      # a code next to a border may go either way: no value for the pages
            return parts[0], None, None
        pools = [torch.zeros(st["k"].shape, dtype=torch.float64, device=DEV) for _ in range(2)]
        for s in range(nseq):
            p = st["pos"][s].long()
            for pool, y in zip(pools, (parts[1][s], x[s, :, heads + kv:].reshape(ntok, -1))):
                pool[table[s, p // page], p % page] = y
        return (parts[0],) + tuple(pools)
    if case["cache"] == "f16":
        K, V = (st[w].view(-1, page, kv, hd) for w in ("k", "v"))
    else:
        K, V = (_value(st[w], page, kv, hd) for w in ("k", "v"))
    M = case["members"]
    out = torch.zeros(st["pos"].shape[0], ntok, heads, hd, dtype=torch.float64, device=DEV)
    for s in range(out.shape[0]):
        p = st["pos"][s].long()[:, None]
        n, pre = int(p.max()) + 1, int(st["prefix"][s // M])
        if n <= 0:
            continue
        j = torch.arange(n, device=DEV)
        at = torch.where(j < pre, table[s - s % M, j // page], table[s, j // page])
        k, v = (x[at, j % page].double().transpose(0, 1) for x in (K, V))       # [kv, n, hd]
        ok = (j <= p) & ((j > p - (case["window"] or n)) | (j < case["sinks"]))
        some = ok.any(1)
        q = st["q"][s].double().view(ntok, kv, heads // kv, hd)[some]
        a = torch.matmul(q.permute(1, 2, 0, 3).reshape(kv, -1, hd), k.transpose(1, 2).contiguous()) / math.sqrt(hd)
        a = a.view(kv, heads // kv, -1, n).masked_fill(~ok[some], -math.inf)
        o = torch.matmul(torch.softmax(a, -1).view(kv, -1, n), v).view(kv, heads // kv, -1, hd)
        out[s, some] = o.permute(2, 0, 1, 3).reshape(-1, heads, hd)
    return out.view(out.shape[0], ntok, heads * hd)
