"""Operators of long-context serving, beside the engine's own per-op calls.

Four of them, in the order in which a layer and an output head use them:

* ``rope``  -- queries, keys and values of many tokens: an RMS norm of each
  query and key head, the rotation of part of it (adjacent or half layout,
  frequencies scaled for long contexts), keys and values into a cache held as
  fp16 or in 4 bits.
* ``attn``  -- attention over an fp16 cache, single tokens of many sequences or
  prompts, with a sliding window and a few first positions that stay visible.
* ``attn4`` -- the same over a cache held in 4 bits.
* ``logp``  -- log probabilities of given tokens, the entropy and the top
  alternatives of rows of logits.

The cache in 4 bits: groups of 32 values of a head's row, each with a step d
and a least value m in fp16; a code n of 0..15 stands for the fp16 number
nearest n d + m.  K and V each lie as [n_kv_heads][n_ctx][head_dim / 2] bytes
of codes and behind them [n_kv_heads][n_ctx][head_dim / 32] pairs (d, m).  A
little-endian 32-bit word holds eight codes, value 2 j in bits 4 j .. 4 j + 3,
value 2 j + 1 in the same bits of the upper half.
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda"
EPS = 1e-6


# --------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------
def _rope(name, heads, kv, hd, rope, half, norm, scaling, cache, nseq, ntok, ctx):
    return {"name": name, "kind": "rope", "heads": heads, "kv": kv, "hd": hd, "rope": rope, "half": half, "norm": norm,
            "scaling": scaling, "cache": cache, "nseq": nseq, "ntok": ntok, "ctx": ctx}


def _attn(name, kind, heads, kv, hd, nseq, ntok, ctx, window, sinks, pad):
    return {"name": name, "kind": kind, "heads": heads, "kv": kv, "hd": hd, "nseq": nseq, "ntok": ntok, "ctx": ctx,
            "window": window, "sinks": sinks, "pad": pad}


def listed():
    return [
        # one token of a chat: the smallest call, an fp16 cache
        _rope("rope 1 token f16", 32, 8, 128, 128, False, True, "none", "f16", 1, 1, 512),
        # one token each of 48 conversations, part of the head rotated, into 4 bits
        _rope("rope 48 seq 4-bit", 32, 8, 128, 64, True, False, "linear", "kv4", 48, 1, 129),
        # a long prompt far beyond the trained length; keys are returned, no cache
        _rope("rope prompt 6000 yarn", 32, 8, 128, 128, True, True, "yarn", "none", 1, 6000, 131072),
        # one token after a short chat: latency
        _attn("attn 1 token 512", "attn", 32, 8, 128, 1, 1, 512, 0, 0, 0),
        # one token each of 24 conversations of ragged lengths, two slots idle, no window
        _attn("attn 24 seq 12000", "attn", 32, 8, 128, 24, 1, 12000, 0, 0, 2),
        # an unending chat's prompt chunk: window and sinks
        _attn("attn prompt 2000 win", "attn", 32, 8, 128, 1, 2000, 16000, 4096, 4, 0),
        # small heads, three ragged prompts in a padded batch
        _attn("attn 3 prompts hd64", "attn", 32, 4, 64, 3, 333, 1500, 512, 1, 70),
        # one token over a long document held in 4 bits
        _attn("attn4 1 token 32768", "attn4", 32, 8, 128, 1, 1, 32768, 0, 0, 0),
        # one token each of 40 conversations in 4 bits, with a window
        _attn("attn4 40 seq win", "attn4", 32, 8, 128, 40, 1, 20011, 8192, 16, 1),
        # a question of 700 tokens about a document held in 4 bits
        _attn("attn4 prompt 700", "attn4", 32, 8, 128, 1, 700, 9000, 0, 0, 0),
        # the sampled token of one step, with the alternatives shown to a user
        {"name": "logp 1 x 32000", "kind": "logp", "rows": 1, "vocab": 32000, "top": 5},
        # a text scored token by token
        {"name": "logp 600 x 151936", "kind": "logp", "rows": 600, "vocab": 151936, "top": 20},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "attn", "attn4", "logp"])
    if kind == "logp":
        vocab = _log(rng, 1000, 160000)
        return {"kind": kind, "rows": _log(rng, 1, min(600, 80000000 // vocab)), "vocab": vocab, "top": rng.randint(0, 20)}
    heads, kv, hd = rng.choice([(32, 8, 128), (32, 32, 128), (16, 2, 128), (32, 4, 64), (12, 12, 64), (16, 8, 256)])
    if kind == "rope":
        cache = rng.choice(["none", "f16", "kv4"])
        nseq = rng.choice([1, 1, 2, 7, 33])
        ntok = _log(rng, 1, 3000 // nseq)
        ctx = ntok + _log(rng, 1, 200) if cache != "none" else _log(rng, 8 * ntok, 400000)
        return {"kind": kind, "heads": heads, "kv": kv, "hd": hd, "rope": rng.choice([hd, hd, hd // 2, 2 * (hd // 5)]),
                "half": rng.random() < 0.5, "norm": rng.random() < 0.5, "scaling": rng.choice(["none", "linear", "yarn"]),
                "cache": cache, "nseq": nseq, "ntok": ntok, "ctx": ctx}
    if rng.random() < 0.5:      # single tokens
        nseq, ntok = _log(rng, 1, 40), 1
        ctx = _log(rng, 100, min(60000, 290000000 // (nseq * kv * hd)))
    else:
        nseq = rng.randint(1, 4)
        ntok = _log(rng, 2, 1000 // nseq)
        ctx = ntok + _log(rng, 1, 6000 // nseq)
    window = 0 if rng.random() < 0.4 else _log(rng, 16, 5000)
    pad = 0 if rng.random() < 0.5 else (min(nseq - 1, 1) if ntok == 1 else ntok // 3)
    return {"kind": kind, "heads": heads, "kv": kv, "hd": hd, "nseq": nseq, "ntok": ntok, "ctx": ctx, "window": window,
            "sinks": 0 if not window else rng.choice([0, 1, 4, 37]), "pad": pad}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _table(rope, scaling):
    """(rope / 2 frequencies as fp32, factor of cos and sin), base 1e6: as trained, every
    position divided by 4, or by parts for 4 x 32768 positions -- fast dims as
    trained, slow ones divided by 4, a ramp between those that turn 32 times
    and once over the trained length."""
    i = np.arange(rope // 2, dtype=np.float64)
    f = 1e6 ** (-2.0 * i / max(rope, 1))
    if scaling == "linear":
        return (f / 4).astype(np.float32), 1.0
    if scaling == "yarn":
        def dim(turns):
            return rope * math.log(32768 / (turns * 2 * math.pi)) / (2 * math.log(1e6))
        lo, hi = max(math.floor(dim(32)), 0), min(math.ceil(dim(1)), rope - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
        return (f * (1 - ramp) + f / 4 * ramp).astype(np.float32), float(np.float32(0.1 * math.log(4) + 1))
    return f.astype(np.float32), 1.0


def _pack(x, ctx, kv, hd):
    """fp32 [nseq, ctx, kv, hd] -> the cache in 4 bits, uint8 [nseq, bytes]."""
    g = x.permute(0, 2, 1, 3).reshape(-1, 32).double()
    m = g.amin(1, True).clamp(-60000, 60000).float().half()
    d = ((g.amax(1, True).clamp(-60000, 60000) - m.double()) / 15).float().clamp(min=0).half()
    n = torch.where(d > 0, ((g - m.double()) / d.double()).round().clamp(0, 15), torch.zeros_like(g)).to(torch.int32)
    n = n.view(-1, 4, 2)
    s = 4 * torch.arange(4, device=DEV, dtype=torch.int32).view(4, 1) + 16 * torch.arange(2, device=DEV, dtype=torch.int32)
    words = (n << s).sum((1, 2), dtype=torch.int64).to(torch.int32)     # sums of disjoint bits; the cast keeps the low 32
    nseq = x.shape[0]
    return torch.cat([words.view(nseq, -1).view(torch.uint8), torch.cat([d, m], 1).view(nseq, -1).view(torch.uint8)], 1)


def _unpack(c, ctx, kv, hd, to):
    """The values a cache in 4 bits stands for: [nseq, ctx, kv, hd]."""
    nseq, nb = c.shape[0], kv * ctx * hd // 2
    w = c[:, :nb].contiguous().view(torch.int32).view(nseq, -1, 1, 1)
    s = 4 * torch.arange(4, device=DEV, dtype=torch.int32).view(4, 1) + 16 * torch.arange(2, device=DEV, dtype=torch.int32)
    n = ((w >> s) & 15).view(nseq, kv, ctx, hd // 32, 32)
    dm = c[:, nb:].contiguous().view(torch.float16).view(nseq, kv, ctx, hd // 32, 2).double()
    v = (n.double() * dm[..., 0:1] + dm[..., 1:2]).to(torch.float16)
    return v.view(nseq, kv, ctx, hd).permute(0, 2, 1, 3).to(to)


def _positions(case, g):
    """The rows' positions, [nseq, ntok] int32; -1 where a slot or the end of a padded row holds no token."""
    nseq, ntok, ctx, pad = case["nseq"], case["ntok"], case["ctx"], case.get("pad", 0)
    if ntok == 1 and nseq > 1:      # ragged: lengths from an eighth of the longest, the first the longest
        p = torch.randint(ctx // 8, ctx, (nseq, 1), generator=g, device=DEV)
        p[0] = ctx - 1
        if pad:
            p[nseq - pad:] = -1
        return p.int()
    p = torch.arange(ctx - ntok, ctx, device=DEV).repeat(nseq, 1)
    for s in range(1, nseq):        # later prompts begin earlier and are shorter
        p[s] -= (ctx - ntok) * s // nseq
        if pad:
            p[s, ntok - pad * s // (nseq - 1):] = -1
    if pad and nseq == 1:
        p[0, ntok - pad:] = -1
    return p.int()


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    if kind == "logp":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn(rows, vocab, generator=g, device=DEV) * 2.5
        toks = torch.randint(0, vocab, (rows,), generator=g, device=DEV).int()
        # what a trained model says: one of the tokens stands out
        x.scatter_(1, torch.randint(0, vocab, (rows, 1), generator=g, device=DEV), 9.0 + 6.0 * torch.rand(rows, 1, generator=g, device=DEV))
        return {"case": case, "logits": x, "toks": toks}
    heads, kv, hd, nseq, ntok, ctx = (case[k] for k in ("heads", "kv", "hd", "nseq", "ntok", "ctx"))
    st = {"case": case, "pos": _positions(case, g)}
    if kind == "rope":
        # the output of a layer's fused q | k | v product
        st["qkv"] = torch.randn(nseq, ntok, (heads + 2 * kv) * hd, generator=g, device=DEV) * 1.5
        f, st["mscale"] = _table(case["rope"], case["scaling"])
        st["freq"] = torch.from_numpy(f).to(DEV)
        st["qw"], st["kw"] = ((1 + 0.2 * torch.randn(hd, generator=g, device=DEV)) if case["norm"] else None for _ in range(2))
        if case["cache"] == "f16":
            st["kc"], st["vc"] = (torch.zeros(nseq, ctx, kv * hd, dtype=torch.float16, device=DEV) for _ in range(2))
        elif case["cache"] == "kv4":
            st["kc"], st["vc"] = (torch.zeros(nseq, kv * ctx * hd // 32 * 20, dtype=torch.uint8, device=DEV) for _ in range(2))
        return st
    st["q"] = torch.randn(nseq, ntok, heads * hd, generator=g, device=DEV) * 1.5
    for n in ("kc", "vc"):
        if kind == "attn":
            st[n] = torch.randn(nseq, ctx, kv * hd, generator=g, device=DEV, dtype=torch.float16)
        else:
            st[n] = torch.cat([_pack(torch.randn(1, ctx, kv, hd, generator=g, device=DEV), ctx, kv, hd) for _ in range(nseq)])
    return st


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(st):
    case = st["case"]
    if own:
        return _run_own(case, st)
    if case["kind"] == "logp":
        return _plain_logp(case, st)
    if case["kind"] == "rope":
        return _plain_rope(case, st)
    return _plain_attn(case, st)


def _run_own(case, st):
    from ligguf_amd import ops
    if case["kind"] == "logp":
        r = ops.logprobs(st["logits"], st["toks"], top=case["top"])
        return (r.logprob, r.entropy) + ((r.top_id, r.top_logprob) if case["top"] else ())
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    if case["kind"] != "rope":
        cache = ops.KvCache(st["kc"], st["vc"], kv, hd, ops.F16 if case["kind"] == "attn" else ops.KV4, case["ctx"])
        return ops.attention_cache(st["q"], cache, st["pos"], window=case["window"], sinks=case["sinks"], max_pos=case["ctx"] - 1)
    q, k, v = st["qkv"].split([heads * hd, kv * hd, kv * hd], 2)
    cache = None
    if case["cache"] != "none":
        cache = ops.KvCache(st["kc"], st["vc"], kv, hd, ops.F16 if case["cache"] == "f16" else ops.KV4, case["ctx"])
    q, k = ops.qk_norm_rope_tokens(q, k, v, st["pos"], st["freq"], hd, rope_dim=case["rope"], half=case["half"], qw=st["qw"],
                                   kw=st["kw"], eps=EPS, mscale=st["mscale"], cache=cache, want_k=cache is None)
    if cache is None:
        return q, k
    if case["cache"] == "f16":
        return q, st["kc"], st["vc"]
    return (q,) + ops.kv_values(cache)


def _rotate(x, w, case, cos, sin):
    """x [nseq, ntok, heads, hd]: norm of each head, rotation of its first `rope` values."""
    r = case["rope"] // 2
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    if case["half"]:
        a, b = x[..., :r], x[..., r:2 * r]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = x[..., 0:2 * r:2], x[..., 1:2 * r:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([y, x[..., 2 * r:]], -1)


def _plain_rope(case, st):
    heads, kv, hd, nseq, ntok = (case[k] for k in ("heads", "kv", "hd", "nseq", "ntok"))
    q, k, v = (x.reshape(nseq, ntok, -1, hd) for x in st["qkv"].split([heads * hd, kv * hd, kv * hd], 2))
    ang = st["pos"].double()[:, :, None, None] * st["freq"].double()
    cos, sin = (ang.cos() * st["mscale"]).float(), (ang.sin() * st["mscale"]).float()
    q, k = _rotate(q, st["qw"], case, cos, sin).reshape(nseq, ntok, -1), _rotate(k, st["kw"], case, cos, sin)
    if case["cache"] == "none":
        return q, k.reshape(nseq, ntok, -1)
    at, pos = torch.arange(nseq, device=DEV)[:, None], st["pos"].long()
    if case["cache"] == "f16":
        st["kc"][at, pos] = k.reshape(nseq, ntok, -1).half()
        st["vc"][at, pos] = v.reshape(nseq, ntok, -1).half()
        return q, st["kc"], st["vc"]
    ctx, out = case["ctx"], [q]
    nb = kv * ctx * hd // 2
    for c, x in ((st["kc"], k), (st["vc"], v)):
        p = _pack(x, ntok, kv, hd)
        n, s = kv * ntok * hd // 2, c[:, nb:].view(nseq, kv, ctx, hd // 8)
        c[:, :nb].view(nseq, kv, ctx, hd // 2)[at, :, pos] = p[:, :n].reshape(nseq, kv, ntok, hd // 2).transpose(1, 2)
        s[at, :, pos] = p[:, n:].reshape(nseq, kv, ntok, hd // 8).transpose(1, 2)
        out.append(_unpack(c, ctx, kv, hd, torch.float16).reshape(nseq, ctx, -1))
    return tuple(out)


def _seen(pos, ctx, window, sinks):
    """[nseq, ntok, ctx]: whether the row at pos sees the key there."""
    key, p = torch.arange(ctx, device=DEV), pos[..., None]
    ok = key <= p
    return ok & ((key > p - window) | (key < sinks)) if window else ok


def _plain_attn(case, st):
    heads, kv, hd, nseq, ntok, ctx = (case[k] for k in ("heads", "kv", "hd", "nseq", "ntok", "ctx"))
    if case["kind"] == "attn":
        K, V = (st[n].view(nseq, ctx, kv, hd).float() for n in ("kc", "vc"))
    else:
        K, V = (_unpack(st[n], ctx, kv, hd, torch.float32) for n in ("kc", "vc"))
    K, V = (x.transpose(1, 2).contiguous() for x in (K, V))
    q = st["q"].view(nseq, ntok, kv, heads // kv, hd).permute(0, 2, 3, 1, 4).reshape(nseq, kv, -1, hd)
    s = torch.matmul(q, K.transpose(2, 3).contiguous()).view(nseq, kv, heads // kv, ntok, ctx) / math.sqrt(hd)
    s = s.masked_fill(~_seen(st["pos"], ctx, case["window"], case["sinks"])[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(nseq, kv, -1, ctx), V).view(nseq, kv, heads // kv, ntok, hd) / torch.where(l == 0, torch.ones_like(l), l)
    return o.permute(0, 3, 1, 2, 4).reshape(nseq, ntok, heads * hd)


def _order(x, ids):
    """Whole numbers that order (value descending, lower id first), of fp32 values and their ids."""
    b = (x + 0.0).view(torch.int32).long()
    return (torch.where(b < 0, -0x80000000 - b, b) << 32) | (0x7FFFFFFF - ids)


def _plain_logp(case, st):
    x, toks = st["logits"], st["toks"].long()
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True)
    lse = z.log()
    out = ((x.gather(1, toks[:, None]) - m - lse)[:, 0], (lse - (e * (x - m)).sum(1, keepdim=True) / z)[:, 0])
    if case["top"]:
        ids = torch.arange(x.shape[1], device=DEV)
        at = 0x7FFFFFFF - (_order(x, ids).topk(case["top"], 1).values & 0x7FFFFFFF)
        out += (at.int(), x.gather(1, at) - m - lse)
    return out


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    if case["kind"] == "logp":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + case["rows"] * (12 + 8 * case["top"]), "flops": 5 * n}
    heads, kv, hd, nseq, ntok, ctx = (case[k] for k in ("heads", "kv", "hd", "nseq", "ntok", "ctx"))
    held = {"f16": 2.0, "kv4": 0.625, "attn": 2.0, "attn4": 0.625}
    if case["kind"] == "rope":
        T = nseq * ntok
        b = 4 * T * hd * (2 * heads + 2 * kv)      # keys out, or values in for the cache
        if case["cache"] != "none":
            b += T * 2 * kv * hd * held[case["cache"]]
        return {"bytes": b + 4 * T, "flops": T * (heads + kv) * hd * 6}
    # positions as _positions() lays them out; ragged single tokens by their mean length
    w, sinks, pad = case["window"] or ctx, case["sinks"], case["pad"]
    if ntok == 1 and nseq > 1:
        n = [min(9 * ctx // 16, w + sinks)] * (nseq - pad)
        keys, pairs = sum(n), sum(n)
    else:
        keys = pairs = 0
        for s in range(nseq):
            p0 = ctx - ntok - (ctx - ntok) * s // nseq
            t = ntok - (pad * s // max(nseq - 1, 1) if nseq > 1 else pad)
            first = max(0, p0 - w + 1)
            keys += p0 + t - first + min(sinks, first) if t else 0
            pairs += sum(min(p + 1, w + min(sinks, max(0, p + 1 - w))) for p in range(p0, p0 + t))
    return {"bytes": 2 * keys * kv * hd * held[case["kind"]] + 8 * nseq * ntok * heads * hd, "flops": 4.0 * pairs * heads * hd}


# --------------------------------------------------------------------------
# the definitions, in 64 bits
# --------------------------------------------------------------------------
def _values(c, ctx, kv, hd):
    """The values one sequence's cache in 4 bits stands for, read byte by byte: float64 [kv, ctx, hd]."""
    nb = kv * ctx * hd // 2
    b = c[:nb].view(-1, 4)
    n = torch.stack([b & 15, b >> 4], 2).flatten(1)[:, [0, 4, 1, 5, 2, 6, 3, 7]].double().view(-1, 32)
    dm = c[nb:].clone().view(torch.float16).double().view(-1, 2)
    return (n * dm[:, :1] + dm[:, 1:]).half().double().view(kv, ctx, hd)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "logp":
        outs = []
        for x, t in zip(st["logits"], st["toks"]):
            y = x.double()
            y = y - torch.logsumexp(y, 0)
            p = y.exp()
            row = [y[t.long()], -(p * y).sum()]
            if case["top"]:
                v, i = torch.sort(x, descending=True, stable=True)
                row += [i[:case["top"]].int(), y[i[:case["top"]]]]
            outs.append(row)
        return tuple(torch.stack(c) for c in zip(*outs))
    heads, kv, hd, nseq, ntok, ctx = (case[k] for k in ("heads", "kv", "hd", "nseq", "ntok", "ctx"))
    if case["kind"] != "rope":
        out = torch.zeros(nseq, ntok, heads, hd, dtype=torch.float64, device=DEV)
        key = torch.arange(ctx, device=DEV)
        for s in range(nseq):
            p = st["pos"][s].long()[:, None]
            ok = (key <= p) & ((key > p - (case["window"] or ctx)) | (key < case["sinks"]))
            some = ok.any(1)
            if case["kind"] == "attn":
                K, V = (st[n][s].view(ctx, kv, hd).transpose(0, 1).double() for n in ("kc", "vc"))
            else:
                K, V = (_values(st[n][s], ctx, kv, hd) for n in ("kc", "vc"))
            for h in range(heads):
                k, v = K[h * kv // heads], V[h * kv // heads]
                q = st["q"][s].view(ntok, heads, hd)[:, h].double()
                a = (q @ k.t() / math.sqrt(hd)).masked_fill(~ok, -math.inf)
                out[s, some, h] = torch.softmax(a[some], 1) @ v
        return out.view(nseq, ntok, heads * hd)
    r, T = case["rope"] // 2, nseq * ntok
    x = st["qkv"].double().view(T, heads + 2 * kv, hd)
    ang = st["pos"].view(T, 1).double() * st["freq"].double()
    turn = torch.polar(torch.full_like(ang, st["mscale"]), ang)[:, None]
    parts = []
    for y, w in ((x[:, :heads], st["qw"]), (x[:, heads:heads + kv], st["kw"])):
        if w is not None:
            y = y / (y.square().sum(-1, keepdim=True) / hd + EPS).sqrt() * w.double()
        y = y.clone()
        if case["half"]:
            z = torch.complex(y[..., :r], y[..., r:2 * r]) * turn
            y[..., :r], y[..., r:2 * r] = z.real, z.imag
        else:
            z = torch.complex(y[..., 0:2 * r:2], y[..., 1:2 * r:2]) * turn
            y[..., 0:2 * r:2], y[..., 1:2 * r:2] = z.real, z.imag
        parts.append(y.reshape(nseq, ntok, -1))
    if case["cache"] == "none":
        return tuple(parts)
    if case["cache"] == "kv4":      # a code next to a border may go either way: no value for the cache
        return parts[0], None, None
    caches = [torch.zeros(nseq, ctx, kv * hd, dtype=torch.float64, device=DEV) for _ in range(2)]
    for s in range(nseq):
        p = st["pos"][s].long()
        caches[0][s, p] = parts[1][s]
        caches[1][s, p] = x.view(nseq, ntok, -1, hd)[s, :, heads + kv:].reshape(ntok, -1)
    return parts[0], caches[0], caches[1]
