"""lg_beam_select against log softmax and a sort in 64 bits, lg_beam_reorder against the
moves made one by one; and a beam search over pages, prompt and steps, against one that
computes every hypothesis anew."""
import math

import numpy as np
import pytest

from ligguf_amd import lib as L

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


# ---------------------------------------------------------------- selection
def choose(x, scores, top, done, end):
    """[(score, beam, token)] of a group in 64 bits, the best first."""
    out = []
    for b, row in enumerate(x.astype(np.float64)):
        s = float(scores[b])
        if not math.isfinite(s):
            continue
        if done is not None and done[b]:
            out.append((s, b, end, 0.0))
            continue
        m = row.max()
        with np.errstate(over="ignore", invalid="ignore"):
            z = m + np.log(np.exp(row - m).sum())
        if not math.isfinite(z):
            continue
        at = np.lexsort((np.arange(row.size), -row))[:top]
        out += [(s + (row[t] - z), b, int(t), row[t]) for t in at if row[t] > -np.inf]
    out.sort(key=lambda c: (-c[0], c[1], -c[3], c[2]))
    return out[:top]


def check(gpu, x, scores, top, done=None, end=7, wide=None):
    import torch
    from ligguf_amd import ops
    ng, nb, vocab = x.shape
    print(f"beam {ng} x {nb} x {vocab}, top {top}", flush=True)
    t = torch.from_numpy(x).to(gpu)
    if wide is not None:
        big = torch.full((ng, nb, wide), 1e30, device=gpu)
        big[..., 1:1 + vocab] = t
        t = big[..., 1:1 + vocab]
    d = None if done is None else torch.from_numpy(done.astype(np.int32)).to(gpu)
    r = ops.beam_select(t, torch.from_numpy(scores).to(gpu), top, done=d, end=end)
    got = [y.cpu().numpy() for y in r]
    for g in range(ng):
        want = choose(x[g], scores[g], vocab * nb if vocab * nb < 4096 else top, None if done is None else done[g], end)
        n = min(len(want), top)
        assert np.all(got[1][g, n:] == -1) and np.all(got[2][g, n:] == -1) and np.all(got[0][g, n:] == -np.inf)
        for i in range(n):
            s, b, tok, _ = want[i]
            # a beam's log sum: its terms' exponents (|x - m| U and 2 U of the exp), under 100 additions in a row
            spread = 2 * np.abs(np.where(np.isfinite(x[g, b]), x[g, b], 0)).max().astype(np.float64)
            tol = (100 + 2 * spread) * U
            mine = (float(got[0][g, i]), int(got[1][g, i]), int(got[2][g, i]))
            assert abs(mine[0] - s) <= tol + U * abs(s) + 1e-37, (mine, want[i])
            if mine[1:] != (b, tok):    # two beams' candidates nearer to each other than the log sums are known
                other = [w for w in want if w[1:3] == mine[1:]]
                assert other and other[0][1] != b and abs(other[0][0] - s) <= 2 * tol, (mine, want[max(0, i - 1):i + 2])
        assert len({(int(a), int(c)) for a, c in zip(got[1][g, :n], got[2][g, :n])}) == n
    return r


def logits(g, *shape):
    x = (g.standard_normal(shape) * 2.5).astype(np.float32)
    for row in x.reshape(-1, shape[-1]):
        row[g.integers(0, shape[-1], 5)] = g.uniform(6, 13, 5)
    return x


@pytest.mark.parametrize("ng,nb,vocab,top", [(1, 1, 1, 1), (1, 1, 1, 5), (2, 3, 2, 6), (1, 4, 5, 64), (3, 2, 31, 4), (2, 4, 257, 8),
                                             (1, 4, 1000, 8), (1, 4, 32000, 8), (7, 5, 5021, 10), (3, 8, 50257, 16), (2, 64, 300, 64),
                                             (1, 64, 9001, 64), (1, 1, 151936, 64), (40, 3, 4099, 6), (130, 8, 700, 16), (1, 33, 40961, 33)])
def test_against_64_bits(gpu, ng, nb, vocab, top):
    g = np.random.default_rng(ng * 1000 + vocab)
    x = logits(g, ng, nb, vocab)
    s = -(g.random((ng, nb)) * 8).astype(np.float32)
    check(gpu, x, s, top)
    check(gpu, x, s, top, wide=vocab + 3)
    check(gpu, x, s, top, done=g.random((ng, nb)) < 0.4)
    s[:, 1:] = -np.inf                   # the first step: one beam
    check(gpu, x, s, top)


def test_ties_go_to_the_lower_beam_and_token(gpu):
    """Equal logits within a beam, and equal beams."""
    g = np.random.default_rng(5)
    for vocab in (50, 1025, 20000):
        x = np.round(logits(g, 1, 1, vocab) * 0.5).astype(np.float32).repeat(3, 1)
        x = np.repeat(x, 2, 0)
        s = np.full((2, 3), -1.5, np.float32)
        check(gpu, x, s, 12)
        x[:] = 0.25                      # every token of every beam the same
        r = check(gpu, x, s, 12)
        assert r.parent[0].tolist() == [0] * 12 and r.token[0].tolist() == list(range(12))
        r = check(gpu, x[:, :, :5], s, 12)
        assert r.parent[0].tolist() == [0] * 5 + [1] * 5 + [2] * 2


def test_what_is_no_number(gpu):
    """Masked vocabularies, beams whose sums are no numbers, scores that are none, finished beams among them."""
    g = np.random.default_rng(6)
    for vocab in (40, 9000):
        x = logits(g, 2, 6, vocab)
        s = -(g.random((2, 6)) * 3).astype(np.float32)
        x[0, 0, 3:] = -np.inf            # three tokens allowed
        x[0, 1] = -np.inf                # none
        x[0, 2, 7] = np.nan
        x[0, 3, 9] = np.inf
        x[0, 4] = np.finfo(np.float32).min
        x[0, 4, 1] = 2.0
        s[0, 5] = np.nan
        x[1, 0] = -np.inf
        x[1, 1, 5] = 3e38
        s[1, 2] = np.inf
        s[1, 3] = -np.inf
        x[1, 4] *= 1e30
        done = np.zeros((2, 6), bool)
        check(gpu, x, s, 20)
        done[0, 1] = done[0, 3] = done[1, 3] = done[1, 5] = True     # (its logits are not read)
        check(gpu, x, s, 20, done=done)
        check(gpu, x, s, 64, done=np.ones((2, 6), bool))


def test_select_captured(gpu):
    import torch
    from ligguf_amd import ops
    g = np.random.default_rng(8)
    x = torch.from_numpy(logits(g, 3, 4, 30011)).to(gpu)
    s = torch.from_numpy(-(g.random((3, 4)) * 3).astype(np.float32)).to(gpu)
    graph, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        ops.beam_select(x, s, 8)
        st.synchronize()
        with torch.cuda.graph(graph, stream=st):
            r = ops.beam_select(x, s, 8)
    torch.cuda.synchronize()
    for _ in range(4):
        graph.replay()
        want = ops.beam_select(x, s, 8)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(r, want))
        x.copy_(x.roll(1234, 2))
        s.sub_(torch.rand_like(s))


def test_select_refusals(gpu):
    import torch
    from ligguf_amd import ops
    x, s = torch.zeros(2, 3, 8, device=gpu), torch.zeros(2, 3, device=gpu)
    for bad in (lambda: ops.beam_select(x.half(), s, 4), lambda: ops.beam_select(x[0], s, 4), lambda: ops.beam_select(x, s[:1], 4),
                lambda: ops.beam_select(x, s.double(), 4), lambda: ops.beam_select(x, s, 0), lambda: ops.beam_select(x, s, 65),
                lambda: ops.beam_select(x.transpose(1, 2), s, 4), lambda: ops.beam_select(x, s, 4, done=s),
                lambda: ops.beam_select(x, s.t().contiguous().t(), 4), lambda: ops.beam_select(x, s, 4, workspace=torch.empty(1, device=gpu))):
        with pytest.raises(L.LgError):
            bad()


# ---------------------------------------------------------------- tables
def moved(table, pools, parent, length, page, beams, n_pages):
    """The moves one by one: pools [n_pages, page, ...] lists, in place."""
    table = table.copy()
    for g, n in enumerate(length):
        if n < 0 or n > table.shape[1] * page:
            continue
        rows = slice(g * beams, (g + 1) * beams)
        old, at, r = table[rows].copy(), n // page, n % page
        par = [p if 0 <= p < beams else i for i, p in enumerate(parent[g])]
        new = old.copy()
        new[:, :at] = old[par, :at]
        if r:
            spare = [old[i, at] for i in range(beams) if i not in par]
            for i, p in enumerate(par):
                if p in par[:i]:
                    new[i, at] = spare.pop(0)
                    src, dst = old[p, at], new[i, at]
                    if 0 <= src < n_pages and 0 <= dst < n_pages:
                        for x in pools:
                            x[dst, :r] = x[src, :r]
                else:
                    new[i, at] = old[p, at]
        table[rows] = new
    return table


@pytest.mark.parametrize("ctype", [L.F16, L.KV4])
@pytest.mark.parametrize("page,kv,hd", [(16, 2, 64), (64, 1, 96), (32, 3, 128)])
@pytest.mark.parametrize("groups,beams,layers", [(1, 1, 1), (1, 4, 3), (5, 3, 2), (2, 64, 1), (3, 7, 70)])
def test_tables_and_copies(gpu, ctype, page, kv, hd, groups, beams, layers):
    import torch
    from ligguf_amd import ops
    g = np.random.default_rng(page + groups + beams)
    most = 150 if (page, layers) == (16, 3) else 5     # (entries in several rounds)
    n = groups * beams * most + 2
    print(f"reorder type {ctype}, {groups} x {beams}, {layers} layers, page {page} of {kv} x {hd}, {most} entries", flush=True)
    if layers == 70 and page > 16:
        n = groups * beams * most + 1
    table = g.permutation(n)[:groups * beams * most].reshape(groups * beams, most).astype(np.int32)
    pools, vals = [], []
    for _ in range(layers):
        pair = []
        for _ in range(2):
            if ctype == L.F16:
                pair.append(torch.randint(-30000, 30000, (n, page, kv * hd), dtype=torch.int16).to(gpu).view(torch.float16))
            else:
                # pairs (d, m) that read back differently for any two byte patterns of a code
                b = torch.randint(0, 256, (n, kv * page * hd // 32 * 20), dtype=torch.uint8)
                dm = torch.randint(0x3C00, 0x4400, (n, kv * page * hd // 16), dtype=torch.int16)
                b[:, kv * page * hd // 2:] = dm.view(torch.uint8)
                pair.append(b.to(gpu))
        pools.append(pair)
    torch.manual_seed(9)
    t = torch.full((groups * beams, most + 3), -7, dtype=torch.int32, device=gpu)
    t[:, :most] = torch.from_numpy(table).to(gpu)
    caches = [ops.PagedKvCache(*p, t[:, :most], kv, hd, ctype, page) for p in pools]
    read = lambda: [y.view(torch.int16).view(n, page, -1).cpu().numpy().copy() for c in caches  # noqa: E731
                    for y in ((c.k, c.v) if ctype == L.F16 else ops.kv_values(c.pool))]
    vals = read()
    handle = ops.PagedLayers(caches)
    for step in range(3):
        parent = g.integers(0, beams, (groups, beams)).astype(np.int32)
        # (lengths grow: pages that beams hold together are full ones)
        length = g.integers(step * most * page // 3, (step + 1) * most * page // 3 + 1, groups).astype(np.int32)
        if step == 0:
            length[:] = length // page * page + page // 2      # part-filled
        if step == 1:
            parent[0] = beams - 1                              # all from one
            parent[-1, 0] = -1                                 # from itself
            if groups > 1:
                length[1] = -1                                 # no groups
                length[0] = most * page + 1
        if step == 2:
            parent[0, -1] = beams + 5
            length[-1] = most * page                           # full
        ops.beam_reorder(handle, torch.from_numpy(parent).to(gpu), torch.from_numpy(length).to(gpu))
        table = moved(table, vals, parent.tolist(), length.tolist(), page, beams, n)
        assert np.array_equal(t[:, :most].cpu().numpy(), table) and bool((t[:, most:] == -7).all())
        for x, y in zip(read(), vals):
            assert np.array_equal(x, y)


def test_reorder_of_pages_that_are_none(gpu):
    """Entries outside the pool are moved like others, and nothing is copied from or to them."""
    import torch
    from ligguf_amd import ops
    table = torch.tensor([[0, 1], [-1, 2], [3, 99], [4, -1]], dtype=torch.int32, device=gpu)
    c = ops.PagedKvCache.empty(ops.F16, 6, 16, 1, 64, table)
    c.k.normal_()
    c.v.normal_()
    vals = [x.view(torch.int16).view(6, 16, 64).cpu().numpy().copy() for x in (c.k, c.v)]
    want = moved(table.cpu().numpy(), vals, [[2, 2, 0, 0]], [20], 16, 4, 6)
    ops.beam_reorder(ops.PagedLayers([c]), torch.tensor([[2, 2, 0, 0]], dtype=torch.int32, device=gpu),
                     torch.tensor([20], dtype=torch.int32, device=gpu))
    assert np.array_equal(table.cpu().numpy(), want)
    assert all(np.array_equal(x.view(torch.int16).view(6, 16, 64).cpu().numpy(), y) for x, y in zip((c.k, c.v), vals))


def test_reorder_captured(gpu):
    """A captured step applied again and again: in place, every replay like the eager call."""
    import torch
    from ligguf_amd import ops
    g = torch.Generator(device=gpu).manual_seed(3)
    tables = [torch.arange(24, dtype=torch.int32, device=gpu).view(6, 4) for _ in range(2)]
    sets = [[ops.PagedKvCache.empty(ops.F16, 24, 16, 2, 64, t) for _ in range(3)] for t in tables]
    for a, b in zip(*sets):
        a.k.normal_(generator=g)
        a.v.normal_(generator=g)
        b.k.copy_(a.k)
        b.v.copy_(a.v)
    parent = torch.tensor([[1, 1, 0], [2, 0, 2]], dtype=torch.int32, device=gpu)
    length = torch.tensor([21, 40], dtype=torch.int32, device=gpu)
    handles = [ops.PagedLayers(s) for s in sets]
    graph, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        for h in handles:
            ops.beam_reorder(h, parent, length)
        st.synchronize()
        with torch.cuda.graph(graph, stream=st):
            ops.beam_reorder(handles[0], parent, length)
    torch.cuda.synchronize()
    for i in range(5):
        graph.replay()
        ops.beam_reorder(handles[1], parent, length)
        torch.cuda.synchronize()
        assert torch.equal(*tables)
        for a, b in zip(*sets):
            assert torch.equal(a.k.view(torch.int16), b.k.view(torch.int16)) and torch.equal(a.v.view(torch.int16), b.v.view(torch.int16))
        parent.copy_(parent.roll(1, 1))
        length.add_(5)


def test_reorder_refusals(gpu):
    import torch
    from ligguf_amd import ops
    table = torch.zeros((4, 2), dtype=torch.int32, device=gpu)
    c = ops.PagedKvCache.empty(ops.F16, 6, 16, 1, 64, table)
    h = ops.PagedLayers([c])
    parent, length = torch.zeros((2, 2), dtype=torch.int32, device=gpu), torch.zeros(2, dtype=torch.int32, device=gpu)
    ops.beam_reorder(h, parent, length)
    for bad in (lambda: ops.beam_reorder(h, parent[:1], length[:1]), lambda: ops.beam_reorder(h, parent.long(), length),
                lambda: ops.beam_reorder(h, parent, length[:1]), lambda: ops.beam_reorder(h, parent.flatten(), length),
                lambda: ops.beam_reorder(h, parent, length.cpu()), lambda: ops.PagedLayers([c, ops.PagedKvCache.empty(ops.F16, 6, 16, 1, 64, table.clone())]),
                lambda: ops.PagedLayers([c, ops.PagedKvCache.empty(ops.KV4, 6, 16, 1, 64, table)]),
                lambda: ops.beam_reorder(ops.PagedLayers([ops.PagedKvCache.empty(ops.F16, 6, 24, 1, 64, table)]), parent, length)):
        with pytest.raises(L.LgError):
            bad()


# ---------------------------------------------------------------- a search
HEADS, KV, HD, VOCAB, LAYERS, PAGE = 4, 2, 64, 300, 2, 16


class Toy:
    """Attention layers between an embedding and an output head; G prompts with B beams over pages."""

    def __init__(self, gpu, ctype, G, B, prompts, steps):
        import torch
        from ligguf_amd import ops
        g = torch.Generator().manual_seed(4)
        w = lambda *s, k: torch.randn(*s, generator=g) * k  # noqa: E731
        self.embd = w(VOCAB, 128, k=1.0)
        self.qkv = [w(128, (HEADS + 2 * KV) * HD, k=0.12) for _ in range(LAYERS)]
        self.mix, self.out = [w(HEADS * HD, 128, k=0.15) for _ in range(LAYERS)], w(128, VOCAB, k=0.25)
        self.kw = [1 + w(HD, k=0.2) for _ in range(LAYERS)]
        self.freq = ops.rope_table(HD, 1e4)[0]
        self.dev = {n: [x.to(gpu) for x in v] if isinstance(v, list) else v.to(gpu) for n, v in vars(self).items()}
        # a prompt's full pages are its first beam's, once; all that is written later lies in pages of each beam
        most = (max(len(p) for p in prompts) + steps) // PAGE + 1
        tab, n = np.zeros((G * B, most), np.int32), 0
        for i, p in enumerate(prompts):
            full = len(p) // PAGE
            tab[i * B:(i + 1) * B, :full] = np.arange(n, n + full)
            n += full
            tab[i * B:(i + 1) * B, full:] = np.arange(n, n + B * (most - full)).reshape(B, -1)
            n += B * (most - full)
        self.table = torch.from_numpy(tab).to(gpu)
        self.caches = [ops.PagedKvCache.empty(ctype, n, PAGE, KV, HD, self.table) for _ in range(LAYERS)]
        self.layers = ops.PagedLayers(self.caches)

    def step(self, toks, pos, **share):
        """logits of rows toks [nseq, n] at pos, over the caches."""
        from ligguf_amd import ops
        d, x = self.dev, self.dev["embd"][toks.long()]
        for l, c in enumerate(self.caches):
            q, k, v = (x @ d["qkv"][l]).split([HEADS * HD, KV * HD, KV * HD], 2)
            q, _ = ops.qk_norm_rope_tokens(q, k, v, pos, d["freq"], HD, kw=d["kw"][l], cache=c)
            x = x + ops.attention_paged(q, c, pos, **share) @ d["mix"][l]
        return x @ d["out"]

    def anew(self, toks):
        """log probabilities of the token behind toks, in 64 bits over fp16 keys and values."""
        x, n = self.embd[toks].double().numpy(), len(toks)
        ang = np.arange(n)[:, None] * self.freq.double().numpy()
        c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]

        def turn(y):
            a, b = y[..., 0::2], y[..., 1::2]
            return np.stack([a * c - b * s, a * s + b * c], -1).reshape(y.shape)
        for l in range(LAYERS):
            r = (x @ self.qkv[l].double().numpy()).reshape(n, HEADS + 2 * KV, HD)
            q, k, v = r[:, :HEADS], r[:, HEADS:HEADS + KV], r[:, HEADS + KV:]
            k = k / np.sqrt((k * k).mean(-1, keepdims=True) + 1e-6) * self.kw[l].double().numpy()
            q, k = turn(q), turn(k).astype(np.float16).astype(np.float64)
            v = v.astype(np.float16).astype(np.float64)
            o = np.zeros((n, HEADS, HD))
            for h in range(HEADS):
                a = q[:, h] @ k[:, h * KV // HEADS].T / math.sqrt(HD)
                a[np.triu_indices(n, 1)] = -np.inf
                a = np.exp(a - a.max(1, keepdims=True))
                o[:, h] = a / a.sum(1, keepdims=True) @ v[:, h * KV // HEADS]
            x = x + o.reshape(n, -1) @ self.mix[l].double().numpy()
        z = x[-1] @ self.out.double().numpy()
        return z - z.max() - np.log(np.exp(z - z.max()).sum())


def search(gpu, toy, prompts, B, steps, end, share):
    """Each step's (score, parent, token), hypotheses held by the program as token lists."""
    import torch
    from ligguf_amd import ops
    G, longest = len(prompts), max(len(p) for p in prompts)
    toks = torch.zeros((G * B, longest), dtype=torch.int32)
    pos = torch.full((G * B, longest), -1, dtype=torch.int32)
    for i, p in enumerate(prompts):                      # the prompt runs once, as the first beam
        toks[i * B, :len(p)] = torch.tensor(p)
        pos[i * B, :len(p)] = torch.arange(len(p))
    out = toy.step(toks.to(gpu), pos.to(gpu))
    length = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=gpu)
    logits = torch.stack([out[i * B, len(p) - 1] for i, p in enumerate(prompts)])[:, None].repeat(1, B, 1).contiguous()
    scores = torch.full((G, B), -math.inf, device=gpu)
    scores[:, 0] = 0
    done, steps_ = torch.zeros((G, B), dtype=torch.int32, device=gpu), []
    prefix = length.clone()
    for _ in range(steps):
        r = ops.beam_select(logits, scores, B, done=done, end=end)
        steps_.append([x.cpu().numpy() for x in r])
        ops.beam_reorder(toy.layers, r.parent, length)
        scores, done = r.score, (r.token == end).int()
        p = length.repeat_interleave(B)[:, None].contiguous()
        logits = toy.step(r.token.view(G * B, 1), p, **(dict(prefix=prefix) if share else {})).view(G, B, VOCAB)
        length += 1
    return steps_


@pytest.mark.parametrize("share", [True, False])
def test_a_search_against_hypotheses_computed_anew(gpu, share):
    """Prompts of 5, 16 and 39 tokens, four beams, an end token that comes up: each chosen continuation's score
    against its hypothesis run from the beginning, and no better candidate left out."""
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, VOCAB, n).tolist() for n in (5, 16, 39)]
    B, steps = 4, 22
    toy = Toy(gpu, L.F16, len(prompts), B, prompts, steps)
    # the token that the first prompt's second step would take ends a hypothesis
    end = int(search(gpu, Toy(gpu, L.F16, len(prompts), B, prompts, steps), prompts, B, 2, -1, share)[1][2][0, 1])
    run = search(gpu, toy, prompts, B, steps, end, share)
    ended = 0
    for i, p in enumerate(prompts):
        beams = [(list(p), 0.0, False)] + [None] * (B - 1)
        for score, parent, token in run:
            cand = []
            for b, h in enumerate(beams):
                if h is None:
                    continue
                if h[2]:
                    cand.append((h[1], b, end))
                    continue
                lp = toy.anew(h[0])
                cand += [(h[1] + lp[t], b, t) for t in range(VOCAB)]
            cand.sort(key=lambda c: -c[0])
            by = {(b, t): s for s, b, t in cand}
            # fp32 rows into fp16 keys and values: a rounding that goes the other way moves a key by 2^-11 of it, a
            # score by 2^-11 sum |q k| / sqrt(hd) (under 4e-3 here), a layer's output by as much of itself; two layers
            # and the head (128 terms of 0.25) leave under 0.02 of a logit in the worst place; steps add up
            far = 0.02 * len(run)
            new = []
            for j in range(B):
                key = (int(parent[i, j]), int(token[i, j]))
                assert key in by and abs(by[key] - score[i, j]) <= far
                assert by[key] >= cand[min(j, len(cand) - 1)][0] - far
                h = beams[key[0]]
                new.append((h[0] if h[2] else h[0] + [key[1]], by[key], key[1] == end))
                ended += key[1] == end
            assert len({(int(a), int(b)) for a, b in zip(parent[i], token[i])}) == B
            beams = new
    assert ended


@pytest.mark.parametrize("ctype", [L.F16, L.KV4])
def test_shared_prompts_choose_like_copies(gpu, ctype):
    """The same search with the prompt's rows read once a group and beam by beam."""
    rng = np.random.default_rng(12)
    prompts = [rng.integers(0, VOCAB, n).tolist() for n in (33, 7)]
    runs = [search(gpu, Toy(gpu, ctype, 2, 5, prompts, 12), prompts, 5, 12, 3, share) for share in (True, False)]
    for (s0, p0, t0), (s1, p1, t1) in zip(*runs):
        assert np.array_equal(p0, p1) and np.array_equal(t0, t1)
        # sums in another order move a score by their roundings (300 of 2^-24 of an attention row, and of the values of 4
        # bits none other than those of fp16: rows already written are the same)
        assert np.max(np.abs(s0 - s1)) <= 2e-2 if ctype == L.KV4 else np.max(np.abs(s0 - s1)) <= 5e-3
