"""The calls over pages: lg_qk_norm_rope_paged against the contiguous call, bit for bit,
and lg_attn_paged against softmax(q K^T / sqrt(hd)) V in 64 bits -- pages of every
size, groups that share rows, missing pages, garbage where nothing is seen,
windows and sinks, single tokens and prompts, captured calls, other streams."""
import numpy as np
import pytest

from ligguf_amd import lib as L
from test_gpu_cattn import kv4_bytes

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [L.F16, L.KV4]


# ---------------------------------------------------------------- append
@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("heads,kv,hd,rope,half,norm,page", [(4, 2, 64, 64, False, True, 16), (8, 2, 128, 64, True, False, 32),
                                                            (3, 1, 96, 96, True, True, 128), (2, 2, 256, 100, False, True, 16)])
def test_append_equals_the_contiguous_call(gpu, ctype, heads, kv, hd, rope, half, norm, page):
    """The same rows at the same positions; what no row writes keeps its bytes."""
    import torch
    from ligguf_amd import ops
    for nseq, T in ((1, 1), (3, 40), (2, 530)):
        print(f"append type {ctype} {heads}/{kv} of {hd}, page {page}, {nseq} x {T}", flush=True)
        g = np.random.default_rng(7)
        most = (2 * T + page - 1) // page + 1
        n_ctx = most * page
        pos = np.stack([g.permutation(n_ctx + 9)[:T] for _ in range(nseq)]).astype(np.int32)     # a few behind the end
        if T > 1:
            pos[-1, T // 2:] = -1
        pages = g.permutation(nseq * most + 3)[:nseq * most].reshape(nseq, most).astype(np.int32)
        pages[0, -1] = -1                                                                        # and some without a page
        if nseq > 1:
            pages[1, 0] = nseq * most + 3
        table = torch.from_numpy(pages).to(gpu)
        t = torch.from_numpy(g.standard_normal((nseq, T, (heads + 2 * kv) * hd)).astype(np.float32)).to(gpu)
        q, k, v = t.split([heads * hd, kv * hd, kv * hd], 2)
        freq = torch.from_numpy((1e4 ** (-2.0 * np.arange(rope // 2) / rope)).astype(np.float32)).to(gpu)
        qw, kw = (torch.from_numpy((1 + 0.3 * g.standard_normal(hd)).astype(np.float32)).to(gpu) if norm else None for _ in range(2))
        flat = ops.KvCache.empty(ctype, n_ctx, kv, hd, nseq, gpu)
        paged = ops.PagedKvCache.empty(ctype, nseq * most + 3, page, kv, hd, table)
        for b in (flat.k, flat.v, paged.k, paged.v):
            b.view(torch.uint8).fill_(0x35)
        kw_ = dict(rope_dim=rope, half=half, qw=qw, kw=kw, mscale=1.25, want_k=True)
        p = torch.from_numpy(pos).to(gpu)
        a = ops.qk_norm_rope_tokens(q, k, v, p, freq, hd, cache=flat, **kw_)
        b = ops.qk_norm_rope_tokens(q, k, v, p, freq, hd, cache=paged, **kw_)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        both = []
        for c in (flat, paged.pool):
            both.append([x.view(-1, c.n_ctx, kv, hd) for x in ((c.k.view(torch.int16), c.v.view(torch.int16)) if ctype == L.F16 else
                                                               [y.view(torch.int16) for y in ops.kv_values(c)])])
        blank = both[1][0].new_full((1, page, kv, hd), 0x3535) if ctype == L.F16 else None
        held = torch.zeros(nseq * most + 3, dtype=torch.bool)
        for s in range(nseq):
            for j in range(most):
                i = int(pages[s, j])
                if not 0 <= i < nseq * most + 3:
                    continue
                held[i] = True
                for x, y in zip(*both):
                    assert torch.equal(x[s, j * page:(j + 1) * page], y[i])
        if blank is not None:
            for y in both[1]:
                assert torch.equal(y[~held.to(gpu)], blank.expand(int((~held).sum()), -1, -1, -1))


# ---------------------------------------------------------------- attention
class Pages:
    """A pool whose unseen rows are NaN or infinities, tables, and what each sequence sees in 64 bits."""

    def __init__(self, gpu, ctype, kv, hd, page, groups, members, prefix, total, g, n_extra=3, value=None, missing=()):
        import torch
        from ligguf_amd import ops
        nseq, most = groups * members, (max(total) + page - 1) // page + 1
        # shared full pages, then each sequence's own (its part-filled page of the shared rows among them)
        tab, n = np.full((nseq, most), -1, np.int32), 0
        for i in range(groups):
            sh, end = prefix[i] // page, [(total[i * members + m] + page - 1) // page for m in range(members)]
            tab[i * members:(i + 1) * members, :sh] = np.arange(n, n + sh)
            n += sh
            for m in range(members):
                e = max(end[m], (prefix[i] + page - 1) // page if m == 0 else 0)
                tab[i * members + m, sh:e] = np.arange(n, n + max(e - sh, 0))
                n += max(e - sh, 0)
        n += n_extra
        perm = g.permutation(n).astype(np.int32)
        tab = np.where(tab >= 0, perm[tab], -1).astype(np.int32)
        for s, j, what in missing:
            tab[s, j] = what
        self.table, self.page, self.n, self.ctype, self.kv, self.hd = tab, page, n, ctype, kv, hd
        vals = []
        for which in range(2):
            x = g.standard_normal((n, page, kv, hd)).astype(np.float32)
            if which == 1:
                x = x * 0.7 + 0.4
            if value is not None:
                value(which, x)
            vals.append(x)
        # rows that no sequence may see: garbage
        used = np.zeros((n, page), bool)
        for s in range(nseq):
            i, first = s // members, s - s % members
            for j in range(total[s]):
                o = tab[first if j < prefix[i] else s, j // page]
                if 0 <= o < n:
                    used[o, j % page] = True
        self.vals, tensors = [], []
        for which, x in enumerate(vals):
            x[~used] = np.nan if which == 0 else np.inf
            if ctype == L.F16:
                h = x.astype(np.float16)
                tensors.append(torch.from_numpy(h.reshape(n, page, kv * hd)).to(gpu))
                self.vals.append(h.astype(np.float64))
            else:
                b, v = zip(*(kv4_bytes(x[i]) for i in range(n)))
                tensors.append(torch.from_numpy(np.stack(b)[:, :kv * page * hd // 32 * 20]).contiguous().to(gpu))
                self.vals.append(np.stack(v).astype(np.float64))
        wide = torch.full((nseq, most + 5), 1 << 30, dtype=torch.int32, device=gpu)      # a table whose rows are part of longer ones
        wide[:, :most] = torch.from_numpy(tab).to(gpu)
        self.cache = ops.PagedKvCache(*tensors, wide[:, :most], kv, hd, ctype, page)

    def rows(self, s, first, pre, n):
        """(K, V, whether there is a page) of rows 0 .. n - 1 as sequence s sees them."""
        j = np.arange(n)
        o = np.where(j < pre, self.table[first, j // self.page], self.table[s, j // self.page])
        ok = (o >= 0) & (o < self.n)
        return self.vals[0][o * ok, j % self.page], self.vals[1][o * ok, j % self.page], ok


def reference(pg, q, pos, members, prefix, window, sinks, max_pos, max_prefix=None):
    """(out, bound): the bound as for the contiguous call (test_gpu_cattn.py), a second join more; and what that
    bound leaves out, weights that are tiny beside the largest.  Held in two fp16 parts a weight is off by
    up to half of fp16's least step, 2^-25, where the largest is 2^7 at least: 2^-32 of it, for each key."""
    nseq, ntok, heads, hd = q.shape
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for s in range(nseq):
        pre = min(max(prefix[s // members], 0), 1 << 30 if max_prefix is None else max_prefix) if members > 1 else 0
        for t in range(ntok):
            p = pos[s, t]
            if p < 0 or p > max_pos:
                continue
            K, V, ok = pg.rows(s, s - s % members, pre, p + 1)
            j = np.arange(p + 1)
            ok &= (j > p - window) | (j < sinks) if window else True
            if not ok.any():
                continue
            for h in range(heads):
                k, v = K[ok, h * pg.kv // heads], V[ok, h * pg.kv // heads]
                x = q[s, t, h].astype(np.float64)
                a = k @ x / np.sqrt(hd)
                A = (np.abs(k) @ np.abs(x)).max() / np.sqrt(hd)
                w = np.exp(a - a.max())
                w /= w.sum()
                out[s, t, h] = w @ v
                tol[s, t, h] = (2 * (A * (hd + 12) + 64) + 2 * ok.sum() + 80) * U * (w @ np.abs(v)) + 2.0 ** -32 * np.abs(v).sum(0) + 1e-37
    return out, tol


def check(gpu, ctype, heads, kv, hd, page, groups, members, prefix, total, ntok, window=0, sinks=0, pos=None, max_pos=None,
          max_prefix=None, seed=1, scale=1.0, tell=None, **kw):
    import torch
    from ligguf_amd import ops
    print(f"paged attn type {ctype} heads {heads}/{kv} of {hd}, page {page}, {groups} x {members}, {ntok} tokens, prefix {prefix}, "
          f"total {total[:4]}, window {window}/{sinks}", flush=True)
    g = np.random.default_rng(seed)
    pg = Pages(gpu, ctype, kv, hd, page, groups, members, prefix, total, g, **kw)
    if pos is None:
        pos = np.asarray(total)[:, None] - ntok + np.arange(ntok)
    pos = np.asarray(pos, np.int32).reshape(groups * members, ntok)
    q = (g.standard_normal((groups * members, ntok, heads, hd)) * scale).astype(np.float32)
    t = torch.from_numpy(q.reshape(groups * members, ntok, -1)).to(gpu)
    out = torch.full_like(t, float("nan"))
    told = torch.tensor(prefix if tell is None else tell, dtype=torch.int32, device=gpu)
    args = dict(window=window, sinks=sinks, max_pos=max_pos, prefix=told if members > 1 else None, max_prefix=max_prefix)
    ops.attention_paged(t, pg.cache, torch.from_numpy(pos).to(gpu), out=out, **args)
    got = out.cpu().numpy().reshape(q.shape).astype(np.float64)
    with np.errstate(invalid="ignore"):
        want, tol = reference(pg, q, pos, members, prefix if tell is None else tell, window, sinks,
                              pg.cache.n_ctx - 1 if max_pos is None else max_pos, max_prefix)
    fine = np.isfinite(want)
    assert not np.isfinite(got[~fine]).any()     # (an infinity in a visible value: infinite or NaN, as the call says)
    err = np.abs(got[fine] - want[fine])
    assert np.all(err <= tol[fine]), float(np.nanmax(err / tol[fine]))
    return got, pg, t, pos, args


HEADS = [(4, 2, 64), (8, 2, 128), (3, 3, 96), (2, 1, 256), (6, 6, 48), (17, 1, 64)]


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("heads,kv,hd", HEADS)
@pytest.mark.parametrize("page", [16, 64])
def test_single_tokens_of_groups(gpu, ctype, heads, kv, hd, page):
    if ctype == L.KV4 and hd == 48:
        pytest.skip("48 values hold no groups of 32")
    # one shared row, part of a page, several pages; beams that hold one own row or many
    check(gpu, ctype, heads, kv, hd, page, 2, 3, [37, 1], [38, 40, 95, 2, 30, 9], 1)
    check(gpu, ctype, heads, kv, hd, page, 1, 7, [300], [301, 310, 333, 420, 305, 302, 380], 1)
    # nothing shared in one of the groups
    check(gpu, ctype, heads, kv, hd, page, 2, 2, [0, 64], [20, 1, 65, 130], 1)
    # no groups at all
    check(gpu, ctype, heads, kv, hd, page, 3, 1, [0, 0, 0], [1, 77, 200], 1)


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_prompts_of_groups(gpu, ctype, page):
    check(gpu, ctype, 4, 2, 64, page, 2, 3, [70, 5], [100, 101, 140, 40, 41, 45], 30)
    check(gpu, ctype, 8, 2, 128, page, 1, 2, [333], [400, 361], 28)
    check(gpu, ctype, 4, 1, 128, page, 2, 1, [0, 0], [150, 90], 90)
    check(gpu, ctype, 2, 1, 256, page, 1, 3, [90], [130, 131, 150], 33)


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 2), (64, 0), (100, 70), (130, 4), (31, 1000), (5000, 4)])
def test_windows(gpu, ctype, window, sinks):
    """Windows that end in the own rows, in the shared ones, before them."""
    for ntok in (1, 20):
        check(gpu, ctype, 8, 2, 64, 32, 2, 5, [200, 90], [222, 230, 300, 400, 251, 120, 111, 130, 170, 240], ntok, window, sinks)


@pytest.mark.parametrize("ctype", TYPES)
def test_positions_inside_the_shared_rows(gpu, ctype):
    """Rows in any order, some whose position lies before the shared rows end, some without a token."""
    pos = [[5, 63, -1], [40, -1, 12], [70, 64, 0], [-1, -1, -1], [20, 33, 3], [1, 2, 90]]
    check(gpu, ctype, 4, 2, 64, 16, 2, 3, [64, 30], [80, 90, 71, 33, 34, 91], 3, pos=pos)
    check(gpu, ctype, 4, 2, 64, 16, 2, 3, [64, 30], [80, 90, 71, 33, 34, 91], 3, window=9, sinks=3, pos=pos, max_pos=70)
    for w in (0, 20):
        check(gpu, ctype, 16, 1, 128, 16, 1, 3, [64], [80, 90, 71], 1, window=w, pos=[[63], [-1], [10]])


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("ntok", [1, 25])
def test_missing_pages(gpu, ctype, ntok):
    """Table entries that are no pages, shared and own, of one sequence and of all: their keys are not seen; a row
    that sees none is zeros."""
    miss = [(0, 1, -1), (0, 4, 10 ** 6), (1, 7, -5), (2, 6, -2 ** 31), (2, 7, 2 ** 31 - 1)]
    check(gpu, ctype, 8, 2, 64, 16, 1, 3, [100], [126, 140, 128], ntok, missing=miss)
    got = check(gpu, ctype, 8, 2, 64, 64, 2, 1, [0, 0], [60, 130], ntok, missing=[(0, 0, -1), (1, 1, 99999)])[0]
    assert not got[0].any()
    check(gpu, ctype, 8, 2, 128, 16, 2, 2, [40, 40], [60, 61, 62, 63], ntok, window=30, sinks=2, missing=[(0, 1, -1), (3, 3, -1)])


@pytest.mark.parametrize("ctype", TYPES)
def test_counts_of_shared_rows_out_of_range(gpu, ctype):
    """Negative counts share nothing, large ones all that max_prefix allows."""
    check(gpu, ctype, 8, 2, 64, 16, 3, 2, [48, 0, 48], [60, 70, 20, 30, 55, 66], 1, tell=[48, -7, 2 ** 31 - 1], max_prefix=48)


@pytest.mark.parametrize("ctype", TYPES)
def test_long_contexts_in_parts(gpu, ctype):
    """Shared rows and own ones over several workgroups each, joined by either kernel."""
    check(gpu, ctype, 8, 2, 128, 64, 1, 2, [5000], [9100, 7000], 1)
    check(gpu, ctype, 4, 1, 64, 32, 1, 40, [3001], [3001 + 7 * i + 1 for i in range(40)], 1)
    check(gpu, ctype, 4, 1, 64, 16, 1, 3, [1500], [1600, 1640, 1655], 50)
    check(gpu, ctype, 1, 1, 256, 16, 2, 9, [700, 650], [700 + 20 * i + 1 for i in range(18)], 1)


def test_infinite_values_of_shared_rows(gpu):
    """An infinity or NaN in a value row that some rows see and others do not."""
    def value(which, x):
        if which == 1:
            x.reshape(-1, 2, 64)[::37, 0, 5] = np.inf
            x.reshape(-1, 2, 64)[5::41, 1, 60] = np.nan
            x.reshape(-1, 2, 64)[7::43, 1, 3] = -np.inf
    for ntok in (1, 12):
        for w, n in ((0, 0), (15, 1)):
            check(gpu, L.F16, 8, 2, 64, 16, 2, 3, [40, 33], [60, 52, 70, 61, 48, 55], ntok, window=w, sinks=n, value=value)


def test_zero_copy_of_a_prompt_equals_copies(gpu):
    """Beams whose tables hold the prompt's pages give what beams with copies of them give, to the last bits
    of the joins' order; and a call without groups over the same tables too."""
    import torch
    from ligguf_amd import ops
    got, pg, t, pos, args = check(gpu, L.F16, 8, 2, 128, 16, 1, 6, [96], [100, 110, 97, 99, 120, 105], 1)
    alone = ops.attention_paged(t, pg.cache, torch.from_numpy(pos).to(gpu))
    scale = float(alone.abs().max())
    # two orders of the same sums: each within (keys + 40) roundings of weights and sums
    assert float((alone.cpu() - torch.from_numpy(got).float().view(alone.shape)).abs().max()) <= 2 * (120 + 200) * U * scale


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("ntok", [1, 20])
def test_captured(gpu, ctype, ntok):
    """One captured call follows positions, counts of shared rows and tables from replay to replay."""
    import torch
    from ligguf_amd import ops
    # (192 rows fill their pages, which all four tables hold: fewer may be told shared)
    got, pg, t, pos, args = check(gpu, ctype, 8, 2, 64, 16, 1, 4, [192], [230, 260, 300, 222], ntok)
    p = torch.from_numpy(pos).to(gpu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(t)
    with torch.cuda.stream(s):
        ops.attention_paged(t, pg.cache, p, out=out, **args)
        s.synchronize()
        with torch.cuda.graph(graph, stream=s):
            ops.attention_paged(t, pg.cache, p, out=out, **args)
    torch.cuda.synchronize()
    for step in range(4):
        graph.replay()
        want = ops.attention_paged(t, pg.cache, p, **args)
        torch.cuda.synchronize()
        assert torch.equal(out, want), step
        p.sub_(1)
        args["prefix"].sub_(17)
        if step == 2:
            pg.cache.table[1].copy_(pg.cache.table[2])


def test_on_streams_of_their_own(gpu):
    """Calls that overlap on two streams, each with its workspace."""
    import torch
    from ligguf_amd import ops
    sets = [check(gpu, L.F16, 8, 2, 128, 16, 1, m, [900], [901 + 30 * i for i in range(m)], n, seed=m) for m, n in ((4, 1), (3, 15))]
    want = [torch.from_numpy(x[0]).float().to(gpu).view(x[2].shape) for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(8):
        for i, (x, s) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(s):
                outs[i].append(ops.attention_paged(x[2], x[1].cache, torch.from_numpy(x[3]).to(gpu), **x[4]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


def test_refusals_of_the_python_call(gpu):
    import torch
    from ligguf_amd import ops
    table = torch.zeros((4, 3), dtype=torch.int32, device=gpu)
    c = ops.PagedKvCache.empty(ops.F16, 5, 16, 2, 64, table)
    q, pos = torch.zeros(4, 1, 256, device=gpu), torch.zeros(4, 1, dtype=torch.int32, device=gpu)
    pre = torch.zeros(2, dtype=torch.int32, device=gpu)
    assert not ops.attention_paged(q, c, pos, prefix=pre).isnan().any()
    for bad in (lambda: ops.attention_paged(q[:3].contiguous(), c, pos), lambda: ops.attention_paged(q, c, pos[:2].contiguous()),
                lambda: ops.attention_paged(q, c, pos, prefix=pre.float()), lambda: ops.attention_paged(q, c, pos, prefix=pre[:0]),
                lambda: ops.attention_paged(q, c, pos, prefix=torch.zeros(3, dtype=torch.int32, device=gpu)),
                lambda: ops.attention_paged(q, c, pos, max_pos=48), lambda: ops.attention_paged(q, c, pos, prefix=pre.cpu()),
                lambda: ops.attention_paged(q, c, pos, prefix=pre, max_prefix=-1),
                lambda: ops.attention_paged(q, c, pos, prefix=pre, workspace=torch.empty(4, device=gpu)),
                lambda: ops.PagedKvCache(c.k, c.v, table.long(), 2, 64), lambda: ops.PagedKvCache(c.k, c.v, table.t(), 2, 64),
                lambda: ops.PagedKvCache(c.k, c.v, table.cpu(), 2, 64), lambda: ops.PagedKvCache(c.k, c.v[:4], table, 2, 64),
                lambda: ops.PagedKvCache(c.k, c.v, table[:0], 2, 64),
                lambda: ops.attention_paged(q, ops.PagedKvCache.empty(ops.F16, 5, 24, 2, 64, table), pos)):
        with pytest.raises(L.LgError):
            bad()
