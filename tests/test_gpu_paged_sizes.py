"""lg_attn_paged where its kernels change over and where their launch was cut for other
sizes than they meet; pools past 4 GiB; rows that are parts of longer ones, workspaces
used again, captured calls between eager ones (bounds and oracle: test_gpu_paged.py)."""
import numpy as np
import pytest

from ligguf_amd import lib as L
from test_gpu_paged import TYPES, U, check

pytestmark = pytest.mark.gpu


def spread(n, prefix, most):
    """Rows of n sequences beyond the shared ones: from one to `most`."""
    return [prefix + 1 + (most - 1) * i // max(n - 1, 1) for i in range(n)]


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("hd", [48, 64, 96, 128, 256])
@pytest.mark.parametrize("cols", [2, 15, 16, 17, 32, 33, 63, 64, 65, 96, 128, 129, 192, 193, 256, 257, 400])
def test_columns_of_shared_rows(gpu, ctype, hd, cols):
    """One query head: as many columns as the group has sequences."""
    if ctype == L.KV4 and hd == 48:
        pytest.skip("48 values hold no groups of 32")
    check(gpu, ctype, 1, 1, hd, 32, 1, cols, [150], spread(cols, 150, 40), 1)


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("hd", [48, 64, 96, 128, 256])
@pytest.mark.parametrize("ntok", [5, 6, 11, 21, 22, 43, 64, 65, 86])
def test_columns_of_prompts(gpu, ctype, hd, ntok):
    """Three query heads a key head: columns whose heads change inside a block of 16; alone and behind shared rows."""
    if ctype == L.KV4 and hd == 48:
        pytest.skip("48 values hold no groups of 32")
    check(gpu, ctype, 3, 1, hd, 16, 1, 1, [0], [ntok + 70], ntok)
    check(gpu, ctype, 3, 1, hd, 16, 1, 2, [45], [46 + ntok, 45 + ntok], ntok)


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("members,ntok", [(30, 1), (100, 1), (3, 9), (2, 70)])
@pytest.mark.parametrize("window,sinks", [(5, 0), (40, 3), (200, 130), (90, 1000)])
def test_windows_of_many_columns(gpu, ctype, members, ntok, window, sinks):
    check(gpu, ctype, 2, 2, 64, 16, 1, members, [301], spread(members, 300 + ntok, 90), ntok, window, sinks)
    check(gpu, ctype, 1, 1, 128, 64, 1, members, [130], spread(members, 129 + ntok, 50), ntok, window, sinks)


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("members,ntok", [(30, 1), (100, 1), (2, 50)])
def test_missing_pages_of_many_columns(gpu, ctype, members, ntok):
    miss = [(0, 0, -1), (0, 3, 10 ** 6), (1, 9, -5), (1, 10, -2 ** 31)]
    for w, n in ((0, 0), (60, 5)):
        check(gpu, ctype, 2, 1, 64, 16, 1, members, [140], spread(members, 139 + ntok, 60), ntok, w, n, missing=miss)
        check(gpu, ctype, 2, 1, 128, 32, 1, members, [140], spread(members, 139 + ntok, 60), ntok, w, n, missing=[(0, 1, -1), (1, 4, 1 << 30)])
    # a group whose shared rows have no page at all
    check(gpu, ctype, 2, 1, 64, 64, 1, members, [128], spread(members, 127 + ntok, 60), ntok, missing=[(0, 0, -1), (0, 1, -1)])


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("members,ntok", [(4, 1), (40, 1), (80, 1), (2, 20), (2, 90)])
def test_other_numbers_of_shared_rows_than_the_launch_was_cut_for(gpu, ctype, members, ntok):
    """max_prefix is a bound: of the groups one shares all of it, one a part, one nothing.  (Full pages, which every table holds.)"""
    for hd in (64, 128, 256):
        check(gpu, ctype, 1, 1, hd, 16, 3, members, [1200] * 3, spread(members, 1199 + ntok, 30) * 3, ntok, tell=[1200, 400, 0], max_prefix=1200,
              max_pos=1230 + ntok)


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("members,ntok", [(3, 1), (24, 1), (70, 1)])
@pytest.mark.parametrize("scale", [1e-41, 1e-30, 60.0])
def test_sizes_of_queries(gpu, ctype, members, ntok, scale):
    """Weights that are all alike, and weights that only a few keys have (the bound grows with the scores)."""
    check(gpu, ctype, 2, 1, 64, 16, 1, members, [333], spread(members, 333, 70), ntok, scale=scale)
    check(gpu, ctype, 2, 1, 128, 16, 1, members, [333], spread(members, 333, 70), ntok, scale=scale)


@pytest.mark.parametrize("members,ntok", [(3, 1), (40, 1), (90, 1), (2, 40)])
def test_far_scores_are_numbers(gpu, members, ntok):
    """Scores of 10^7 and more (their bound says little): averages of values, however the weights fall."""
    for hd in (64, 128):
        got, pg, *_ = check(gpu, L.F16, 2, 1, hd, 16, 1, members, [333], spread(members, 332 + ntok, 70), ntok, scale=1e7)
        v = np.where(np.isfinite(pg.vals[1]), pg.vals[1], 0)
        assert np.abs(got).max() <= np.abs(v).max() * (1 + 500 * U)


@pytest.mark.parametrize("members,ntok", [(3, 1), (24, 1), (100, 1), (2, 12), (2, 60)])
def test_infinities_and_no_numbers_in_many_columns(gpu, members, ntok):
    """In value rows and in key rows that some rows see: those whose 64-bit result is a number are that number."""
    def value(which, x):
        y = x.reshape(-1, x.shape[-1])
        if which == 1:
            y[::67, 5] = np.inf
            y[5::71, 60] = np.nan
            y[7::73, 3] = -np.inf
        else:
            y[200::97, 9] = np.nan
    for hd in (64, 128):
        for w, n in ((0, 0), (15, 1)):
            check(gpu, L.F16, 2, 1, hd, 16, 1, members, [40], spread(members, 39 + ntok, 40), ntok, w, n, value=value)


@pytest.mark.parametrize("members", [3, 24, 100])
def test_infinite_keys(gpu, members):
    """A key whose score is -infinity has no weight, at +infinity the row's head is no number; a row of such keys
    alone is zeros."""
    import torch
    from ligguf_amd import ops
    table = torch.arange(3, dtype=torch.int32, device=gpu)[None].repeat(members, 1)
    c = ops.PagedKvCache.empty(ops.F16, 3, 16, 1, 64, table)
    g = torch.Generator(device=gpu).manual_seed(1)
    c.k.normal_(generator=g)
    c.v.normal_(generator=g)
    q = torch.randn(members, 1, 64, device=gpu, generator=g).abs() + 0.1
    pos = torch.full((members, 1), 40, dtype=torch.int32, device=gpu)
    prefix = torch.tensor([32], dtype=torch.int32, device=gpu)
    run = lambda: ops.attention_paged(q, c, pos, prefix=prefix, max_prefix=32)  # noqa: E731
    c.k.view(48, 64)[7] = -np.inf
    c.k.view(48, 64)[35, 1] = -np.inf
    K, V = (x.view(48, 64).cpu().numpy().astype(np.float64) for x in (c.k, c.v))
    ok = np.arange(41)
    ok = ok[(ok != 7) & (ok != 35)]
    a = q[:, 0].cpu().numpy().astype(np.float64) @ K[ok].T / 8
    w = np.exp(a - a.max(1, keepdims=True))
    want = w / w.sum(1, keepdims=True) @ V[ok]
    A = (np.abs(q[:, 0].cpu().numpy()) @ np.abs(K[ok].T)).max() / 8
    tol = (2 * (A * 76 + 64) + 2 * 41 + 80) * U * np.abs(V).max()
    assert np.abs(run()[:, 0].cpu().numpy() - want).max() <= tol
    c.k.view(48, 64)[20, 3] = np.inf
    assert not run().isfinite().any()
    c.k.fill_(-np.inf)
    assert not run().any()


@pytest.mark.parametrize("ntok", [1, 30])
def test_bounds_that_bound_nothing(gpu, ntok):
    """A window and a number of shared rows as large as an int are no window and all rows."""
    import torch
    from ligguf_amd import ops
    got, pg, t, pos, args = check(gpu, L.F16, 4, 1, 64, 16, 1, 5, [160], spread(5, 159 + ntok, 60), ntok, max_prefix=160)
    p = torch.from_numpy(pos).to(gpu)
    want = ops.attention_paged(t, pg.cache, p, prefix=args["prefix"], max_prefix=pg.cache.n_ctx)
    top = 2 ** 31 - 1
    for kw in (dict(max_prefix=top), dict(max_prefix=pg.cache.n_ctx, window=top), dict(max_prefix=pg.cache.n_ctx, window=top, sinks=top),
               dict(max_prefix=pg.cache.n_ctx, window=pg.cache.n_ctx), dict(max_prefix=pg.cache.n_ctx, sinks=9)):
        assert torch.equal(ops.attention_paged(t, pg.cache, p, prefix=args["prefix"], **kw), want), kw
    # one less is a window, which of these positions all are inside of
    check(gpu, L.F16, 4, 1, 64, 16, 1, 5, [160], spread(5, 159 + ntok, 60), ntok, window=159 + ntok + 60, max_pos=159 + ntok + 60)


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("ntok", [1, 20])
def test_pools_past_4_gib(gpu, ctype, ntok):
    """Pages spread over 5 GiB of keys give what the same pages in a small pool give, bit for bit: written, read, moved."""
    import torch
    from ligguf_amd import ops
    kv, hd, page, members, most = 8, 128, 64, 5, 4
    n = (5 << 30) // (page * kv * hd * 2 if ctype == L.F16 else page * kv * hd * 5 // 8)
    at = torch.cat([torch.randperm(n - 40, generator=torch.Generator().manual_seed(2))[:members * most - 3],
                    torch.tensor([n - 1, n - 2, 0])]).to(gpu)                       # (0 and the last ones among them)
    table = torch.arange(members * most, dtype=torch.int32, device=gpu).view(members, most)
    table[:, :2] = table[0, :2]
    small = ops.PagedKvCache.empty(ctype, members * most, page, kv, hd, table)
    shape = (n, page, kv * hd) if ctype == L.F16 else (n, page * kv * hd * 5 // 8)
    big = ops.PagedKvCache(*(torch.empty(shape, dtype=small.k.dtype, device=gpu) for _ in range(2)), at.int()[table.long()], kv, hd, ctype, page)
    g = torch.Generator(device=gpu).manual_seed(3)
    freq = ops.rope_table(hd, 1e4)[0].to(gpu)
    prompt = torch.randn(1, 2 * page + 9, 2 * kv * hd, device=gpu, generator=g)
    big.k[at], big.v[at] = 0, 0
    for c in (small, big):
        one = ops.PagedKvCache(c.k, c.v, c.table[:1], kv, hd, ctype, page)
        k, v = prompt.split(kv * hd, 2)
        ops.qk_norm_rope_tokens(None, k, v, torch.arange(2 * page + 9, dtype=torch.int32, device=gpu)[None], freq, hd, cache=one)
    length = torch.tensor([2 * page + 9], dtype=torch.int32, device=gpu)
    parent = torch.zeros(1, members, dtype=torch.int32, device=gpu)
    for _ in range(3):
        for c in (small, big):
            ops.beam_reorder(ops.PagedLayers([c]), parent, length)
        assert torch.equal(at.int()[small.table.long()], big.table)
        x = torch.randn(members, ntok, 4 * kv * hd, device=gpu, generator=g)
        q, k, v = x.split([2 * kv * hd, kv * hd, kv * hd], 2)
        pos = length + torch.arange(ntok, dtype=torch.int32, device=gpu)[None].repeat(members, 1)
        prefix = torch.full((1,), 2 * page, dtype=torch.int32, device=gpu)
        outs = []
        for c in (small, big):
            r, _ = ops.qk_norm_rope_tokens(q, k, v, pos, freq, hd, cache=c)
            outs.append(ops.attention_paged(r, c, pos, prefix=prefix, max_prefix=2 * page))
        assert torch.equal(*outs) and outs[0].isfinite().all() and outs[0].any()
        for a, b in ((small.k, big.k), (small.v, big.v)):
            same = torch.equal(a.view(torch.uint8), b[at].view(torch.uint8))
            assert same
        length += ntok
        parent = torch.tensor([[1, 1, 4, 1, 0]], dtype=torch.int32, device=gpu)


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("members,ntok", [(3, 1), (24, 1), (2, 40)])
def test_rows_of_longer_ones_and_a_workspace_used_again(gpu, ctype, members, ntok):
    import torch
    from ligguf_amd import ops
    work = torch.empty(1 << 22, device=gpu)
    for hd, prefix in ((64, 400), (128, 90), (64, 2000)):
        got, pg, t, pos, args = check(gpu, ctype, 4, 2, hd, 16, 1, members, [prefix], spread(members, prefix - 1 + ntok, 60), ntok)
        p = torch.from_numpy(pos).to(gpu)
        wide = torch.full((members, ntok, 4 * hd + 24), float("nan"), device=gpu)
        wide[:, :, 8:4 * hd + 8] = t
        out = torch.full((members, ntok, 4 * hd + 12), 7.0, device=gpu)
        for _ in range(2):
            ops.attention_paged(wide[:, :, 8:4 * hd + 8], pg.cache, p, out=out[:, :, 4:4 * hd + 4], workspace=work, **args)
            assert torch.equal(out[:, :, 4:4 * hd + 4], torch.from_numpy(got).float().to(gpu).view(t.shape))
            assert (out[:, :, :4] == 7).all() and (out[:, :, 4 * hd + 4:] == 7).all()
            work.fill_(float("nan"))


def test_two_captured_calls_and_eager_ones(gpu):
    """Two graphs of one memory pool, replayed by turns with eager calls and other work between."""
    import torch
    from ligguf_amd import ops
    sets = [check(gpu, L.F16, 8, 2, 128, 16, 1, m, [640], spread(m, 639 + n, 50), n, seed=m) for m, n in ((4, 1), (20, 1), (2, 40))]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs, outs, want, pool = [], [], [], None
    calls = [lambda o, x=x, p=torch.from_numpy(x[3]).to(gpu): ops.attention_paged(x[2], x[1].cache, p, out=o, **x[4]) for x in sets]
    with torch.cuda.stream(s):
        for x, call in zip(sets, calls):
            o = torch.empty_like(x[2])
            call(o)
            s.synchronize()
            want.append(o.clone())
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s, pool=pool):
                call(o)
            pool = pool or graph.pool()
            graphs.append(graph)
            outs.append(o)
    torch.cuda.synchronize()
    for turn in range(5):
        for i in ((0, 1, 2), (2, 0, 1), (1, 2, 0), (0, 2, 1), (2, 1, 0))[turn]:
            outs[i].fill_(float("nan"))
            graphs[i].replay()
            eager = torch.empty_like(outs[i])
            calls[(i + 1) % 3](torch.empty_like(outs[(i + 1) % 3]))
            calls[i](eager)
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want[i]) and torch.equal(eager, want[i]), (turn, i)


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("heads", [1, 6])
def test_one_key_head_in_as_many_parts_as_there_are(gpu, ctype, heads):
    """A single key head over long contexts: shared and own rows each in hundreds of parts."""
    check(gpu, ctype, heads, 1, 64, 64, 1, 2, [50000], [90000, 70001], 1)
    check(gpu, ctype, heads, 1, 64, 64, 1, 1, [0], [100000], 1)


def test_the_other_kind_of_cache_is_refused(gpu):
    """Before anything is launched: a table has other sequences than its pool has pages."""
    import torch
    from ligguf_amd import ops
    paged = ops.PagedKvCache.empty(ops.KV4, 3, 16, 2, 64, torch.zeros((8, 2), dtype=torch.int32, device=gpu))
    flat = ops.KvCache.empty(ops.KV4, 32, 2, 64, 8, gpu)
    q, pos = torch.zeros(8, 1, 256, device=gpu), torch.zeros(8, 1, dtype=torch.int32, device=gpu)
    for bad in (lambda: ops.attention_cache(q, paged, pos, max_pos=8), lambda: ops.attention_paged(q, flat, pos), lambda: ops.kv_values(paged),
                lambda: ops.PagedLayers([flat])):
        with pytest.raises(L.LgError):
            bad()

    class Mine(ops.PagedKvCache):
        pass

    mine = Mine(paged.k, paged.v, paged.table, 2, 64, ops.KV4, 16)
    pos[1:] = -1          # (one row, or all would write to one place)
    r, _ = ops.qk_norm_rope_tokens(q, q[:, :, :128], q[:, :, 128:], pos, torch.ones(32, device=gpu), 64, cache=mine)
    assert ops.attention_paged(r, mine, pos).isfinite().all() and ops.kv_values(paged.pool)[0].shape == (3, 16, 128)
