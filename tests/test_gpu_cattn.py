"""lg_attn_cache against softmax(q K^T / sqrt(hd)) V in 64 bits: both caches, every
head width, single tokens and prompts, windows and sinks, rows in any order and
without a token, infinities and NaN in invisible places, large caches, captured
calls, refusals."""
import ctypes as C

import numpy as np
import pytest

from ligguf_amd import lib as L
from test_gpu_kvrope import pack, words

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def kv4_bytes(x):
    """float [n_ctx, kv, hd] -> one sequence's 4-bit cache (uint8, padded to 16) and its values."""
    n_ctx, kv, hd = x.shape
    c, d, m, v = pack(x.transpose(1, 0, 2))
    b = np.concatenate([words(c).view(np.uint8), np.stack([d, m], 1).reshape(-1).view(np.uint8)])
    return np.concatenate([b, np.zeros(-b.size % 16, np.uint8)]), v.reshape(kv, n_ctx, hd).transpose(1, 0, 2)


def make(gpu, ctype, nseq, n_ctx, kv, hd, g, edit=None):
    """A cache of random rows and its values, float64 [nseq, n_ctx, kv, hd] each."""
    import torch
    from ligguf_amd import ops
    tensors, vals = [], []
    for which in range(2):
        x = g.standard_normal((nseq, n_ctx, kv, hd)).astype(np.float32)
        if which == 1:
            x = x * 0.7 + 0.4
        if edit is not None:
            edit(which, x)
        if ctype == L.F16:
            h = x.astype(np.float16)
            tensors.append(torch.from_numpy(h.reshape(nseq, n_ctx, kv * hd)).to(gpu))
            vals.append(h.astype(np.float64))
        else:
            b, v = zip(*(kv4_bytes(x[s]) for s in range(nseq)))
            tensors.append(torch.from_numpy(np.stack(b)).to(gpu))
            vals.append(np.stack(v).astype(np.float64))
    return ops.KvCache(*tensors, kv, hd, ctype, n_ctx), vals


def seen(p, n_ctx, window, sinks, max_pos):
    j = np.arange(n_ctx)
    if p < 0 or p > max_pos:
        return np.zeros(n_ctx, bool)
    return (j <= p) & ((j > p - window) | (j < sinks) if window else True)


def reference(q, K, V, pos, window, sinks, max_pos):
    """(out, bound) [nseq, ntok, heads, hd] in 64 bits.  Keys and values that a row does not
    see take no part.  The bound: a score is off by its products' roundings (parts of 22 bits:
    4 U, and hd + 8 additions) and its exponent's (64 U covers |s log2 e| up to 64, the rest by
    A); a weight by twice that (its own and the maximum's) and the exp2's 4 U; sums by one U per
    key and 32 for the joins."""
    nseq, ntok, heads, hd = q.shape
    kv = K.shape[2]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for s in range(nseq):
        for t in range(ntok):
            ok = seen(pos[s, t], K.shape[1], window, sinks, max_pos)
            if not ok.any():
                continue
            for h in range(heads):
                k, v = K[s, ok, h * kv // heads], V[s, ok, h * kv // heads]
                a = k @ q[s, t, h].astype(np.float64) / np.sqrt(hd)
                A = (np.abs(k) @ np.abs(q[s, t, h].astype(np.float64))).max() / np.sqrt(hd)
                p = np.exp(a - a.max())
                p /= p.sum()
                out[s, t, h] = p @ v
                rel = 2 * (A * (hd + 12) + 64) * U + (2 * ok.sum() + 40) * U
                tol[s, t, h] = rel * (p @ np.abs(v)) + 1e-37
    return out, tol


def check(gpu, ctype, heads, kv, hd, nseq, ntok, n_ctx, window, sinks, pos, max_pos=None, scale=1.0, edit=None, seed=1):
    import torch
    from ligguf_amd import ops
    g = np.random.default_rng(seed)
    pos = np.asarray(pos, np.int32).reshape(nseq, ntok)
    cache, (K, V) = make(gpu, ctype, nseq, n_ctx, kv, hd, g, edit)
    q = (g.standard_normal((nseq, ntok, heads, hd)) * scale).astype(np.float32)
    t = torch.from_numpy(q.reshape(nseq, ntok, -1)).to(gpu)
    out = torch.full_like(t, float("nan"))
    ops.attention_cache(t, cache, torch.from_numpy(pos).to(gpu), window=window, sinks=sinks, max_pos=max_pos, out=out)
    got = out.cpu().numpy().reshape(q.shape).astype(np.float64)
    with np.errstate(invalid="ignore"):
        want, tol = reference(q, K, V, pos, window, sinks, n_ctx - 1 if max_pos is None else max_pos)
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine], equal_nan=True)
    err = np.abs(got[fine] - want[fine])
    assert np.all(err <= tol[fine]), float(np.max(err / tol[fine]))
    return got, cache, t


TYPES = [L.F16, L.KV4]
HEADS = [(4, 2, 64), (8, 2, 128), (3, 3, 96), (2, 1, 256), (6, 6, 48), (17, 1, 64), (32, 2, 128), (5, 1, 128)]


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("heads,kv,hd", HEADS)
@pytest.mark.parametrize("n_ctx", [1, 33, 700])
def test_single_tokens(gpu, ctype, heads, kv, hd, n_ctx):
    if ctype == L.KV4 and hd == 48:
        pytest.skip("48 values hold no groups of 32")
    print(f"attn single: type {ctype} heads {heads}/{kv} of {hd} ctx {n_ctx}", flush=True)
    pos = [n_ctx - 1, 0, n_ctx // 2]
    check(gpu, ctype, heads, kv, hd, 3, 1, n_ctx, 0, 0, pos)
    check(gpu, ctype, heads, kv, hd, 3, 1, n_ctx, 20, 3, pos)


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 1), (64, 0), (65, 4), (100, 70), (500, 33), (5000, 4), (31, 1000)])
def test_windows(gpu, ctype, window, sinks):
    for ntok, n_ctx in ((1, 1000), (3, 700), (90, 600)):
        print(f"attn window {window} sinks {sinks} type {ctype}: {ntok} rows, {n_ctx} keys", flush=True)
        check(gpu, ctype, 4, 2, 64, 1, ntok, n_ctx, window, sinks, np.arange(n_ctx - ntok, n_ctx))


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("heads,kv,hd", HEADS)
@pytest.mark.parametrize("ntok,n_ctx", [(2, 2), (5, 70), (33, 300), (130, 130)])
def test_prompts(gpu, ctype, heads, kv, hd, ntok, n_ctx):
    if ctype == L.KV4 and hd == 48:
        pytest.skip("48 values hold no groups of 32")
    print(f"attn prompt: type {ctype} heads {heads}/{kv} of {hd}: {ntok} rows, {n_ctx} keys", flush=True)
    pos = np.stack([np.arange(n_ctx - ntok, n_ctx), np.arange(ntok)])
    check(gpu, ctype, heads, kv, hd, 2, ntok, n_ctx, 0, 0, pos)
    check(gpu, ctype, heads, kv, hd, 2, ntok, n_ctx, 37, 2, pos)


@pytest.mark.parametrize("ctype", TYPES)
def test_many_keys_few_rows(gpu, ctype):
    """Keys split over workgroups and joined."""
    check(gpu, ctype, 4, 2, 64, 1, 1, 9000, 0, 0, [8999])
    check(gpu, ctype, 8, 1, 128, 2, 2, 5000, 0, 0, [[4998, 4999], [3, 2000]])
    check(gpu, ctype, 4, 2, 64, 1, 20, 6000, 0, 0, np.arange(5980, 6000))
    check(gpu, ctype, 4, 2, 64, 1, 20, 6000, 3000, 100, np.arange(5980, 6000))


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("ntok", [1, 4, 60])
def test_rows_in_any_order_and_without_a_token(gpu, ctype, ntok):
    g = np.random.default_rng(5)
    n_ctx = 400
    for window, sinks in ((0, 0), (50, 3)):
        pos = g.integers(-3, n_ctx + 4, (5, ntok))
        pos[2] = -1                     # a sequence without any
        pos[3] = 2 ** 31 - 1
        pos[4, 0] = -2 ** 31
        got, _, _ = check(gpu, ctype, 8, 4, 64, 5, ntok, n_ctx, window, sinks, pos, max_pos=380)
        assert not got[2].any() and not got[3].any()


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("ntok", [1, 3, 70])
def test_what_invisible_rows_hold(gpu, ctype, bad, ntok):
    """NaN and infinities in rows that no row sees, and in a value row that only later ones see
    (4 bits hold no infinity: there only NaN differs from a large value)."""
    n_ctx, window, sinks = 300, 60, 2
    last = 250

    def edit(which, x):
        x[:, last + 1:] = bad                  # behind the last position
        x[:, 2:last - ntok - window] = bad     # between the sinks and every window
        if which == 1 and ntok > 1:
            x[:, last, 0, 5] = bad             # the last row's own value
    pos = np.arange(last - ntok + 1, last + 1)
    got, _, _ = check(gpu, ctype, 4, 2, 64, 1, ntok, n_ctx, window, sinks, pos, edit=edit)
    assert np.isfinite(got[:, :-1] if ntok > 1 else got).all()
    if ntok > 1 and (ctype == L.F16 or np.isnan(bad)):
        assert not np.isfinite(got[:, -1]).all()     # the row that sees it


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("scale", [1e-6, 30.0, 1e6])
def test_query_sizes(gpu, ctype, scale):
    """Tiny queries (equal weights), large ones (one key takes all) and ones beyond fp16."""
    check(gpu, ctype, 4, 2, 128, 1, 1, 300, 0, 0, [299], scale=scale)
    check(gpu, ctype, 4, 2, 128, 1, 40, 300, 0, 0, np.arange(260, 300), scale=scale)


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("scale", [1e-42, 1e-38, 1e32])
def test_queries_at_the_ends_of_fp32(gpu, ctype, scale):
    """Denormal queries (equal weights: the mean of what is seen) and ones whose scores near fp32's
    end (one key takes all), in tiles of which a row sees nothing."""
    import torch
    from ligguf_amd import ops
    g = np.random.default_rng(7)
    n_ctx, window = 500, 40
    cache, (K, V) = make(gpu, ctype, 1, n_ctx, 2, 64, g)
    for ntok in (1, 4, 60):
        q = (g.standard_normal((1, ntok, 4, 64)) * scale).astype(np.float32)
        pos = np.linspace(5, n_ctx - 1, ntok).astype(np.int32).reshape(1, -1)
        got = ops.attention_cache(torch.from_numpy(q.reshape(1, ntok, -1)).to(gpu), cache, torch.from_numpy(pos).to(gpu),
                                  window=window, sinks=1).cpu().numpy().reshape(q.shape)
        want, _ = reference(q, K, V, pos, window, 1, n_ctx - 1)
        assert np.max(np.abs(got - want)) <= 1e-5 * np.abs(V).max()


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("order", ["up", "down", "any"])
@pytest.mark.parametrize("hd", [64, 256])
def test_scores_that_come_from_afar(gpu, ctype, order, hd):
    """Maxima that move from -10^7 .. -10^4 past 0 to 10^4 .. 10^7, near and far columns in one
    wave.  A key's score is one product of an integer by a power of two, exact, and differs by over
    600 powers of two from the next, so the six keys of the highest share the row: their weights
    are equal, in parts 4 U off, their sums and the joins 40 U, the quotient 2 U."""
    import torch
    from ligguf_amd import ops
    g = np.random.default_rng(3)
    n_ctx, heads, kv = 3100, 8, 2
    k0 = (np.arange(n_ctx) // 6 * 4 - 1000.0)[{"up": slice(None), "down": slice(None, None, -1), "any": g.permutation(n_ctx)}[order]]

    def edit(which, x):
        if which == 0:
            x[:] = 0
            x[0, :, :, 0] = k0[:, None]
    cache, (K, V) = make(gpu, ctype, 1, n_ctx, kv, hd, g, edit)
    for ntok, window, sinks in ((1, 0, 0), (1, 300, 5), (4, 0, 0), (60, 0, 0), (60, 300, 5)):
        q = np.zeros((1, ntok, heads, hd), np.float32)
        q[..., 0] = np.array([2 ** 10, 2 ** 15, -2 ** 18, 2 ** 19, -2 ** 15, 2 ** 18, 2 ** 10, -2 ** 11]) * np.sqrt(hd / 64)
        pos = (np.array([n_ctx - 1]) if ntok == 1 else np.linspace(3, n_ctx - 1, ntok)).astype(np.int32).reshape(1, -1)
        got = ops.attention_cache(torch.from_numpy(q.reshape(1, ntok, -1)).to(gpu), cache, torch.from_numpy(pos).to(gpu),
                                  window=window, sinks=sinks).cpu().numpy().reshape(q.shape)
        want, _ = reference(q, K, V, pos, window, sinks, n_ctx - 1)
        size, _ = reference(q, K, np.abs(V), pos, window, sinks, n_ctx - 1)
        assert np.all(np.abs(got - want) <= 64 * U * size + 1e-37), (ntok, window, float(np.abs(got - want).max()))


def test_visible_key_nan_makes_its_rows_nan(gpu):
    for ntok in (1, 5, 50):
        def edit(which, x):
            if which == 0:
                x[:, 100, 0, 3] = np.nan
        got, _, _ = check(gpu, L.F16, 4, 2, 64, 1, ntok, 200, 0, 0, np.arange(200 - ntok, 200), edit=edit)
        assert np.isnan(got[0, :, :2]).all() and np.isfinite(got[0, :, 2:]).all()


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_ctx", [257, 400, 512])
def test_short_contexts_whose_rows_end_early(gpu, ctype, hd, n_ctx):
    """Single tokens at the borders of tiles and idle slots, NaN behind every position, whatever is
    read before the positions are known."""
    pos = [n_ctx - 1, 0, -1, 31, 32, 255, 256, n_ctx - 2, n_ctx]

    def edit(which, x):
        for s, p in enumerate(pos):
            x[s, p + 1 if p < n_ctx else 0:] = np.nan
    got, _, _ = check(gpu, ctype, 8, 2, hd, len(pos), 1, n_ctx, 0, 0, pos, edit=edit)
    assert not got[2].any() and not got[-1].any()


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("ntok", [1, 4, 40])
def test_queries_of_rows_without_a_token(gpu, ctype, ntok):
    """NaN and infinities in the queries of idle rows stay there, and their outputs are zeros."""
    import torch
    from ligguf_amd import ops
    g = np.random.default_rng(4)
    for n_ctx in (200, 2500):
        cache, _ = make(gpu, ctype, 3, n_ctx, 2, 64, g)
        q = torch.randn(3, ntok, 256, device=gpu)
        pos = torch.from_numpy(g.integers(0, n_ctx, (3, ntok)).astype(np.int32)).to(gpu)
        pos[1] = -1
        pos[2, 0] = n_ctx
        want = ops.attention_cache(q, cache, pos)
        q[1] = float("nan")
        q[2, 0] = float("inf")
        got = ops.attention_cache(q, cache, pos)
        assert torch.equal(got, want) and not got[1].any() and not got[2, 0].any()


def test_visible_infinity_in_a_value(gpu):
    """Where every row sees it, and far from any edge: its dim of every row that does is not finite,
    the other dims are as without it."""
    import torch
    from ligguf_amd import ops
    g = np.random.default_rng(6)
    for ntok in (1, 40):
        cache, _ = make(gpu, L.F16, 1, 600, 1, 64, g)
        q, pos = torch.randn(1, ntok, 128, device=gpu), torch.arange(600 - ntok, 600, dtype=torch.int32, device=gpu).view(1, -1)
        want = ops.attention_cache(q, cache, pos)
        cache.v[0, 70, 9] = float("inf")
        got = ops.attention_cache(q, cache, pos)
        bad = torch.zeros(64, dtype=torch.bool, device=gpu)
        bad[9] = True
        got, want = got.view(ntok, 2, 64), want.view(ntok, 2, 64)
        assert not torch.isfinite(got[..., bad]).any() and torch.equal(got[..., ~bad], want[..., ~bad])


@pytest.mark.parametrize("ntok", [1, 4, 60])
@pytest.mark.parametrize("n_ctx", [200, 3100])
def test_visible_infinity_in_a_value_of_no_weight(gpu, ntok, n_ctx):
    """Also where the key's weight, or that of all the keys of its part, is 0 in fp32."""
    import torch
    from ligguf_amd import ops
    g = np.random.default_rng(6)

    def edit(which, x):
        x[0, :, :, 0] = [np.linspace(-50, 50, n_ctx)[:, None], x[0, :, :, 0]][which]
        if which == 1:
            x[0, 7, 1, 5] = np.inf
    cache, _ = make(gpu, L.F16, 1, n_ctx, 2, 64, g, edit)
    q = torch.randn(1, ntok, 4, 64, generator=torch.Generator().manual_seed(2)).to(gpu)
    q[..., 0] = 100.0
    pos = torch.arange(n_ctx - ntok, n_ctx, dtype=torch.int32, device=gpu)[None]
    got = ops.attention_cache(q.flatten(2), cache, pos).view(ntok, 4, 64).isfinite()
    assert got[:, :2].all() and not got[:, 2:, 5].any()
    got[:, 2:, 5] = True
    assert got.all()


def test_prompts_over_many_column_blocks_and_parts(gpu):
    """Several blocks of columns, the last one cut, whole and with the keys in parts."""
    check(gpu, L.F16, 4, 2, 64, 1, 333, 340, 0, 0, np.arange(7, 340))
    check(gpu, L.KV4, 8, 1, 64, 1, 70, 5000, 0, 0, np.arange(4930, 5000))
    check(gpu, L.F16, 2, 1, 256, 1, 150, 1300, 700, 5, np.arange(1150, 1300))


def test_strided_rows_and_what_lies_between(gpu):
    import torch
    from ligguf_amd import ops
    g = np.random.default_rng(3)
    cache, _ = make(gpu, L.F16, 2, 50, 2, 64, g)
    pos = torch.arange(80, dtype=torch.int32, device=gpu).view(2, 40) % 50
    wide = torch.randn(2, 40, 4 * 64 + 12, device=gpu)
    q = wide[:, :, 4:260]
    want = ops.attention_cache(q.contiguous(), cache, pos)
    buf = torch.full((2, 40, 300), 7.0, device=gpu)
    ops.attention_cache(q, cache, pos, out=buf[:, :, 8:264])
    assert torch.equal(buf[:, :, 8:264], want)
    assert (buf[:, :, :8] == 7).all() and (buf[:, :, 264:] == 7).all()


@pytest.mark.parametrize("ctype", TYPES)
def test_offsets_past_32_bits(gpu, ctype):
    """Rows beyond 4 GiB of a cache, and a second sequence beyond it."""
    import torch
    from ligguf_amd import ops
    kv, hd = 8, 128
    n_ctx = (2 ** 32 + 2 ** 27) // (kv * hd * 2 if ctype == L.F16 else kv * hd * 5 // 8) // 16 * 16
    cache = ops.KvCache.empty(ctype, n_ctx, kv, hd, 2, gpu)
    x = torch.randn(2, 300, 2 * kv * hd, device=gpu)
    at = torch.arange(n_ctx - 300, n_ctx, dtype=torch.int32, device=gpu).repeat(2, 1)
    ops.qk_norm_rope_tokens(None, x[..., :kv * hd], x[..., kv * hd:], at, None, hd, rope_dim=0, cache=cache)
    small = ops.KvCache.empty(ctype, 300, kv, hd, 2, gpu)
    near = torch.arange(300, dtype=torch.int32, device=gpu).repeat(2, 1)
    ops.qk_norm_rope_tokens(None, x[..., :kv * hd], x[..., kv * hd:], near, None, hd, rope_dim=0, cache=small)
    for ntok in (1, 40):
        q = torch.randn(2, ntok, 16 * hd, device=gpu)
        a = ops.attention_cache(q, cache, at[:, -ntok:].contiguous(), window=200)
        b = ops.attention_cache(q, small, near[:, -ntok:].contiguous(), window=200)
        # the same keys, in tiles that begin elsewhere: sums in another order
        assert float((a - b).abs().max()) <= 1e-5 * float(b.abs().max()) and float(b.abs().max()) > 0.1
    del cache
    torch.cuda.empty_cache()


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("ntok,n_ctx,heads", [(1, 3000, 8), (4, 500, 4), (50, 700, 4)])
def test_captured_calls(gpu, ctype, ntok, n_ctx, heads):
    """Two captured calls with a workspace each, replayed with other positions and queries, next to
    eager calls; every replay equals the eager result bit for bit."""
    import torch
    from ligguf_amd import ops
    g = np.random.default_rng(8)
    cache, _ = make(gpu, ctype, 2, n_ctx, 2, 64, g)
    q = [torch.randn(2, ntok, heads * 64, device=gpu) for _ in range(2)]
    pos = [torch.zeros(2, ntok, dtype=torch.int32, device=gpu) for _ in range(2)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(s):
        for i in range(2):
            ops.attention_cache(q[i], cache, pos[i], window=300 * i, sinks=2)
            s.synchronize()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=s):
                outs.append(ops.attention_cache(q[i], cache, pos[i], window=300 * i, sinks=2))
            graphs.append(gr)
    torch.cuda.synchronize()
    for r in range(5):
        for i in range(2):
            q[i].normal_()
            pos[i].copy_(torch.from_numpy(g.integers(-1, n_ctx, (2, ntok)).astype(np.int32)))
        for gr in graphs:
            gr.replay()
        want = [ops.attention_cache(q[i], cache, pos[i], window=300 * i, sinks=2) for i in range(2)]
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], want[i])


def test_same_results_every_time(gpu):
    import torch
    from ligguf_amd import ops
    g = np.random.default_rng(9)
    cache, _ = make(gpu, L.KV4, 1, 5000, 2, 128, g)
    for ntok in (1, 24, 300):
        q = torch.randn(1, ntok, 8 * 128, device=gpu)
        pos = torch.arange(5000 - ntok, 5000, dtype=torch.int32, device=gpu).view(1, -1)
        a = ops.attention_cache(q, cache, pos)
        for _ in range(5):
            assert torch.equal(ops.attention_cache(q, cache, pos), a)


def test_python_refusals(gpu):
    import torch
    from ligguf_amd import ops
    cache = ops.KvCache.empty(ops.F16, 20, 2, 64, 2, gpu)
    q, pos = torch.zeros(2, 3, 256, device=gpu), torch.zeros(2, 3, dtype=torch.int32, device=gpu)
    ops.attention_cache(q, cache, pos)
    for bad in (dict(q=q[:1]), dict(q=q[..., :250]), dict(q=q[..., :192]), dict(q=q.half()), dict(pos=pos.long()),
                dict(pos=pos[:1].contiguous()), dict(window=-1), dict(sinks=-1), dict(max_pos=20), dict(max_pos=-1),
                dict(out=q[:, :2]), dict(out=torch.zeros(2, 3, 258, device=gpu)[..., 1:257])):
        with pytest.raises(L.LgError):
            ops.attention_cache(**{**dict(q=q, cache=cache, pos=pos), **bad})


def test_workspace_must_hold_the_partials(gpu):
    import torch
    from ligguf_amd import ops
    lib = L.load()
    cache = ops.KvCache.empty(ops.F16, 9000, 2, 64, 1, gpu)
    q, pos = torch.zeros(1, 1, 256, device=gpu), torch.full((1, 1), 8999, dtype=torch.int32, device=gpu)
    need = lib.lg_attn_cache_workspace_size(C.byref(cache.desc), 1, 1, 4, 0, 0, 8999)
    assert need > 0
    ops.attention_cache(q, cache, pos, workspace=torch.empty(need, dtype=torch.uint8, device=gpu))
    for ws in (torch.empty(need - 1, dtype=torch.uint8, device=gpu), torch.empty(need + 8, dtype=torch.uint8, device=gpu)[8:]):
        with pytest.raises(L.LgError):
            ops.attention_cache(q, cache, pos, workspace=ws)
    c = C.c_void_p
    assert lib.lg_attn_cache(c(q.data_ptr()), 256, C.byref(cache.desc), c(pos.data_ptr()), 1, 1, 4, 0, 0, 8999,
                             c(q.data_ptr()), 256, None, 0, None) == -1
