"""lg_attn_cache over the sizes that queries may have: small ones in tiles that a row does not
see or whose scores lie far below, large ones of which one key takes all, and the 22 bits
that queries and weights keep."""
import numpy as np
import pytest

from ligguf_amd import lib as L
from test_gpu_cattn import TYPES, U, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("scale", [3e-6, 1e-5, 1e-4, 1e-3, 1e-2, 0.05, 0.2])
def test_small_queries_whose_first_tile_is_not_theirs(gpu, ctype, hd, scale):
    """Windows without sinks, whose rows begin in different tiles; rows on both sides of a tile's
    border; parts of the keys that begin behind some rows."""
    for ntok, n_ctx, window, pos in ((4, 200, 0, [62, 63, 64, 65]), (3, 700, 0, [31, 32, 640]), (4, 300, 40, [70, 101, 130, 299]),
                                     (1, 300, 50, [270]), (60, 400, 70, np.arange(340, 400)), (90, 300, 0, np.arange(20, 110)),
                                     (3, 4000, 0, [40, 2047, 3999]), (40, 4000, 0, np.linspace(100, 3999, 40).astype(int))):
        print(f"attn small queries: type {ctype} hd {hd} scale {scale}: {ntok} rows, {n_ctx} keys, window {window}", flush=True)
        got, _, _ = check(gpu, ctype, 4, 2, hd, 1, ntok, n_ctx, window, 0, pos, scale=scale)
        assert np.isfinite(got).all()


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("ntok", [1, 4, 60])
def test_small_queries_after_keys_far_below(gpu, ctype, ntok):
    """A first tile whose scores lie hundreds of powers of two below 0 has no weight: every row is as
    without it, up to the order of sums (40 U and two roundings per key, of the sum of the values'
    sizes)."""
    import torch
    from ligguf_amd import ops
    g = np.random.default_rng(2)
    n_ctx, hd, low = 300, 64, 64

    def edit(which, x):
        if which == 0:
            x[:, :, :, 0] = 0
            x[:, :low, :, 0] = -30000
    cache, (K, V) = make(gpu, ctype, 1, n_ctx, 2, hd, g, edit)
    q = (g.standard_normal((1, ntok, 4, hd)) * 0.02).astype(np.float32)
    q[..., 0] = 0.2                               # -750 nats; the other dims of a 4-bit row, wide steps apart, add 75 at most
    pos = np.arange(n_ctx - ntok, n_ctx, dtype=np.int32)[None]
    got = ops.attention_cache(torch.from_numpy(q.reshape(1, ntok, -1)).to(gpu), cache, torch.from_numpy(pos).to(gpu))
    got = got.cpu().numpy().reshape(q.shape).astype(np.float64)
    for t in range(ntok):
        for h in range(4):
            k, v = K[0, low:pos[0, t] + 1, h // 2], V[0, low:pos[0, t] + 1, h // 2]
            a = k @ q[0, t, h].astype(np.float64) / 8
            p = np.exp(a - a.max())
            p /= p.sum()
            assert np.all(np.abs(got[0, t, h] - p @ v) <= (2 * len(k) + 168) * U * (p @ np.abs(v)))


@pytest.mark.parametrize("ctype", TYPES)
def test_large_queries_give_the_top_keys_value(gpu, ctype):
    """Scores of 10^6 and more, whose highest lies thousands above the next: its value, off by the
    parts of its weight (4 U), the sum's and the quotient's roundings."""
    import torch
    from ligguf_amd import ops
    g = np.random.default_rng(1)
    for hd in (64, 128, 256):
        for ntok, n_ctx in ((1, 300), (40, 300), (2, 5000)):
            cache, (K, V) = make(gpu, ctype, 1, n_ctx, 2, hd, g)
            q = (g.standard_normal((1, ntok, 4, hd)) * 1e6).astype(np.float32)
            pos = np.arange(n_ctx - ntok, n_ctx, dtype=np.int32)[None]
            got = ops.attention_cache(torch.from_numpy(q.reshape(1, ntok, -1)).to(gpu), cache, torch.from_numpy(pos).to(gpu))
            got = got.cpu().numpy().reshape(q.shape)
            seen = 0
            for t in range(ntok):
                for h in range(4):
                    a = K[0, :pos[0, t] + 1, h // 2] @ q[0, t, h].astype(np.float64) / np.sqrt(hd)
                    top = np.sort(a)[-2:]
                    if top[1] - top[0] < 3000:    # (scores of 10^7 are 1 or so off in fp32)
                        continue
                    v = V[0, a.argmax(), h // 2]
                    assert np.all(np.abs(got[0, t, h] - v) <= 16 * U * np.abs(v))
                    seen += 1
            assert seen >= 2 * ntok


def in_half(x):
    """x as the first fp16 part alone would hold it, under the power of two of its largest value."""
    e = np.frexp(np.abs(x).max(-1, keepdims=True))[1]
    return np.ldexp(np.ldexp(x, 14 - e).astype(np.float16).astype(np.float64), e - 14)


@pytest.mark.parametrize("ctype,hd", [(L.F16, 48), (L.F16, 64), (L.F16, 128), (L.F16, 256), (L.KV4, 64), (L.KV4, 128), (L.KV4, 256)])
@pytest.mark.parametrize("ntok,n_ctx", [(1, 300), (1, 5000), (4, 5000), (60, 300), (60, 5000)])
def test_queries_and_weights_keep_22_bits(gpu, ctype, hd, ntok, n_ctx):
    """40 keys, spread over the context, of one value each, in dims of their own, with scores within
    4; the rest lie 200 below and have no weight.  So a score is one product, off by the parts of the
    query value (4 nats x 4 U, and 2 U of its own for 4-bit values), and an output is one weight by
    the sum: 8 nats x 2.5 U of the scale's rounding, 6 U of the exponent's (up to 16), 2 U of exp2, 4 U
    of the weight's parts, 3 U each for at most 40 rescalings by a new maximum, 18 U for two joins, 2 U for
    the quotient: 190 U, as much for the sum, and 50 U of its additions.  One part alone is off by
    up to 2^12 U."""
    import torch
    from ligguf_amd import ops
    g = np.random.default_rng(hd + n_ctx)
    n, heads, kv = 40, 8, 2
    at = np.linspace(3, n_ctx - ntok, n).astype(int)
    dims = np.stack([1 + g.permutation(hd - 1)[:n] for _ in range(kv)])

    def edit(which, x):
        if which == 0:
            x[:] = 0
            x[0, :, :, 0] = -64 * np.sqrt(hd) / 8
        x[0, at] = 0
        for k in range(kv):
            x[0, at, k, dims[k]] = 1
    cache, (K, V) = make(gpu, ctype, 1, n_ctx, kv, hd, g, edit)
    q = g.uniform(-4, 4, (1, ntok, heads, hd)) * np.sqrt(hd)
    q[..., 0] = 32
    q = q.astype(np.float32)
    pos = np.arange(n_ctx - ntok, n_ctx, dtype=np.int32)[None]
    got = ops.attention_cache(torch.from_numpy(q.reshape(1, ntok, -1)).to(gpu), cache, torch.from_numpy(pos).to(gpu))
    got = got.cpu().numpy().reshape(q.shape).astype(np.float64)

    def weights(q, part):
        k = np.stack([K[0, at, h * kv // heads] for h in range(heads)])
        a = (k[None] @ q[0].astype(np.float64)[..., None])[..., 0] / np.sqrt(hd)
        p = np.exp(a - a.max(-1, keepdims=True))
        return (in_half(p) if part else p) / p.sum(-1, keepdims=True)
    want, tol = weights(q, False), 450 * U
    val = np.stack([V[0, at, h * kv // heads, dims[h * kv // heads]] for h in range(heads)])
    out = np.stack([got[0, :, h, dims[h * kv // heads]].T for h in range(heads)], 1)
    assert np.abs(out / val / want - 1).max() <= tol
    # what the bound is for: it would not hold with one part
    assert np.abs(weights(in_half(q.astype(np.float64)), False) / want - 1).max() > 4 * tol
    assert np.abs(weights(q, True) / want - 1).max() > 4 * tol
