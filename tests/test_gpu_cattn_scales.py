"""lg_attn_cache over the sizes that queries may have: small ones in tiles that a row does not
see or whose scores lie far below."""
import numpy as np
import pytest

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
