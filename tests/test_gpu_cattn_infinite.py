"""Infinities in visible keys: the score is -infinity (no weight), +infinity or, against a
query value of 0, NaN (both make the row's head NaN), whatever the query value's bits."""
import numpy as np
import pytest

from ligguf_amd import lib as L
from test_gpu_cattn import U, make

pytestmark = pytest.mark.gpu

# exact in one fp16 part; above and below what one part holds; small and denormal next to the others
VALUES = [1.0, 1 + 2.0 ** -13, 1 - 2.0 ** -13, 0.3, 1e-6, 1e-30, 1e-42]


def plain(q, K, V, pos):
    """softmax(q K^T / sqrt(hd)) V [ntok, heads, hd] in 64 bits and, where that is finite, its bound: scores
    of |a| under 32 are 12 + hd roundings of sum |q k| off, exponents 64 U, exp2 and parts 12 U, sums a
    rounding per key and 40 for the joins."""
    ntok, heads, hd = q.shape
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for t in range(ntok):
        for h in range(heads):
            g = h * K.shape[1] // heads
            k, v = K[:pos[t] + 1, g], V[:pos[t] + 1, g]
            with np.errstate(invalid="ignore"):
                a = (k * q[t, h].astype(np.float64)).sum(1) / np.sqrt(hd)
                p = np.exp(a - a.max())
                p = p / p.sum()
                out[t, h] = p @ v
            A = (np.abs(k[np.isfinite(a)]) @ np.abs(q[t, h].astype(np.float64))).max(initial=0) / np.sqrt(hd)
            tol[t, h] = (2 * A * (hd + 12) + 200 + 2 * len(k)) * U * np.abs(v).max()
    return out, tol


def run(gpu, cache, q, pos):
    import torch
    from ligguf_amd import ops
    t = torch.from_numpy(q.reshape(1, len(pos), -1)).to(gpu)
    got = ops.attention_cache(t, cache, torch.from_numpy(np.asarray(pos, np.int32)[None]).to(gpu))
    return got.cpu().numpy().reshape(q.shape)


def compare(got, want, tol):
    bad = np.isnan(want)
    assert np.array_equal(np.isnan(got), bad)
    assert np.all(np.abs(got - want)[~bad] <= tol[~bad])


@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("hd", [48, 64, 128, 256])
@pytest.mark.parametrize("ntok,n_ctx", [(1, 100), (4, 2500), (50, 300)])
def test_infinite_keys(gpu, value, hd, ntok, n_ctx):
    """Keys of either infinity against query values of both signs and 0."""
    g = np.random.default_rng(4)
    for inf in (np.inf, -np.inf):
        def edit(which, x):
            if which == 0:
                x[0, [7, n_ctx // 2], 0, 3] = inf
        cache, (K, V) = make(gpu, L.F16, 1, n_ctx, 2, hd, g, edit)
        q = g.standard_normal((ntok, 12, hd)).astype(np.float32)
        q[:, :, 3] = np.float32(value) * np.tile([1, -1, 0], 4)
        pos = np.arange(n_ctx - ntok, n_ctx)
        want, tol = plain(q, K[0], V[0], pos)
        up = 0 if inf < 0 else 1
        assert np.isfinite(want[:, up:6:3]).all() and np.isnan(np.delete(want[:, :6], [up, up + 3], 1)).all()
        compare(run(gpu, cache, q, pos), want, tol)


@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("ntok,n_ctx", [(1, 1), (1, 100), (2, 3000), (40, 200), (40, 3000)])
def test_rows_that_see_nothing_but_minus_infinity(gpu, hd, ntok, n_ctx):
    """0 / 0: such a row's head is NaN, one without a token stays 0."""
    g = np.random.default_rng(5)

    def edit(which, x):
        if which == 0:
            x[0, :, 0, 9] = -np.inf
    cache, (K, V) = make(gpu, L.F16, 1, n_ctx, 2, hd, g, edit)
    q = g.standard_normal((ntok, 4, hd)).astype(np.float32)
    q[:, :, 9] = 0.7
    pos = np.arange(n_ctx - ntok, n_ctx)
    want, tol = plain(q, K[0], V[0], pos)
    if ntok > 1:
        pos[0] = -1
        want[0] = 0
    assert np.isnan(want[1:, :2]).all()
    compare(run(gpu, cache, q, pos), want, tol)


def test_keys_of_minus_infinity_before_others(gpu):
    """Whole tiles and parts of such keys, then keys that count."""
    g = np.random.default_rng(6)
    for ntok, n_ctx, low in ((1, 300, 128), (1, 4000, 2000), (3, 3000, 2990), (40, 300, 200), (40, 4000, 3000)):
        def edit(which, x):
            if which == 0:
                x[0, :low, 1, 2] = -np.inf
        cache, (K, V) = make(gpu, L.F16, 1, n_ctx, 2, 64, g, edit)
        q = g.standard_normal((ntok, 4, 64)).astype(np.float32)
        q[:, :, 2] = 1 + 2.0 ** -13
        pos = np.arange(n_ctx - ntok, n_ctx)
        want, tol = plain(q, K[0], V[0], pos)
        assert np.isfinite(want).all()
        compare(run(gpu, cache, q, pos), want, tol)
