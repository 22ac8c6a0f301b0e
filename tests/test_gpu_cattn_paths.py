"""lg_attn_cache's ways through long prompts, every row of each against 64 bits: several blocks
of columns in workgroups of eight waves, whole and with the keys in a few parts that a thread
joins (many rows) or in many that a workgroup does."""
import ctypes as C

import numpy as np
import pytest

from ligguf_amd import lib as L
from test_gpu_cattn import TYPES, U, make

pytestmark = pytest.mark.gpu


def plain(q, K, V, pos, window, sinks):
    """(out, bound) [ntok, heads, hd] in 64 bits on the GPU; the bound as in test_gpu_cattn.reference."""
    import torch
    ntok, heads, hd = q.shape
    out, tol = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    j, p = torch.arange(K.shape[0], device=q.device), pos[:, None].long()
    ok = (j <= p) & ((j > p - window) | (j < sinks) if window else True) & (p >= 0) & (p < K.shape[0])
    on = ok.any(1)
    for h in range(heads):
        k, v = (x[:, h * K.shape[1] // heads].contiguous() for x in (K, V))
        x = q[:, h].double()
        a = (x @ k.T.contiguous() / hd ** 0.5).masked_fill(~ok, -float("inf"))
        A = (x.abs() @ k.abs().T.contiguous() / hd ** 0.5).masked_fill(~ok, 0).amax(1)
        w = torch.softmax(a[on], 1)
        out[on, h] = w @ v
        rel = 2 * (A * (hd + 12) + 64) * U + (2 * ok.sum(1) + 40) * U
        tol[on, h] = rel[on, None] * (w @ v.abs()) + 1e-37
    return out, tol


# (sequences, tokens, heads, key heads, head_dim, keys, window, sinks), parts at least and at most
@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("shape,parts", [
    ((4, 300, 32, 8, 64, 400, 0, 0), (1, 1)), ((4, 300, 32, 8, 128, 400, 150, 3), (1, 1)), ((1, 260, 32, 8, 64, 2000, 0, 0), (2, 8)),
    ((1, 300, 32, 8, 128, 1500, 0, 0), (2, 8)), ((1, 300, 32, 8, 96, 1500, 0, 0), (2, 8)), ((1, 520, 32, 8, 128, 2000, 900, 70), (2, 8)),
    ((2, 150, 64, 8, 64, 1000, 0, 0), (2, 8)), ((1, 300, 16, 2, 64, 3000, 0, 0), (9, 64))])
def test_eight_waves_over_several_blocks(gpu, ctype, shape, parts):
    run(gpu, ctype, shape, parts, eight=True)


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("shape,parts", [
    ((1, 300, 32, 2, 64, 1000, 0, 0), (2, 8)), ((1, 300, 16, 4, 256, 2000, 0, 0), (2, 8)), ((1, 300, 16, 4, 256, 600, 100, 2), (1, 8))])
def test_other_long_prompts(gpu, ctype, shape, parts):
    run(gpu, ctype, shape, parts, eight=False)


def run(gpu, ctype, shape, parts, eight):
    import torch
    from ligguf_amd import ops
    nseq, ntok, heads, kv, hd, n_ctx, window, sinks = shape
    print(f"attn long prompt: type {ctype} {shape}", flush=True)
    g = np.random.default_rng(ntok + hd)
    cache, (K, V) = make(gpu, ctype, nseq, n_ctx, kv, hd, g)
    need = L.load().lg_attn_cache_workspace_size(C.byref(cache.desc), nseq, ntok, heads, window, sinks, n_ctx - 1)
    nsplit = need // (nseq * ntok * heads * (hd + 2) * 4) if need else 1
    # the way that is meant: so many parts; workgroups of four waves only where all of them, of 128 columns
    # each, fit the 256 CUs at once; rows enough that a thread joins
    assert parts[0] <= nsplit <= parts[1] and (nsplit in (1, *range(9, 65)) or nseq * ntok * heads > 4096)
    cols = ntok * heads // kv
    if eight:
        assert nseq * kv * -(-cols // 128) * nsplit > 256 and cols > 256
    q = torch.from_numpy(g.standard_normal((nseq, ntok, heads * hd)).astype(np.float32)).to(gpu)
    # each sequence's last tokens, the odd ones' ragged and padded, with idle rows between
    pos = np.tile(np.arange(n_ctx - ntok, n_ctx), (nseq, 1))
    pos[1::2] = np.where(np.arange(ntok) < ntok - 37, np.arange(ntok) + 11, -1)
    pos[:, [2, ntok // 2]] = [-1, n_ctx]
    p = torch.from_numpy(pos.astype(np.int32)).to(gpu)
    got = ops.attention_cache(q, cache, p, window=window, sinks=sinks).view(nseq, ntok, heads, hd)
    for s in range(nseq):
        want, tol = plain(q[s].view(ntok, heads, hd), *(torch.from_numpy(x[s]).to(gpu) for x in (K, V)), p[s], window, sinks)
        err = (got[s] - want).abs()
        assert bool((err <= tol).all()), (s, float((err / (tol + 1e-300)).max()))
        idle = (p[s] < 0) | (p[s] >= n_ctx)
        assert not got[s][idle].any() and got[s][~idle].any()
