"""lg_attn_paged where launches fill the chip, so that many columns are multiplied by tiles in LDS:
prompts and single tokens of many heads, against 64 bits on the GPU (bounds: test_gpu_paged.py)."""
import numpy as np
import pytest

from ligguf_amd import lib as L
from test_gpu_paged import TYPES, U, Pages

pytestmark = pytest.mark.gpu


def compare(gpu, ctype, heads, kv, hd, page, groups, members, prefix, total, ntok, window=0, sinks=0, idle=0, scale=1.0, **kw):
    import torch
    from ligguf_amd import ops
    print(f"paged attn type {ctype} heads {heads}/{kv} of {hd}, page {page}, {groups} x {members}, {ntok} tokens, prefix {prefix}, "
          f"total {total[:4]}, window {window}/{sinks}", flush=True)
    g = np.random.default_rng(4)
    pg = Pages(gpu, ctype, kv, hd, page, groups, members, prefix, total, g, **kw)
    nseq, rep = groups * members, heads // kv
    pos = np.asarray(total)[:, None] - ntok + np.arange(ntok)
    if idle:
        pos[1::2, ntok - idle:] = -1
    q = torch.from_numpy((g.standard_normal((nseq, ntok, heads, hd)) * scale).astype(np.float32)).to(gpu)
    told = torch.tensor(prefix, dtype=torch.int32, device=gpu) if members > 1 else None
    got = ops.attention_paged(q.view(nseq, ntok, -1), pg.cache, torch.from_numpy(pos.astype(np.int32)).to(gpu), window=window, sinks=sinks,
                              max_pos=max(total) - 1, prefix=told, max_prefix=max(prefix) if members > 1 else None).view(q.shape)
    vals = [torch.from_numpy(x).to(gpu) for x in pg.vals]
    for s in range(nseq):
        n, pre = max(int(pos[s].max()) + 1, 1), prefix[s // members] if members > 1 else 0
        j = np.arange(n)
        at = np.where(j < pre, pg.table[s - s % members, j // page], pg.table[s, j // page])
        held = torch.from_numpy((at >= 0) & (at < pg.n)).to(gpu)
        at = torch.from_numpy(np.where((at >= 0) & (at < pg.n), at, 0).astype(np.int64)).to(gpu)
        k, v = (x[at, torch.from_numpy(j % page).to(gpu)].transpose(0, 1).contiguous() for x in vals)        # [kv, n, hd]
        p, t = torch.from_numpy(pos[s].astype(np.int64)).to(gpu)[:, None], torch.from_numpy(j).to(gpu)
        ok = (t <= p) & held
        if window:
            ok &= (t > p - window) | (t < sinks)
        k, v = (torch.where(ok.any(0)[None, :, None], x, 0.0) for x in (k, v))                                # (garbage that nothing sees)
        x = q[s].double().view(ntok, kv, rep, hd).permute(1, 0, 2, 3).reshape(kv, ntok * rep, hd)
        mask = ok.repeat_interleave(rep, 0)[None]
        a = (torch.bmm(x, k.transpose(1, 2).contiguous()) / hd ** 0.5).masked_fill(~mask, -np.inf)
        most = (torch.bmm(x.abs(), k.abs().transpose(1, 2).contiguous()) / hd ** 0.5).masked_fill(~mask, 0.0).amax(-1)
        some, m = mask.any(-1), a.amax(-1, keepdim=True)
        w = torch.exp(a - torch.where(m == -np.inf, torch.zeros_like(m), m))
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
        seen = mask.double().expand(kv, -1, -1)
        want = torch.bmm(w, v) * some[..., None]
        tol = (2 * (most * (hd + 12) + 64) + 2 * mask.sum(-1) + 80)[..., None] * U * torch.bmm(w, v.abs()) + 2.0 ** -32 * torch.bmm(seen.contiguous(), v.abs()) + 1e-37
        mine = got[s].double().view(ntok, kv, rep, hd).permute(1, 0, 2, 3).reshape(want.shape)
        worst = float(((mine - want).abs() / tol).max())
        assert worst <= 1, (s, worst)


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("hd", [48, 64, 96, 128, 256])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 3), (333, 40)])
def test_prompts(gpu, ctype, hd, window, sinks):
    if ctype == L.KV4 and hd == 48:
        pytest.skip("48 values hold no groups of 32")
    total = [530, 400, 131, 512, 640, 257, 300, 600]
    compare(gpu, ctype, 16, 8, hd, 16, 8, 1, [0] * 8, total, 131, window, sinks, idle=50)
    compare(gpu, ctype, 16, 8, hd, 64, 8, 1, [0] * 8, total, 130, window, sinks, missing=[(0, 3, -1), (1, 0, 10 ** 6), (2, 1, -7), (3, 7, -1)])


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("hd", [48, 64, 96, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 5)])
def test_prompts_behind_shared_rows(gpu, ctype, hd, window, sinks):
    if ctype == L.KV4 and hd == 48:
        pytest.skip("48 values hold no groups of 32")
    miss = [(0, 3, -1), (0, 40, 10 ** 6), (4, 0, -7), (5, 95, -1)]
    total = [1500 + 200 + 9 * i for i in range(4)] + [1300 + 190 + 20 * i for i in range(4)]
    compare(gpu, ctype, 32, 16, hd, 16, 2, 4, [1500, 1300], total, 140, window, sinks, idle=30, missing=miss)


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("hd,prefix", [(64, 20000), (128, 9000)])
@pytest.mark.parametrize("scale", [1.0, 1e-41, 50.0])
def test_single_tokens_behind_many_shared_rows(gpu, ctype, hd, prefix, scale):
    members = 60
    total = [prefix + 1 + 3 * (i % 20) for i in range(members)]
    compare(gpu, ctype, 32, 8, hd, 64, 1, members, [prefix], total, 1, scale=scale, missing=[(0, 7, -1), (0, 100, 1 << 30)])
    compare(gpu, ctype, 32, 8, hd, 64, 1, members, [prefix], total, 1, window=prefix // 2, sinks=77, scale=scale)
