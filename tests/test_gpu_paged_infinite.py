"""Infinities and NaN in visible value rows over pages: they make their dim infinite or NaN for every row that sees
them, and no other row's, wherever the tiles of keys are seen whole by some rows of a launch and in part by others
-- prompts and windows whose ends lie inside a tile, own and shared rows -- against 64 bits on the GPU (bounds:
test_gpu_paged.py)."""
import numpy as np
import pytest

from ligguf_amd import lib as L
from test_gpu_paged import TYPES, U, Pages

pytestmark = pytest.mark.gpu


def compare(gpu, ctype, heads, kv, hd, page, groups, members, prefix, total, ntok, window=0, sinks=0, every=41, max_prefix=None):
    """Values of every `every`-th row of a page have one infinity or NaN (4 bits: a group of 32 is NaN); returns how many
    outputs have to be no numbers."""
    import torch
    from ligguf_amd import ops
    print(f"paged attn type {ctype} heads {heads}/{kv} of {hd}, page {page}, {groups} x {members}, {ntok} tokens, prefix {prefix}, "
          f"total {total[:4]}, window {window}/{sinks}", flush=True)
    g = np.random.default_rng(11)

    def value(which, x):
        if which == 1:
            y = x.reshape(-1, x.shape[-1])
            at = np.arange(3, len(y), every)
            y[at, g.integers(0, hd, at.size)] = np.nan if ctype == L.KV4 else np.array([np.inf, -np.inf, np.nan], np.float32)[at % 3]
    pg = Pages(gpu, ctype, kv, hd, page, groups, members, prefix, total, g, value=value)
    nseq, rep = groups * members, heads // kv
    pos = np.asarray(total)[:, None] - ntok + np.arange(ntok)
    q = torch.from_numpy(g.standard_normal((nseq, ntok, heads, hd)).astype(np.float32)).to(gpu)
    told = torch.tensor(prefix, dtype=torch.int32, device=gpu) if members > 1 else None
    got = ops.attention_paged(q.view(nseq, ntok, -1), pg.cache, torch.from_numpy(pos.astype(np.int32)).to(gpu), window=window, sinks=sinks,
                              max_pos=max(total) - 1, prefix=told, max_prefix=max(prefix) if members > 1 else None).view(q.shape)
    vals, none = [torch.from_numpy(x).to(gpu) for x in pg.vals], 0
    for s in range(nseq):
        n, pre = int(pos[s].max()) + 1, prefix[s // members] if members > 1 else 0
        j = np.arange(n)
        at = torch.from_numpy(np.where(j < pre, pg.table[s - s % members, j // page], pg.table[s, j // page]).astype(np.int64)).to(gpu)
        k, v = (x[at, torch.from_numpy(j % page).to(gpu)].transpose(0, 1).contiguous() for x in vals)        # [kv, n, hd]
        bad = (~v.isfinite()).double()
        v = torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0)
        p, t = torch.from_numpy(pos[s].astype(np.int64)).to(gpu)[:, None], torch.from_numpy(j).to(gpu)
        ok = (t <= p) & ((t > p - window) | (t < sinks)) if window else t <= p
        x = q[s].double().view(ntok, kv, rep, hd).permute(1, 0, 2, 3).reshape(kv, ntok * rep, hd)
        mask = ok.repeat_interleave(rep, 0)[None]
        a = (torch.bmm(x, k.transpose(1, 2).contiguous()) / hd ** 0.5).masked_fill(~mask, -np.inf)
        most = (torch.bmm(x.abs(), k.abs().transpose(1, 2).contiguous()) / hd ** 0.5).masked_fill(~mask, 0.0).amax(-1)
        w = torch.softmax(a, -1)
        seen = mask.double().expand(kv, -1, -1).contiguous()
        want, hit = torch.bmm(w, v), torch.bmm(seen, bad) > 0
        tol = (2 * (most * (hd + 12) + 64) + 2 * mask.sum(-1) + 80)[..., None] * U * torch.bmm(w, v.abs()) + 2.0 ** -32 * torch.bmm(seen, v.abs()) + 1e-37
        mine = got[s].double().view(ntok, kv, rep, hd).permute(1, 0, 2, 3).reshape(want.shape)
        assert torch.equal(~mine.isfinite(), hit), (s, int((mine.isfinite() & hit).sum()), int((~mine.isfinite() & ~hit).sum()))
        worst = float(((mine - want).abs() / tol)[~hit].max()) if (~hit).any() else 0.0
        assert worst <= 1, (s, worst)
        none += int(hit.sum())
    return none


def types(ctype, hd):
    if ctype == L.KV4 and hd == 48:
        pytest.skip("48 values hold no groups of 32")


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("hd", [48, 64, 96, 128, 256])
@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 0), (90, 20)])
def test_prompts_from_the_first_position(gpu, ctype, hd, window, sinks):
    """Rows whose last key lies in the first tile beside rows that see all of it."""
    types(ctype, hd)
    assert compare(gpu, ctype, 4, 1, hd, 64, 1, 1, [0], [200], 200, window, sinks) > 0
    assert compare(gpu, ctype, 8, 2, hd, 32, 16, 1, [0] * 16, [330] * 8 + [300] * 8, 300, window, sinks, every=83) > 0


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("hd", [48, 64, 96, 128, 256])
@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 5), (1200, 0)])
def test_prompts_behind_shared_rows(gpu, ctype, hd, window, sinks):
    types(ctype, hd)
    total = [1500 + 200 + 9 * i for i in range(4)] + [1300 + 190 + 20 * i for i in range(4)]
    assert compare(gpu, ctype, 32, 16, hd, 16, 2, 4, [1500, 1300], total, 140, window, sinks, every=251) > 0


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("hd,prefix", [(64, 20000), (128, 9000)])
def test_single_tokens_whose_windows_begin_apart(gpu, ctype, hd, prefix):
    """Sequences of one group up to 500 positions apart: windows that begin in other tiles of the shared rows."""
    members = 60
    total = [prefix + 1 + 500 * i // (members - 1) for i in range(members)]
    assert compare(gpu, ctype, 32, 8, hd, 64, 1, members, [prefix], total, 1, prefix // 2, 77, every=173) > 0
