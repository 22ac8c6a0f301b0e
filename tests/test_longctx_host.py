"""The refusals of lg_attn_cache and lg_logprobs (no GPU: every refusal comes before
the first device call)."""
import ctypes as C

import pytest

from ligguf_amd import lib as L
from test_kvrope_host import P, cache


def attn(q=P, qs=256, c=None, pos=P, nseq=1, ntok=1, heads=4, window=0, sinks=0, max_pos=31, out=P, os=256, ws=P, wb=1 << 30):
    c = cache() if c is None else c
    return L.load().lg_attn_cache(q, qs, C.byref(c), pos, nseq, ntok, heads, window, sinks, max_pos, out, os, ws, wb, None)


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(q=P + 4), dict(qs=255), dict(qs=128), dict(out=None), dict(out=P + 8), dict(os=258), dict(os=64), dict(pos=None),
    dict(nseq=-1), dict(ntok=-1), dict(heads=0), dict(heads=3), dict(heads=-4), dict(heads=1 << 20), dict(window=-1), dict(sinks=-1),
    dict(max_pos=-1), dict(max_pos=32), dict(nseq=1 << 15, ntok=1 << 15, c=cache(seq=1 << 20)), dict(c=cache(hd=80)),
    dict(c=cache(hd=48, type=L.KV4, seq=16)), dict(c=cache(hd=32)), dict(c=cache(k=None)), dict(c=cache(v=P + 4)),
    dict(nseq=2, c=cache(seq=16)), dict(c=cache(kv=0)),
])
def test_attention_refusals(kw):
    assert attn(**kw) == -1 and L.load().lg_last_error(None)


def test_attention_refuses_an_unknown_cache_type():
    assert attn(c=cache(type=L.Q8_0, seq=1 << 20)) == -2
    assert L.load().lg_attn_cache(P, 256, None, P, 1, 1, 4, 0, 0, 31, P, 256, P, 1 << 20, None) == -1


def test_attention_refuses_a_workspace_too_small():
    c = cache(n_ctx=9000)
    need = L.load().lg_attn_cache_workspace_size(C.byref(c), 1, 1, 4, 0, 0, 8999)
    assert need > 0
    for ws, wb in ((None, need), (P, need - 1), (P + 8, need)):
        assert attn(c=c, max_pos=8999, ws=ws, wb=wb) == -1
    # sizes that no call takes need none
    for a in ((0, 1, 4, 0, 0, 8999), (1, -1, 4, 0, 0, 8999), (1, 1, 0, 0, 0, 8999), (1, 1, 4, -1, 0, 8999), (1, 1, 4, 0, 0, -1)):
        assert L.load().lg_attn_cache_workspace_size(C.byref(c), *a) == 0
    assert L.load().lg_attn_cache_workspace_size(None, 1, 1, 4, 0, 0, 8999) == 0


def test_no_rows_is_no_work():
    assert attn(nseq=0) == 0 and attn(ntok=0) == 0 and logp(rows=0) == 0


def logp(x=P, stride=100, rows=2, vocab=100, toks=P, top=3, lp=P, ent=P, ids=P, tl=P):
    return L.load().lg_logprobs(x, stride, rows, vocab, toks, top, lp, ent, ids, tl, None)


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(x=P + 2), dict(stride=99), dict(stride=0), dict(rows=-1), dict(vocab=0), dict(vocab=-1), dict(top=-1), dict(top=33),
    dict(vocab=2, top=3), dict(toks=None), dict(lp=None), dict(ids=None), dict(tl=None), dict(top=0),
])
def test_logprobs_refusals(kw):
    assert logp(**kw) == -1 and L.load().lg_last_error(None)


def test_grids_past_32_bits_are_refused():
    """2^24 workgroups of 256 threads, 2^22 of 1024: more than a launch takes."""
    err = L.load().lg_last_error
    assert attn(nseq=1 << 23, heads=2) == -1 and b"too many" in err(None)
    assert attn(nseq=1 << 20, ntok=64, heads=8, qs=512, os=512, c=cache(kv=8)) == -1 and b"too many" in err(None)
    assert logp(rows=1 << 24) == -1 and b"too many" in err(None)
    assert logp(rows=1 << 22, vocab=40000, stride=40000) == -1 and b"too many" in err(None)
