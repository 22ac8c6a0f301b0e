"""The refusals of the calls over pages and of beam search (no GPU: every refusal comes
before the first device call), and what their Python handles refuse."""
import ctypes as C

import pytest

from ligguf_amd import lib as L
from test_kvrope_host import P, cache


def pages(type=L.F16, page=16, kv=2, hd=64, n=8, most=10, table=P, stride=None, **kw):
    return L.LgKvPages(cache(type=type, n_ctx=page, kv=kv, hd=hd, **kw), n, most, table, most if stride is None else stride)


BAD_PAGES = [dict(page=8), dict(page=17), dict(page=48), dict(page=1 << 17), dict(n=0), dict(n=-3), dict(most=0), dict(most=-1),
             dict(most=1 << 27), dict(table=None), dict(table=P + 2), dict(stride=9), dict(stride=1 << 33), dict(k=None), dict(v=P + 8),
             dict(seq=16), dict(seq=(1 << 32)), dict(kv=0), dict(hd=0)]


def attn(q=P, qs=256, c=None, pos=P, nseq=4, ntok=1, heads=4, window=0, sinks=0, max_pos=31, prefix=P, group=2, max_prefix=20, out=P,
         os=256, ws=P, wb=1 << 40):
    c = pages() if c is None else c
    return L.load().lg_attn_paged(q, qs, C.byref(c), pos, nseq, ntok, heads, window, sinks, max_pos, prefix, group, max_prefix, out, os, ws,
                                  wb, None)


@pytest.mark.parametrize("kw", BAD_PAGES)
def test_pages_refused(kw):
    assert attn(c=pages(**kw)) == -1 and L.load().lg_last_error(None)
    assert append(c=pages(**kw)) == -1


def test_unknown_types_are_refused():
    c = pages(type=L.Q8_0, seq=1 << 20)
    assert attn(c=c) == -2 and append(c=c) == -2
    assert L.load().lg_beam_reorder((L.LgKvCache * 1)(c.pool), 1, 8, P, 10, 10, P, P, 1, 4, P, 1 << 20, None) == -2


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(q=P + 4), dict(qs=255), dict(qs=128), dict(out=None), dict(out=P + 8), dict(os=258), dict(os=64), dict(pos=None),
    dict(nseq=-1), dict(ntok=-1), dict(heads=0), dict(heads=3), dict(heads=-4), dict(heads=1 << 20), dict(window=-1), dict(sinks=-1),
    dict(max_pos=-1), dict(max_pos=160), dict(c=pages(hd=80)), dict(c=pages(hd=32)), dict(c=pages(type=L.KV4, hd=48, seq=1 << 12)),
    dict(group=0), dict(group=-2), dict(group=3), dict(max_prefix=-1), dict(prefix=None), dict(nseq=1 << 15, ntok=1 << 15), dict(ws=None),
    dict(ws=P + 8), dict(wb=64),
])
def test_attention_refusals(kw):
    assert attn(**kw) == -1 and L.load().lg_last_error(None)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kv,heads", [(1, 1), (1, 8), (2, 4), (8, 32)])
def test_parts_of_long_contexts(kv, heads, hd):
    """The join takes 512 parts at most, however many keys are shared and own."""
    need = L.load().lg_attn_paged_workspace_size
    c = pages(page=1 << 15, kv=kv, hd=hd, most=1 << 10)
    for members in (1, 2, 3, 16):
        for last in (1000, 50000, 90000, 10 ** 6, (1 << 25) - 1):
            for prefix in (0, last // 3, last // 2, last):
                n = need(C.byref(c), members, 1, heads, 0, 0, last, members, prefix)
                assert n % (members * heads * (hd + 2) * 4) == 0 and n // (members * heads * (hd + 2) * 4) <= 512, (members, last, prefix)


def test_attention_workspace():
    need = L.load().lg_attn_paged_workspace_size
    c = pages(most=1000)
    n = need(C.byref(c), 4, 1, 4, 0, 0, 9000, 2, 8000)
    assert n > 0 and attn(c=c, max_pos=9000, max_prefix=8000, wb=n - 1) == -1
    assert need(C.byref(c), 4, 1, 4, 0, 0, 31, 1, 0) == 0           # nothing shared, few keys: written out at once
    for a in ((0, 1, 4, 0, 0, 9000, 2, 10), (4, -1, 4, 0, 0, 9000, 2, 10), (4, 1, 0, 0, 0, 9000, 2, 10), (4, 1, 4, -1, 0, 9000, 2, 10),
              (4, 1, 4, 0, 0, -1, 2, 10), (4, 1, 4, 0, 0, 9000, 0, 10), (4, 1, 4, 0, 0, 9000, 3, 10), (4, 1, 4, 0, 0, 9000, 2, -1)):
        assert need(C.byref(c), *a) == 0
    assert need(None, 4, 1, 4, 0, 0, 9000, 2, 10) == 0


def append(c=None, null=False, k=P, ks=128, v=P, vs=128, nseq=2, ntok=3, kv=2, hd=64, rope=64, pos=P):
    c = pages() if c is None else c
    return L.load().lg_qk_norm_rope_paged(P, 256, P, 256, k, ks, None, 0, v, vs, None, None, 4, kv, hd, rope, 0, P, 1.0, 1e-6, pos, nseq,
                                          ntok, None if null else C.byref(c), None)


@pytest.mark.parametrize("kw", [dict(null=True), dict(k=None), dict(v=None), dict(vs=64), dict(kv=1), dict(hd=62), dict(rope=66), dict(pos=None),
                                dict(nseq=-1), dict(nseq=1 << 20, ntok=1 << 10)])
def test_append_refusals(kw):
    assert append(**kw) == -1 and L.load().lg_last_error(None)


def select(x=P, stride=100, scores=P, done=None, end=1, groups=2, beams=4, vocab=100, top=8, out=(P, P, P), ws=P, wb=1 << 30):
    return L.load().lg_beam_select(x, stride, scores, done, end, groups, beams, vocab, top, *out, ws, wb, None)


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(x=P + 2), dict(stride=99), dict(scores=None), dict(groups=-1), dict(beams=0), dict(beams=65), dict(vocab=0),
    dict(vocab=-1), dict(vocab=2 ** 31 - 8, stride=2 ** 31), dict(top=0), dict(top=65), dict(out=(None, P, P)), dict(out=(P, None, P)),
    dict(out=(P, P, None)), dict(ws=None), dict(ws=P + 8), dict(wb=100), dict(groups=1 << 21),
])
def test_select_refusals(kw):
    assert select(**kw) == -1 and L.load().lg_last_error(None)
    need = L.load().lg_beam_select_workspace_size
    assert need(2, 65, 100, 8) == 0 and need(2, 4, 0, 8) == 0 and need(-1, 4, 100, 8) == 0 and need(2, 4, 100, 8) > 0


def reorder(c=None, n=1, pools=None, n_pages=8, table=P, stride=10, most=10, parent=P, length=P, groups=2, beams=4, ws=P, wb=1 << 20):
    c = cache(n_ctx=16) if c is None else c
    pools = (L.LgKvCache * max(n, 1))(*[c] * max(n, 1)) if pools is None else pools
    return L.load().lg_beam_reorder(pools, n, n_pages, table, stride, most, parent, length, groups, beams, ws, wb, None)


@pytest.mark.parametrize("kw", [
    dict(n=0), dict(n=-1), dict(n_pages=0), dict(table=None), dict(table=P + 1), dict(stride=9), dict(most=0), dict(parent=None),
    dict(length=None), dict(groups=-1), dict(groups=1 << 23), dict(beams=0), dict(beams=65), dict(ws=None), dict(ws=P + 8), dict(wb=127),
    dict(c=cache(n_ctx=24)), dict(c=cache(n_ctx=16, k=None)), dict(c=cache(n_ctx=16, hd=63)),
    dict(n=2, pools=(L.LgKvCache * 2)(cache(n_ctx=16), cache(n_ctx=32))),
    dict(n=2, pools=(L.LgKvCache * 2)(cache(n_ctx=16), cache(n_ctx=16, type=L.KV4, seq=cache(n_ctx=16).seq_bytes))),
    dict(c=cache(n_ctx=65536, kv=64, hd=256, seq=2 ** 32 - 16)),
])
def test_reorder_refusals(kw):
    assert reorder(**kw) == -1 and L.load().lg_last_error(None)


def test_no_rows_is_no_work():
    assert attn(nseq=0) == 0 and attn(ntok=0) == 0 and append(nseq=0) == 0 and select(groups=0) == 0 and reorder(groups=0) == 0


def test_python_handles_refuse_tensors_elsewhere():
    """Tables and pools have to lie on one GPU."""
    import torch
    from ligguf_amd import ops
    k = torch.zeros(4, 16, 128, dtype=torch.float16)
    with pytest.raises(L.LgError):
        ops.PagedKvCache(k, k, torch.zeros(2, 3, dtype=torch.int32), 2, 64)
    with pytest.raises(L.LgError):
        ops.PagedLayers([])
    with pytest.raises(L.LgError):
        ops.beam_select(torch.zeros(1, 2, 9), torch.zeros(1, 2), 3)


@pytest.mark.parametrize("kw", [
    dict(page=65536, kv=512, hd=128), dict(page=65536, kv=128, hd=256), dict(page=32768, kv=1 << 10, hd=64),
    dict(page=65536, kv=1024, hd=128, type=L.KV4), dict(page=65536, kv=2048, hd=64, type=L.KV4),
])
def test_a_single_page_past_32_bits_is_refused(kw):
    """Rows are found in their page by 32 bits; seq_bytes, which says nothing of a pool of one page, does not hide its size."""
    for seq in (0, 16, None):
        c = pages(n=1, **kw, **({} if seq is None else dict(seq=seq)))
        assert attn(c=c, heads=kw["kv"], nseq=0) == -1 and b"bytes below" in L.load().lg_last_error(None)
        if kw["hd"] == 64:
            assert append(c=c, kv=kw["kv"], ks=kw["kv"] * 64, vs=kw["kv"] * 64) == -1 and b"bytes below" in L.load().lg_last_error(None)
        assert reorder(c=c.pool, n_pages=1, groups=0) == -1 and b"bytes below" in L.load().lg_last_error(None)
    # the largest page that fits is none of these
    assert attn(c=pages(page=65536, kv=255, hd=128, n=1, seq=0), heads=255, nseq=0) == 0
