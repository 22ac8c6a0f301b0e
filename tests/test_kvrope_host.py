"""Rotary tables, cache sizes and the refusals of the many-token calls (no GPU:
every refusal comes before the first device call)."""
import ctypes as C
import math

import numpy as np
import pytest

from ligguf_amd import lib as L

P = 4096      # a 16-byte aligned address that no refused call follows


def cache(type=L.F16, n_ctx=32, kv=2, hd=64, k=P, v=P, seq=None):
    need = L.load().lg_kv_bytes(type, n_ctx, kv, hd)
    return L.LgKvCache(k, v, type, n_ctx, kv, hd, max(need, 0) if seq is None else seq)


def test_cache_bytes():
    b = L.load().lg_kv_bytes
    assert b(L.F16, 100, 8, 128) == 100 * 8 * 128 * 2
    assert b(L.KV4, 100, 8, 128) == 100 * 8 * (64 + 16)
    assert b(L.KV4, 100, 8, 48) == -1          # no groups of 32
    assert b(L.F16, (1 << 30) + 1, 1, 64) == -1
    assert b(L.F16, 1 << 30, 8, 128) == (1 << 30) * 2048     # past 32 bits
    for bad in [(L.F32, 1, 1, 64), (L.F16, 0, 1, 64), (L.F16, 1, 0, 64), (L.F16, 1, 1, 0), (L.F16, 1, 1, 257), (99, 1, 1, 64)]:
        assert b(*bad) == -1


def table(scaling, rope, base, factor=1.0, ctx=0, p0=0.0, p1=0.0):
    f, m = np.empty(max(rope, 0) // 2, np.float32), C.c_float()
    rc = L.load().lg_rope_table(scaling, rope, base, factor, ctx, p0, p1, f.ctypes.data, C.byref(m))
    return rc, f, m.value


@pytest.mark.parametrize("rope", [2, 6, 48, 64, 128, 256])
@pytest.mark.parametrize("base", [1e4, 1e6])
def test_rope_tables(rope, base):
    i = np.arange(rope // 2, dtype=np.float64)
    plain = base ** (-2 * i / rope)
    half = np.finfo(np.float32).eps / 2      # the one rounding; pow of two libraries: 1e-13 is ample
    tol = dict(rtol=half + 1e-13, atol=0)
    rc, f, m = table(L.ROPE_PLAIN, rope, base)
    assert rc == 0 and m == 1.0
    np.testing.assert_allclose(f.astype(np.float64), plain, **tol)
    rc, f, m = table(L.ROPE_LINEAR, rope, base, 4.0)
    assert rc == 0 and m == 1.0
    np.testing.assert_allclose(f.astype(np.float64), plain / 4, **tol)
    if rope > 2:
        rc, f, m = table(L.ROPE_NTK, rope, base, 8.0)
        assert rc == 0 and m == 1.0
        np.testing.assert_allclose(f.astype(np.float64), (base * 8.0 ** (rope / (rope - 2))) ** (-2 * i / rope), **tol)
        # its point: the slowest pair turns `factor` times slower, the fastest as trained
        np.testing.assert_allclose(f[-1], plain[-1] / 8, rtol=1e-6)
        assert f[0] == 1.0
    ctx = 8192
    turns = ctx * plain / (2 * math.pi)
    rc, f, m = table(L.ROPE_BANDS, rope, base, 8.0, ctx, 4.0, 1.0)
    w = np.clip((turns - 1) / 3, 0, 1)
    assert rc == 0 and m == 1.0
    np.testing.assert_allclose(f.astype(np.float64), plain / 8 * (1 - w) + plain * w, **tol)
    rc, f, m = table(L.ROPE_YARN, rope, base, 4.0, ctx, 32.0, 1.0)
    lo = max(math.floor(rope * math.log(ctx / (32 * 2 * math.pi)) / (2 * math.log(base))), 0)
    hi = min(math.ceil(rope * math.log(ctx / (2 * math.pi)) / (2 * math.log(base))), rope - 1)
    w = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
    assert rc == 0 and m == np.float32(1 + 0.1 * math.log(4))
    np.testing.assert_allclose(f.astype(np.float64), plain * (1 - w) + plain / 4 * w, **tol)


@pytest.mark.parametrize("args", [(9, 64, 1e4), (0, 63, 1e4), (0, 0, 1e4), (0, 258, 1e4), (0, 64, 1.0), (0, 64, float("nan")),
                                  (0, 64, float("inf")), (1, 64, 1e4, 0.5), (1, 64, 1e4, float("nan")), (2, 2, 1e4, 2.0),
                                  (3, 64, 1e4, 2.0, 0, 32.0, 1.0), (3, 64, 1e4, 2.0, 100, 1.0, 32.0), (4, 64, 1e4, 2.0, 100, 4.0, 0.0),
                                  (4, 64, 1e4, 2.0, 100, float("nan"), 1.0)])
def test_rope_table_refusals(args):
    assert table(*args)[0] == -1 and L.load().lg_last_error(None)


def rope(q=P, qs=256, qo=P, qos=256, k=P, ks=128, ko=P, kos=128, v=P, vs=128, qw=None, kw=None, nh=4, kv=2, hd=64, rd=64,
         layout=0, freq=P, mscale=1.0, eps=1e-6, pos=P, nseq=1, ntok=1, c=None):
    return L.load().lg_qk_norm_rope_tokens(q, qs, qo, qos, k, ks, ko, kos, v, vs, qw, kw, nh, kv, hd, rd, layout, freq, mscale,
                                           eps, pos, nseq, ntok, None if c is None else C.byref(c), None)


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(qo=None), dict(q=P + 4), dict(qs=254), dict(qs=250), dict(qos=255), dict(k=None), dict(k=P + 8), dict(ks=64),
    dict(ko=P + 4), dict(kos=64), dict(ko=None), dict(v=None, c=cache()), dict(v=P + 4, c=cache()), dict(vs=64, c=cache()),
    dict(nh=-1), dict(kv=0), dict(hd=0), dict(hd=63), dict(hd=258, qs=2000, qos=2000, ks=2000, kos=2000), dict(rd=66), dict(rd=-2),
    dict(rd=31), dict(layout=2), dict(freq=None), dict(pos=None), dict(eps=-1.0), dict(eps=float("nan")), dict(nseq=-1), dict(ntok=-1),
    dict(nseq=1 << 20, ntok=1 << 20), dict(c=cache(kv=3)), dict(c=cache(hd=128)), dict(c=cache(n_ctx=0)), dict(c=cache(k=None)),
    dict(c=cache(v=P + 8)), dict(nseq=2, c=cache(seq=16)), dict(nseq=2, c=cache(seq=32 * 256 + 8)),
    dict(nseq=2, c=cache(seq=1 << 60)),
    dict(hd=48, rd=48, qs=192, qos=192, ks=96, kos=96, vs=96, c=cache(type=L.KV4, hd=48, seq=0)),
])
def test_rope_refusals(kw):
    assert rope(**kw) == -1 and L.load().lg_last_error(None)


def test_rope_refuses_an_unknown_cache_type():
    assert rope(c=cache(type=L.F32, seq=1 << 20)) == -2


def test_no_rows_is_no_work():
    assert rope(nseq=0) == 0 and rope(ntok=0, c=cache()) == 0


@pytest.mark.parametrize("a", [dict(c=None), dict(nseq=-1), dict(nseq=70000), dict(pos0=-1), dict(npos=-1), dict(npos=33),
                               dict(pos0=30, npos=3), dict(k=None), dict(v=P + 2)])
def test_read_refusals(a):
    a = {**dict(c=cache(type=L.KV4), nseq=1, pos0=0, npos=1, k=P, v=P), **a}
    rc = L.load().lg_kv4_read(None if a["c"] is None else C.byref(a["c"]), a["nseq"], a["pos0"], a["npos"], a["k"], a["v"], None)
    assert rc == -1 and L.load().lg_last_error(None)


def test_read_refuses_an_fp16_cache():
    c = cache()
    assert L.load().lg_kv4_read(C.byref(c), 1, 0, 1, P, P, None) == -2
    c = cache(type=L.KV4)
    assert L.load().lg_kv4_read(C.byref(c), 1, 32, 0, P, P, None) == 0


def test_grids_past_32_bits_are_refused():
    """2^24 workgroups of 256 threads: more than a launch takes."""
    err = L.load().lg_last_error
    assert rope(ntok=1 << 24) == -1 and b"too many" in err(None)
    assert rope(nseq=1 << 14, ntok=1 << 10, nh=0, kv=1, c=cache(n_ctx=1 << 20, kv=1)) == -1 and b"too many" in err(None)
    c = cache(type=L.KV4, n_ctx=1 << 28)
    for npos in (1 << 28, (1 << 28) - 15):       # 2 heads of eight words: 2^32 words, 2^24 workgroups
        assert L.load().lg_kv4_read(C.byref(c), 1, 0, npos, P, P, None) == -1 and b"too many" in err(None)
