"""lg_qk_norm_rope_tokens and lg_kv4_read against the formulas in 64 bits: norm,
rotation in both layouts, fp16 and 4-bit cache rows, rows without a token,
strided and in-place rows, far positions, large caches, captured calls."""
import math

import numpy as np
import pytest

from ligguf_amd import lib as L

pytestmark = pytest.mark.gpu
U = 2.0 ** -24          # half a step of fp32, relative


def pack(x):
    """float [..., 32 n] -> codes and (d, m) of the 4-bit form, float64 throughout."""
    g = np.clip(np.asarray(x, np.float64), -60000, 60000).reshape(-1, 32)
    m = g.min(1).astype(np.float32).astype(np.float16)
    d = np.maximum(((g.max(1) - m.astype(np.float64)) / 15).astype(np.float32), 0).astype(np.float16)
    dd = np.where(d > 0, d.astype(np.float64), 1.0)
    c = np.where((d > 0)[:, None], np.clip(np.rint((g - m.astype(np.float64)[:, None]) / dd[:, None]), 0, 15), 0)
    nan = np.isnan(np.asarray(x)).reshape(-1, 32).any(1)
    d[nan] = m[nan] = np.float16("nan")
    c[nan] = 0
    v = (c * d.astype(np.float64)[:, None] + m.astype(np.float64)[:, None]).astype(np.float16)
    return c.astype(np.uint32), d, m, v.reshape(np.shape(x))


def words(c):
    c = c.reshape(-1, 4, 2)
    return sum(c[:, j, i] << np.uint32(4 * j + 16 * i) for j in range(4) for i in range(2))


def expected(x, w, pos, freq, rope, half, mscale, eps):
    """(values, bound on the fp32 error) of rows x [T, heads, hd] in 64 bits."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    r = rope // 2
    ang = pos.astype(np.float64)[:, None] * freq.astype(np.float64)
    c, s = (f(ang)[:, None] * float(np.float32(mscale)) for f in (np.cos, np.sin))
    y, size = x.copy(), np.abs(x)
    i0, i1 = (np.arange(r), np.arange(r) + r) if half else (2 * np.arange(r), 2 * np.arange(r) + 1)
    a, b = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = a * c - b * s, a * s + b * c
    size[..., i0] = size[..., i1] = (np.abs(a) + np.abs(b)) * abs(mscale)
    # norm: 12 additions of squares (relative, halved by the root), the mean, eps, root, quotient, two
    # products: under 13 half steps; cos and sin: 2 (their own, mscale's); the products and sum: 2
    return y, size * 17 * U


def run_case(gpu, T, nseq, heads, kv, hd, rope, half, norm, ctype, pos=None, mscale=1.0, n_ctx=None, seed=0):
    import torch
    from ligguf_amd import ops
    g = np.random.default_rng(seed)
    pos = np.stack([g.permutation(n_ctx or 4 * T)[:T] for _ in range(nseq)]) if pos is None else np.asarray(pos)
    pos = pos.astype(np.int32).reshape(nseq, T)
    n_ctx = n_ctx or 4 * T
    qkv = (g.standard_normal((nseq, T, (heads + 2 * kv) * hd)) * 2).astype(np.float32)
    freq = (1e6 ** (-2.0 * np.arange(rope // 2) / max(rope, 1))).astype(np.float32)
    qw, kw = ((1 + 0.3 * g.standard_normal(hd)).astype(np.float32) if norm else None for _ in range(2))
    dev = lambda a: None if a is None else torch.from_numpy(a).to(gpu)   # noqa: E731
    t = dev(qkv)
    q, k, v = t.split([heads * hd, kv * hd, kv * hd], 2)
    cache = None
    if ctype is not None:
        cache = ops.KvCache.empty(ctype, n_ctx, kv, hd, nseq, gpu)
        for b in (cache.k, cache.v):
            b.view(torch.uint8).fill_(0x5A)      # what no row writes has to stay
    qo, ko = ops.qk_norm_rope_tokens(q, k, v if cache else None, dev(pos), dev(freq), hd, rope_dim=rope, half=half, qw=dev(qw),
                                     kw=dev(kw), mscale=mscale, cache=cache, want_k=True)
    torch.cuda.synchronize()
    assert np.array_equal(t.cpu().numpy(), qkv)          # inputs untouched
    on = ((pos >= 0) & (pos < (n_ctx if cache else 2 ** 31))).reshape(-1)
    rows = qkv.reshape(nseq * T, heads + 2 * kv, hd)
    for got, x, w in ((qo, rows[:, :heads], qw), (ko, rows[:, heads:heads + kv], kw)):
        y, tol = expected(x, w, pos.reshape(-1), freq, rope, half, mscale, 1e-6)
        got = got.cpu().numpy().reshape(y.shape).astype(np.float64)
        assert not got[~on].any()
        assert np.all(np.abs(got - y)[on] <= tol[on] + 1e-30), np.max((np.abs(got - y) / (tol + 1e-30))[on])
    if cache is None:
        return
    k32, v32 = ko.cpu().numpy().reshape(nseq, T, kv, hd), rows[:, heads + kv:].reshape(nseq, T, kv, hd)
    on = on.reshape(nseq, T)
    if ctype == L.F16:
        for b, x in ((cache.k, k32), (cache.v, v32)):
            want = np.full((nseq, n_ctx, kv, hd), 0x5A5A, np.uint16)
            for s in range(nseq):
                want[s, pos[s][on[s]]] = x[s][on[s]].astype(np.float16).view(np.uint16)
            assert np.array_equal(b.cpu().numpy().view(np.uint16).reshape(want.shape), want)
        return
    vals = [x.cpu().numpy().reshape(nseq, n_ctx, kv, hd) for x in ops.kv_values(cache)]
    torch.cuda.synchronize()
    for b, x, val in ((cache.k, k32, vals[0]), (cache.v, v32, vals[1])):
        raw = b.cpu().numpy()
        nb = kv * n_ctx * hd // 2
        want_c = np.full((nseq, kv, n_ctx, hd // 8), 0x5A5A5A5A, np.uint32)
        want_s = np.full((nseq, kv, n_ctx, hd // 32, 2), 0x5A5A, np.uint16)
        for s in range(nseq):
            sel = on[s]
            c, d, m, w = pack(x[s][sel])
            n = sel.sum()
            want_c[s][:, pos[s][sel]] = words(c).reshape(n, kv, hd // 8).transpose(1, 0, 2)
            want_s[s][:, pos[s][sel]] = np.stack([d, m], 1).view(np.uint16).reshape(n, kv, hd // 32, 2).transpose(1, 0, 2, 3)
            assert np.array_equal(val[s][pos[s][sel]], w, equal_nan=True)
        assert np.array_equal(raw[:, :nb].copy().view(np.uint32).reshape(want_c.shape), want_c)
        assert np.array_equal(raw[:, nb:].copy().view(np.uint16).reshape(want_s.shape), want_s)


@pytest.mark.parametrize("ctype", [None, L.F16, L.KV4])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("T,nseq,heads,kv,hd,rope,norm", [
    (1, 1, 32, 8, 128, 128, True), (1, 1, 1, 1, 32, 32, False), (5, 3, 6, 2, 64, 26, True), (3, 2, 4, 4, 256, 256, True),
    (2, 1, 16, 2, 256, 102, False), (7, 1, 3, 1, 96, 2, True), (4, 2, 5, 5, 64, 0, True), (1030, 1, 2, 1, 64, 64, True),
    (300, 4, 3, 2, 128, 128, False)])
def test_rows(gpu, T, nseq, heads, kv, hd, rope, norm, half, ctype):
    print(f"rope rows: {nseq} x {T} heads {heads}/{kv} of {hd} rope {rope} half {half} cache {ctype}", flush=True)
    run_case(gpu, T, nseq, heads, kv, hd, rope, half, norm, ctype, mscale=1.1386)


@pytest.mark.parametrize("hd,kv", [(48, 6), (2, 4), (6, 2), (250, 2)])
def test_odd_heads(gpu, hd, kv):
    for half in (False, True):
        run_case(gpu, 3, 2, 2 * kv, kv, hd, hd, half, True, L.F16 if hd % 8 == 0 else None)


def test_far_positions(gpu):
    """2^31 - 1 radians: fp32 would leave none of the angle, and a double's product with 1 / 2 pi
    2e-7 turns unless its rounding is taken along."""
    run_case(gpu, 5, 1, 2, 1, 64, 64, False, False, None, pos=[0, 1, 131071, 10 ** 7 + 1, 2 ** 31 - 1])


@pytest.mark.parametrize("ctype", [L.F16, L.KV4])
def test_rows_without_a_token(gpu, ctype):
    run_case(gpu, 4, 2, 3, 1, 64, 64, True, True, ctype, pos=[[3, -1, 7, 8], [-2 ** 31, 2 ** 31 - 1, 0, 5]], n_ctx=8)


def test_special_values(gpu):
    """Groups of equal values, ties, tiny and huge ones, infinities and NaN, in the 4-bit cache."""
    import torch
    from ligguf_amd import ops
    rows = [np.zeros(32), np.full(32, -3.25), np.arange(32) % 16, np.arange(32) / 2.0, np.arange(32) * 0.25 - 4,
            np.linspace(-1e38, 1e38, 32), np.linspace(-6e4, 6e4, 32), np.linspace(0, 1e-7, 32), np.full(32, 65504.0),
            np.linspace(2.0 ** -25, 2.0 ** -23, 32), np.linspace(1000, 1000.3, 32), -np.linspace(3, 5, 32) ** 3]
    for bad in (np.nan, np.inf, -np.inf):
        r = np.linspace(-2, 3, 32)
        r[11] = bad
        rows.append(r)
    x = np.array(rows, np.float32)
    n = len(rows)
    t = torch.from_numpy(x).to(gpu).view(n, 1, 32)
    cache = ops.KvCache.empty(ops.KV4, 3, 1, 32, n, gpu)
    pos = torch.ones(n, 1, dtype=torch.int32, device=gpu)
    ops.qk_norm_rope_tokens(None, t, t, pos, None, 32, rope_dim=0, cache=cache)
    k, v = ops.kv_values(cache, 1, 1)
    c, d, m, w = pack(x)
    for got in (k, v):
        assert np.array_equal(got.cpu().numpy().reshape(n, 32), w, equal_nan=True)
    assert np.isfinite(w[:12]).all() and np.isnan(w[12]).all() and np.isfinite(w[13:]).all()
    assert not any(z.any() for z in (ops.kv_values(cache, 0, 1) + ops.kv_values(cache, 2, 1)))
    # a value's distance from what it stands for: half a step of d between codes; at the top 15 times what
    # fp16 rounding took from d (2^-11 of it, or half the least step, 2^-25: a range of 1e-7 has no step at
    # all); the roundings of m and of the result, 2^-11 of the largest or 2^-25 each
    f = np.isfinite(x).all(1) & (np.abs(x).max(1) <= 6e4)
    err = np.abs(w[f].astype(np.float64) - x[f])
    big = np.abs(x[f]).max(1, keepdims=True)
    d = d[f].astype(np.float64)[:, None]
    assert np.all(err <= 0.5 * d + 15 * np.maximum(d * 2.0 ** -11, 2.0 ** -25) + 2 * (2.0 ** -11 * big + 2.0 ** -25))


def test_in_place_and_fused_rows(gpu):
    import torch
    from ligguf_amd import ops
    g = torch.Generator(device=gpu).manual_seed(3)
    qkv = torch.randn(2, 9, 6 * 64, generator=g, device=gpu)
    pos = torch.arange(18, dtype=torch.int32, device=gpu).view(2, 9)
    freq = ops.rope_table(64, 1e4)[0].to(gpu)
    q, k, v = qkv.split([256, 64, 64], 2)
    for half in (False, True):
        a = ops.qk_norm_rope_tokens(q.contiguous(), k.contiguous(), None, pos, freq, 64, half=half, want_k=True)
        f = qkv.clone()
        fq, fk, fv = f.split([256, 64, 64], 2)
        ops.qk_norm_rope_tokens(fq, fk, None, pos, freq, 64, half=half, q_out=fq, k_out=fk)
        assert torch.equal(fq, a[0]) and torch.equal(fk, a[1]) and torch.equal(fv, v)


@pytest.mark.parametrize("ctype", [L.F16, L.KV4])
def test_offsets_past_32_bits(gpu, ctype):
    """The last row of a cache of more than 4 GiB (of keys; as many of values)."""
    import torch
    from ligguf_amd import ops
    kv, hd = 8, 256
    n_ctx = (2 ** 32 + 2 ** 28) // (kv * hd * 2 if ctype == L.F16 else kv * hd * 5 // 8)
    cache = ops.KvCache.empty(ctype, n_ctx, kv, hd, 1, gpu)
    x = torch.randn(1, 2, kv * hd, device=gpu)
    pos = torch.tensor([[n_ctx - 1, n_ctx // 2]], dtype=torch.int32, device=gpu)
    ops.qk_norm_rope_tokens(None, x, x, pos, None, hd, rope_dim=0, cache=cache)
    for p, row in ((n_ctx - 1, 0), (n_ctx // 2, 1)):
        want = x[0, row].half().cpu().numpy() if ctype == L.F16 else pack(x[0, row].cpu().numpy())[3]
        for t in ((cache.k[0, p], cache.v[0, p]) if ctype == L.F16 else ops.kv_values(cache, p, 1)):
            assert np.array_equal(t.cpu().numpy().reshape(-1), want)
    some = (cache.k.view(torch.int64) != 0).sum() + (cache.v.view(torch.int64) != 0).sum()
    row = kv * hd * (2 if ctype == L.F16 else 0.625) / 8
    assert 0.9 * 4 * row <= int(some) <= 4 * row       # the two rows' words and no others
    del cache
    torch.cuda.empty_cache()


def test_captured_call_follows_positions(gpu):
    import torch
    from ligguf_amd import ops
    kv, hd = 2, 64
    x = torch.randn(3, 1, 4 * kv * hd, device=gpu)
    q, k, v = x.split([2 * kv * hd, kv * hd, kv * hd], 2)
    freq = ops.rope_table(hd, 1e4)[0].to(gpu)
    pos = torch.zeros(3, 1, dtype=torch.int32, device=gpu)
    caches = [ops.KvCache.empty(ops.KV4, 40, kv, hd, 3, gpu) for _ in range(2)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        ops.qk_norm_rope_tokens(q, k, v, pos, freq, hd, cache=caches[0])
        s.synchronize()
        with torch.cuda.graph(graph, stream=s):
            out = ops.qk_norm_rope_tokens(q, k, v, pos, freq, hd, cache=caches[0])[0]
    torch.cuda.synchronize()
    for i in range(6):
        pos.copy_(torch.tensor([[i], [39 - i], [-1 if i == 3 else 2 * i]], dtype=torch.int32))
        x.normal_()
        graph.replay()
        want = ops.qk_norm_rope_tokens(q, k, v, pos, freq, hd, cache=caches[1])[0]
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    # (row 0 of the first cache also has the warm-up's and the capture's zero position)
    a, b = (torch.stack(ops.kv_values(c)) for c in caches)
    assert torch.equal(a[:, :, 1:], b[:, :, 1:]) and torch.equal(a[:, 0], b[:, 0])


def test_other_stream(gpu):
    import torch
    from ligguf_amd import ops
    x = torch.randn(1, 2000, 8 * 128, device=gpu)
    pos = torch.arange(2000, dtype=torch.int32, device=gpu).view(1, -1)
    freq = ops.rope_table(128, 1e4)[0].to(gpu)
    want = ops.qk_norm_rope_tokens(x, x, None, pos, freq, 128, want_k=True)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        y = x * 1.0
        got = ops.qk_norm_rope_tokens(y, y, None, pos, freq, 128, want_k=True)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_one_norm_only_and_weights_on_any_boundary(gpu):
    import torch
    from ligguf_amd import ops
    g = torch.Generator(device=gpu).manual_seed(8)
    q, k = torch.randn(2, 7, 4 * 64, generator=g, device=gpu), torch.randn(2, 7, 2 * 64, generator=g, device=gpu)
    w = torch.randn(65, generator=g, device=gpu)
    pos = torch.arange(14, dtype=torch.int32, device=gpu).view(2, 7)
    freq = ops.rope_table(64, 1e4)[0].to(gpu)
    plain = ops.qk_norm_rope_tokens(q, k, None, pos, freq, 64, want_k=True)
    both = ops.qk_norm_rope_tokens(q, k, None, pos, freq, 64, qw=w[:64].contiguous(), kw=w[1:].clone(), want_k=True)
    a = ops.qk_norm_rope_tokens(q, k, None, pos, freq, 64, qw=w[:64], want_k=True)
    b = ops.qk_norm_rope_tokens(q, k, None, pos, freq, 64, kw=w[1:].clone(), want_k=True)
    assert torch.equal(a[0], both[0]) and torch.equal(a[1], plain[1])
    assert torch.equal(b[0], plain[0]) and torch.equal(b[1], both[1])
    # weights four bytes off a 16-byte boundary take the one-pair form: sums in another order
    off = ops.qk_norm_rope_tokens(q, k, None, pos, freq, 64, qw=w[:64], kw=w[1:], want_k=True)
    for x, y in zip(off, both):
        assert float((x - y).abs().max()) <= 40 * U * float(y.abs().max())


def test_no_rows(gpu):
    import torch
    from ligguf_amd import ops
    for shape in ((0, 3), (2, 0)):
        x, pos = torch.zeros(*shape, 128, device=gpu), torch.zeros(shape, dtype=torch.int32, device=gpu)
        q, k = ops.qk_norm_rope_tokens(x, x, None, pos, torch.zeros(32, device=gpu), 64, want_k=True)
        assert q.shape == k.shape == x.shape
    cache = ops.KvCache.empty(ops.F16, 4, 2, 64, 2, gpu)
    pos = torch.zeros(2, 0, dtype=torch.int32, device=gpu)
    assert ops.attention_cache(torch.zeros(2, 0, 128, device=gpu), cache, pos).shape == (2, 0, 128)


def test_python_refusals(gpu):
    import torch
    from ligguf_amd import ops
    x = torch.zeros(1, 2, 128, device=gpu)
    pos = torch.zeros(1, 2, dtype=torch.int32, device=gpu)
    freq = torch.zeros(32, device=gpu)
    ok = dict(q=x, k=x, v=None, pos=pos, freq=freq, head_dim=64, want_k=True)
    ops.qk_norm_rope_tokens(**ok)
    cache = ops.KvCache.empty(ops.F16, 4, 2, 64, 1, gpu)
    for bad in (dict(q=x.half()), dict(q=x.cpu()), dict(q=x[:, :1]), dict(k=x[..., ::2]), dict(pos=pos.long()), dict(pos=pos.cpu()),
                dict(pos=pos[0]), dict(head_dim=60), dict(head_dim=0), dict(freq=freq[:31]), dict(freq=freq.double()), dict(qw=freq),
                dict(rope_dim=128), dict(rope_dim=-2), dict(cache=cache), dict(k_out=x[..., :64]),
                dict(q=torch.zeros(1, 2, 130, device=gpu)[..., :128]), dict(q=torch.zeros(2, 1, 128, device=gpu).transpose(0, 1)[:, :, 1:])):
        with pytest.raises(L.LgError):
            ops.qk_norm_rope_tokens(**{**ok, **bad})
    for bad in (dict(type=L.F32), dict(head_dim=32), dict(n_ctx=5), dict(type=ops.KV4), dict(k=cache.k[:, :, ::2]), dict(v=cache.v.cpu())):
        with pytest.raises(L.LgError):
            ops.KvCache(**{**dict(k=cache.k, v=cache.v, n_kv_heads=2, head_dim=64, n_ctx=4), **bad})
    with pytest.raises(L.LgError):
        ops.kv_values(cache)
    four = ops.KvCache.empty(ops.KV4, 4, 2, 64, 1, gpu)
    for a in ((-1, 1), (0, 5), (3, 2), (5, None)):
        with pytest.raises(L.LgError):
            ops.kv_values(four, *a)


def test_few_rows_of_more_heads_than_a_grid_takes(gpu):
    """511 rows of 65536 query, key and value heads of two values: a workgroup per round of heads would be 25
    million of them."""
    import torch
    from ligguf_amd import ops
    n, heads = 511, 65536
    g = torch.Generator(device=gpu).manual_seed(5)
    q, k, v = (torch.randn(1, n, 2 * heads, generator=g, device=gpu) for _ in range(3))
    pos = torch.arange(n, dtype=torch.int32, device=gpu)[None]
    cache = ops.KvCache.empty(ops.F16, n, heads, 2, 1, gpu)
    freq = torch.full((1,), 0.1, device=gpu)
    qo, ko = ops.qk_norm_rope_tokens(q, k, v, pos, freq, 2, cache=cache, want_k=True)
    for x, y in ((q, qo), (k, ko)):
        for t in (0, 300, n - 1):
            want, tol = expected(x[0, t].cpu().numpy().reshape(1, heads, 2), None, np.array([t]), freq.cpu().numpy(), 2, False, 1.0, 1e-6)
            assert np.all(np.abs(y[0, t].cpu().numpy().reshape(want.shape) - want) <= tol + 1e-30)
    assert torch.equal(cache.k, ko.half()) and torch.equal(cache.v, v.half())
    del q, k, v, qo, ko, x, y, cache
    torch.cuda.empty_cache()


def test_reading_back_past_31_bits_of_words(gpu):
    """More than 2^31 words of codes in one call, rows on both sides of the border (34 GB each of keys
    and values; the cache's keys and values are the same memory)."""
    import torch
    from ligguf_amd import ops
    kv, hd, n = 8, 256, (1 << 23) + 40
    if torch.cuda.mem_get_info(gpu)[0] < 100 << 30:
        pytest.skip("needs 80 GB of device memory")
    x = torch.randn(1, 6, kv * hd, generator=torch.Generator(device=gpu).manual_seed(6), device=gpu)
    mem = torch.zeros(1, L.load().lg_kv_bytes(L.KV4, n, kv, hd), dtype=torch.uint8, device=gpu)
    cache = ops.KvCache(mem, mem, kv, hd, ops.KV4, n)
    at = [0, 1, (1 << 22) + 3, (1 << 23) - 1, 1 << 23, n - 1]
    pos = torch.tensor([at], dtype=torch.int32, device=gpu)
    ops.qk_norm_rope_tokens(None, x, x, pos, None, hd, rope_dim=0, cache=cache)
    out = ops.kv_values(cache)
    want = pack(x.cpu().numpy())[3].reshape(6, -1)
    for t in out:
        for i, p in enumerate(at):
            assert np.array_equal(t[0, p].cpu().numpy(), want[i])
        for p in (2, (1 << 22) + 2, (1 << 23) - 2, (1 << 23) + 1, n - 2):
            assert not t[0, p].any()
    del out, t, mem, cache
    torch.cuda.empty_cache()


def test_rotation_by_a_scaled_angle_rounds_once(gpu):
    """The pair (1, 0) becomes mscale (cos, sin) itself: the factors, rounded to fp32 once."""
    import torch
    from ligguf_amd import ops
    hd, n = 128, 500
    freq, mscale = ops.rope_table(hd, 1e4, L.ROPE_YARN, 4.0, 4096, 32.0, 1.0)
    assert mscale != 1.0
    pos = torch.arange(0, 37 * n, 37, dtype=torch.int32, device=gpu)[None]
    x = torch.zeros(1, n, hd, device=gpu)
    x[..., ::2] = 1.0
    got = ops.qk_norm_rope_tokens(None, x, None, pos, freq.to(gpu), hd, mscale=mscale, want_k=True)[1]
    got = got.cpu().numpy().reshape(n, hd // 2, 2).astype(np.float64)
    ang = pos.cpu().numpy().reshape(-1, 1).astype(np.float64) * freq.numpy().astype(np.float64)
    for e, f in enumerate((np.cos, np.sin)):
        want = f(ang) * float(np.float32(mscale))
        # half a step, and what the angle's rounding to a double (2 10^4 radians: 2e-12) leaves near a border
        assert np.all(np.abs(got[..., e] - want) <= np.spacing(np.abs(want).astype(np.float32)) / 2.0 + 1e-11)


def test_padded_rows_of_odd_widths(gpu):
    """Rows of 18 and 6 values, 16-byte aligned by padding: outputs made by the call as well as given ones."""
    import torch
    from ligguf_amd import ops
    g = np.random.default_rng(2)
    buf = torch.from_numpy(g.standard_normal((2, 5, 28)).astype(np.float32)).to(gpu)
    q, k = buf[..., :18], buf[..., 20:26]
    pos = torch.arange(10, dtype=torch.int32, device=gpu).view(2, 5)
    freq = ops.rope_table(6, 1e4)[0].to(gpu)
    want = [torch.zeros(2, 5, n, device=gpu) for n in (20, 8)]
    ops.qk_norm_rope_tokens(q, k, None, pos, freq, 6, q_out=want[0][..., :18], k_out=want[1][..., :6])
    y, tol = expected(q.cpu().numpy().reshape(10, 3, 6), None, pos.cpu().numpy().reshape(-1), freq.cpu().numpy(), 6, False, 1.0, 1e-6)
    assert np.all(np.abs(want[0][..., :18].cpu().numpy().reshape(y.shape) - y) <= tol + 1e-30)
    got = ops.qk_norm_rope_tokens(q, k, None, pos, freq, 6, want_k=True)
    assert got[0].shape == q.shape and got[1].shape == k.shape
    assert torch.equal(got[0], want[0][..., :18]) and torch.equal(got[1], want[1][..., :6])
