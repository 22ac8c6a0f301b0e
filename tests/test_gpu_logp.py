"""lg_logprobs against log softmax in 64 bits: given tokens, entropy, top entries in
order, ties, infinities and NaN, odd sizes and strides, captured calls, refusals."""
import numpy as np
import pytest

from ligguf_amd import lib as L

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def reference(x):
    y = x.astype(np.float64)
    m = y.max(1, keepdims=True)
    with np.errstate(over="ignore"):
        lz = np.log(np.exp(y - m).sum(1, keepdims=True))
    lp = y - m - lz
    p = np.exp(lp)
    ent = -np.where(p > 0, p * np.where(p > 0, lp, 0), 0).sum(1)
    return lp, ent


def check(gpu, x, toks, top, wide=None):
    import torch
    from ligguf_amd import ops
    rows, vocab = x.shape
    t = torch.from_numpy(x).to(gpu)
    if wide is not None:
        big = torch.full((rows, wide), 1e30, device=gpu)
        big[:, 1:1 + vocab] = t
        t = big[:, 1:1 + vocab]
    r = ops.logprobs(t, None if toks is None else torch.from_numpy(toks.astype(np.int32)).to(gpu), top=top)
    lp, ent = reference(x)
    # log z: the terms' exponents (|x - m| U and 2 U of the exp), vocab additions at worst in
    # lanes and joins (a row's parts are 64 long or shorter per lane, 20 levels above them: 100 covers it),
    # the logarithm's 2 U; x - m and the difference one U each of their sizes
    spread = np.abs(np.where(np.isfinite(x), x, 0)).max(1).astype(np.float64) * 2
    tol = (100 + 2 * spread) * U + 1e-37
    if toks is not None:
        at = lp[np.arange(rows), toks]
        assert np.all(np.abs(r.logprob.cpu().numpy() - at) <= tol + 4 * U * np.abs(at))
    # entropy = log z - h / z, both sums of terms of one sign
    e = r.entropy.cpu().numpy()
    assert np.all(np.abs(e - ent) <= tol + (200 + 4 * spread) * U * (np.abs(ent) + 1))
    if top:
        ids = r.top_id.cpu().numpy()
        want = np.stack([np.lexsort((np.arange(vocab), -row))[:top] for row in x.astype(np.float64)])
        assert np.array_equal(ids, want)
        at = np.take_along_axis(lp, want, 1)
        got = r.top_logprob.cpu().numpy()
        fine = np.isfinite(at)
        assert np.array_equal(got[~fine], at[~fine])
        assert np.all(np.abs(got[fine] - at[fine]) <= (tol[:, None] + 4 * U * np.where(fine, np.abs(at), 0))[fine])
    else:
        assert r.top_id is None and r.top_logprob is None
    return r


@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 2), (3, 31), (2, 64), (1, 1000), (5, 1023), (2, 2049), (1, 32000), (40, 5000),
                                        (3, 50257), (1, 151936), (300, 4097), (700, 600), (3, 16389),
                                        (520, 9001), (2, 40001)])
@pytest.mark.parametrize("top", [0, 1, 5, 20, 32])
def test_rows(gpu, rows, vocab, top):
    print(f"logprobs: {rows} x {vocab} top {top}", flush=True)
    g = np.random.default_rng(rows + vocab + top)
    x = (g.standard_normal((rows, vocab)) * 3).astype(np.float32)
    top = min(top, vocab)
    check(gpu, x, g.integers(0, vocab, rows), top)
    check(gpu, x, None, top, wide=vocab + 5)      # rows on 4-byte boundaries, between other values


@pytest.mark.parametrize("vocab", [40, 3000, 40000])
def test_orders_that_fill_the_lists(gpu, vocab):
    """Equal rows, ascending and descending ones, few distinct values, the largest in one place."""
    g = np.random.default_rng(vocab)
    i = np.arange(vocab, dtype=np.float32)
    rows = [np.zeros(vocab), np.full(vocab, -7.5), i / vocab, -i / vocab, np.floor(4 * g.random(vocab)), np.where(i % 2, 0.0, -0.0),
            np.where((i >= vocab // 2) & (i < vocab // 2 + 36), 5 + (i % 3), 0), np.where(i % 64 == 7, 3 + i / vocab, 0),
            np.where(i == vocab - 1, 50, i % 5), np.repeat(g.random(vocab // 4 + 1), 4)[:vocab]]
    x = np.stack(rows).astype(np.float32)
    for top in (1, 32):
        check(gpu, x, g.integers(0, vocab, len(rows)), top)


@pytest.mark.parametrize("vocab", [70, 20000])
def test_infinities(gpu, vocab):
    g = np.random.default_rng(1)
    x = (g.standard_normal((6, vocab)) * 2).astype(np.float32)
    x[0, ::2] = -np.inf                      # half of them masked
    x[1, 1:] = -np.inf                       # one left: certain
    x[2] = -np.inf
    x[2, vocab // 2:vocab // 2 + 40] = 1.0   # whole parts of the row masked
    x[3, :] = np.finfo(np.float32).min       # the type's lowest value everywhere: uniform
    x[4, 5:] = np.finfo(np.float32).min
    x[5] *= 1e4
    r = check(gpu, x, np.array([1, 0, vocab // 2, 3, 2, 9]), 32)
    assert r.logprob[1] == 0 and r.entropy[1] == 0


def test_rows_without_probabilities(gpu):
    import torch
    from ligguf_amd import ops
    for vocab in (50, 30000):
        x = torch.zeros(4, vocab, device=gpu)
        x[0, 7] = float("nan")
        x[1, 9] = float("inf")
        x[2] = float("-inf")
        toks = torch.full((4,), 3, dtype=torch.int32, device=gpu)
        r = ops.logprobs(x, toks, top=3)
        assert torch.isnan(r.logprob[:3]).all() and torch.isnan(r.entropy[:3]).all() and torch.isnan(r.top_logprob[:3]).all()
        assert torch.isfinite(r.logprob[3]) and torch.isfinite(r.top_logprob[3]).all()
        assert r.top_id.tolist() == [[7, 0, 1], [9, 0, 1], [0, 1, 2], [0, 1, 2]]


def test_tokens_that_are_no_ids(gpu):
    import torch
    from ligguf_amd import ops
    x = torch.randn(4, 99, device=gpu)
    toks = torch.tensor([-1, 99, 2 ** 31 - 1, 98], dtype=torch.int32, device=gpu)
    r = ops.logprobs(x, toks)
    assert torch.isnan(r.logprob[:3]).all() and torch.isfinite(r.logprob[3])


def test_offsets_past_32_bits(gpu):
    """A row that begins beyond 2^32 bytes, and beyond 2^31 values."""
    import torch
    from ligguf_amd import ops
    stride = 2 ** 30 + 2 ** 29 + 4
    buf = torch.full((2 * stride + 1000,), float("nan"), device=gpu)
    x = torch.randn(3, 1000, device=gpu)
    t = buf.as_strided((3, 1000), (stride, 1))
    t.copy_(x)
    toks = torch.tensor([5, 6, 7], dtype=torch.int32, device=gpu)
    a, b = ops.logprobs(t, toks, top=4), ops.logprobs(x, toks, top=4)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    del buf, t
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,vocab", [(1, 40000), (200, 3000)])
def test_captured_calls(gpu, rows, vocab):
    import torch
    from ligguf_amd import ops
    x, toks = torch.randn(rows, vocab, device=gpu), torch.zeros(rows, dtype=torch.int32, device=gpu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        ops.logprobs(x, toks, top=7)
        s.synchronize()
        with torch.cuda.graph(graph, stream=s):
            r = ops.logprobs(x, toks, top=7)
    torch.cuda.synchronize()
    for i in range(5):
        x.normal_()
        toks.random_(0, vocab)
        graph.replay()
        want = ops.logprobs(x, toks, top=7)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(r, want))


@pytest.mark.parametrize("rows,vocab", [(1, 31000), (60, 3000), (2, 151936), (300, 5000)])
def test_same_results_every_time(gpu, rows, vocab):
    """Which thread writes an entry depends on the order of LDS atomics; what it writes does not."""
    import torch
    from ligguf_amd import ops
    x, toks = torch.randn(rows, vocab, device=gpu), torch.zeros(rows, dtype=torch.int32, device=gpu)
    a = ops.logprobs(x, toks, top=20)
    for _ in range(20):
        assert all(torch.equal(p, q) for p, q in zip(ops.logprobs(x, toks, top=20), a))


def test_python_refusals(gpu):
    import torch
    from ligguf_amd import ops
    x, toks = torch.zeros(3, 50, device=gpu), torch.zeros(3, dtype=torch.int32, device=gpu)
    ops.logprobs(x, toks, top=32)
    assert ops.logprobs(x[:0], toks[:0], top=3).top_id.shape == (0, 3)
    for a in ((x.half(), toks), (x.cpu(), toks), (x[0], toks), (x[:, ::2], toks), (x, toks.long()), (x, toks[:2]), (x, toks.cpu()),
              (x, toks, -1), (x, toks, 33), (x[:, :4], toks, 5), (x[:1].expand(3, 50), toks)):
        with pytest.raises(L.LgError):
            ops.logprobs(*a)
