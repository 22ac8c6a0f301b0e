"""The many-token calls in a row, as a serving loop makes them: rotation and cache
write, attention, the output head's log probabilities -- prompts, then single
tokens, eager and captured, over both caches; and next to a context."""
import math

import numpy as np
import pytest

from ligguf_amd import lib as L
from test_gpu_cattn import reference
from test_gpu_kvrope import expected

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HEADS, KV, HD, VOCAB = 8, 2, 64, 700


class Toy:
    """One attention layer between an embedding and an output head, two conversations."""

    def __init__(self, gpu, ctype, window, sinks, n_ctx=260):
        import torch
        from ligguf_amd import ops
        g = torch.Generator(device=gpu).manual_seed(11)

        def w(*shape, s):
            return torch.randn(*shape, generator=g, device=gpu) * s
        self.embd, self.qkv = w(VOCAB, 128, s=1.0), w(128, (HEADS + 2 * KV) * HD, s=0.12)
        self.out, self.qw, self.kw = w(HEADS * HD, VOCAB, s=0.3), 1 + w(HD, s=0.2), 1 + w(HD, s=0.2)
        self.freq, self.mscale = ops.rope_table(HD, 1e4, L.ROPE_YARN, 4.0, 64, 32.0, 1.0)
        self.freq, self.window, self.sinks = self.freq.to(gpu), window, sinks
        self.cache = ops.KvCache.empty(ctype, n_ctx, KV, HD, 2, gpu)

    def step(self, toks, pos):
        """(rotated queries, attention, logits, log probabilities of the next tokens) of toks [2, n] at pos [2, n]."""
        from ligguf_amd import ops
        rows = self.embd[toks.long()] @ self.qkv
        q, k, v = rows.split([HEADS * HD, KV * HD, KV * HD], 2)
        q, _ = ops.qk_norm_rope_tokens(q, k, v, pos, self.freq, HD, half=True, qw=self.qw, kw=self.kw, mscale=self.mscale,
                                       cache=self.cache)
        att = ops.attention_cache(q, self.cache, pos, window=self.window, sinks=self.sinks)
        logits = att.flatten(0, 1) @ self.out
        return rows, q, att, logits, ops.logprobs(logits, toks.flatten(), top=5)

    def values(self):
        from ligguf_amd import ops
        kv = (self.cache.k, self.cache.v) if self.cache.type == L.F16 else ops.kv_values(self.cache)
        return [t.cpu().numpy().astype(np.float64).reshape(2, -1, KV, HD) for t in kv]


def check(toy, pos, got):
    rows, q, att, logits, lp = got
    p, n = pos.cpu().numpy(), pos.shape[1]
    on = (p >= 0).reshape(-1)
    x = rows.cpu().numpy().reshape(2 * n, HEADS + 2 * KV, HD)
    f = toy.freq.cpu().numpy()
    y, tol = expected(x[:, :HEADS], toy.qw.cpu().numpy(), p.reshape(-1), f, HD, True, toy.mscale, 1e-6)
    assert np.all(np.abs(q.cpu().numpy().reshape(y.shape) - y)[on] <= tol[on] + 1e-30)
    K, V = toy.values()
    want, tol = reference(q.cpu().numpy().reshape(2, n, HEADS, HD), K, V, p, toy.window, toy.sinks, toy.cache.n_ctx - 1)
    assert np.all(np.abs(att.cpu().numpy().reshape(want.shape) - want) <= tol)
    z = logits.cpu().numpy().astype(np.float64)
    z = z - z.max(1, keepdims=True)
    ref = z - np.log(np.exp(z).sum(1, keepdims=True))
    ids = np.argsort(-z, axis=1, kind="stable")[:, :5]
    assert np.array_equal(lp.top_id.cpu().numpy(), ids)
    near = (200 + 4 * np.abs(z).max()) * U        # as in the calls' own tests
    assert np.max(np.abs(lp.top_logprob.cpu().numpy() - np.take_along_axis(ref, ids, 1))) <= near
    assert np.max(np.abs(lp.entropy.cpu().numpy() + (np.exp(ref) * ref).sum(1))) <= near * (1 + math.log(VOCAB))


@pytest.mark.parametrize("ctype", [L.F16, L.KV4])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
def test_prompt_then_tokens(gpu, ctype, window, sinks):
    """Prompts of 150 and 97 tokens in one padded call, then single tokens; the same tokens one by
    one give the same cache and, up to the order of sums, the same attention."""
    import torch
    toy, one = Toy(gpu, ctype, window, sinks), Toy(gpu, ctype, window, sinks)
    toks = torch.randint(0, VOCAB, (2, 150), generator=torch.Generator().manual_seed(5)).int().to(gpu)
    pos = torch.arange(150, dtype=torch.int32, device=gpu).repeat(2, 1)
    pos[1, 97:] = -1
    got = toy.step(toks, pos)
    check(toy, pos, got)
    assert not got[2][1, 97:].any()
    for t in range(150):
        r = one.step(toks[:, t:t + 1].contiguous(), pos[:, t:t + 1].contiguous())
        scale = float(got[2][:, t].abs().max())
        # torch's products for 1 and 150 rows differ in the last bits, so an fp16 key or value may round the
        # other way (2^-11 of it): a score moves by 2^-11 sum |q k| / sqrt(hd), under 3.5e-3 here, a weight by as
        # much of itself, a value by 5e-4; a 4-bit code may move by a whole step
        if ctype == L.F16:
            assert float((r[2][:, 0] - got[2][:, t]).abs().max()) <= 4e-3 * scale
    for i in range(12):
        p = torch.tensor([[150 + i], [97 + i]], dtype=torch.int32, device=gpu)
        t = toks[:, i:i + 1].contiguous()
        check(toy, p, toy.step(t, p))


@pytest.mark.parametrize("ctype", [L.F16, L.KV4])
def test_captured_generation(gpu, ctype):
    """A captured step that takes its own greedy tokens and moves its positions on, against the
    same steps eagerly."""
    import torch

    def loop(toy, toks, pos):
        r = toy.step(toks, pos)
        toks.copy_(r[4].top_id[:, :1])
        pos.add_(1)
        return r
    a, b = Toy(gpu, ctype, 30, 2), Toy(gpu, ctype, 30, 2)
    state = [(torch.tensor([[3], [9]], dtype=torch.int32, device=gpu), torch.tensor([[0], [5]], dtype=torch.int32, device=gpu))
             for _ in range(2)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        loop(a, *state[0])
        s.synchronize()
        with torch.cuda.graph(graph, stream=s):
            r = loop(a, *state[0])
    torch.cuda.synchronize()
    loop(b, *state[1])
    for i in range(60):
        graph.replay()
        want = loop(b, *state[1])
        torch.cuda.synchronize()
        assert torch.equal(state[0][0], state[1][0]) and torch.equal(state[0][1], state[1][1])
        assert torch.equal(r[2], want[2]) and all(torch.equal(x, y) for x, y in zip(r[4], want[4]))


def test_two_streams_with_workspaces_of_their_own(gpu):
    """Calls that overlap on two streams, each with its workspace, as often as not at once."""
    import torch
    from ligguf_amd import ops
    g = torch.Generator(device=gpu).manual_seed(1)
    cache = ops.KvCache.empty(ops.F16, 6000, KV, HD, 1, gpu)
    cache.k.normal_(generator=g)
    cache.v.normal_(generator=g)
    q = [torch.randn(1, n, HEADS * HD, generator=g, device=gpu) for n in (1, 40)]
    pos = [torch.arange(6000 - n, 6000, dtype=torch.int32, device=gpu).view(1, -1) for n in (1, 40)]
    want = [ops.attention_cache(a, cache, p) for a, p in zip(q, pos)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(ops.attention_cache(q[i], cache, pos[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


def test_over_a_contexts_logits(gpu):
    """Engine.logprobs: a context's own logits, step after step."""
    from ligguf_amd.model import TINY, Engine, HostModel
    eng = Engine(0)
    with pytest.raises(L.LgError):
        eng.logprobs(1)
    eng.load(HostModel.synthetic(TINY))
    for i, tok in enumerate((5, 900, 17)):
        lg = eng.decode(tok, i).astype(np.float64)
        z = lg - lg.max()
        ref = z - math.log(np.exp(z).sum())
        near = (200 + 4 * np.abs(z).max()) * U
        lp, ent, alts = eng.logprobs(77, top=8)
        order = np.argsort(-lg, kind="stable")[:8]
        assert [a[0] for a in alts] == order.tolist() and alts[0][0] == eng.argmax()
        assert abs(lp - ref[77]) <= near and abs(ent + (np.exp(ref) * ref).sum()) <= near * (1 + math.log(lg.size))
        assert max(abs(a[1] - ref[a[0]]) for a in alts) <= near
    assert eng.logprobs(77)[2] == []
    eng.close()


@pytest.mark.parametrize("ctype", [L.F16, L.KV4])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
def test_tokens_one_by_one(gpu, ctype, window, sinks):
    """Every step of a conversation of single tokens against the formulas over its own cache, and that
    cache against a prompt's.  The rows of both come from torch products of another shape, which differ in
    the last bits: an fp16 value is off by one rounding, a 4-bit one by one code (a step of d, a fifteenth
    of its group's range) and the roundings of d at 15 and of m."""
    import torch
    toy, one = Toy(gpu, ctype, window, sinks), Toy(gpu, ctype, window, sinks)
    toks = torch.randint(0, VOCAB, (2, 150), generator=torch.Generator().manual_seed(5)).int().to(gpu)
    pos = torch.arange(150, dtype=torch.int32, device=gpu).repeat(2, 1)
    pos[1, 97:] = -1
    toy.step(toks, pos)
    for t in range(150):
        p = pos[:, t:t + 1].contiguous()
        check(one, p, one.step(toks[:, t:t + 1].contiguous(), p))
    for a, b in zip(toy.values(), one.values()):
        assert not a[0, 150:].any() and not a[1, 97:].any() and not b[0, 150:].any() and not b[1, 97:].any()
        x, y = (z.reshape(2, -1, KV, HD // 32, 32) for z in (a, b))
        top = np.abs(y).max(-1, keepdims=True)
        if ctype == L.F16:
            near = np.abs(y) * 2.0 ** -10 + 2.0 ** -24
        else:
            near = (y.max(-1, keepdims=True) - y.min(-1, keepdims=True)) / 15 * (1 + 16 * 2.0 ** -10) + 3 * 2.0 ** -10 * top + 2.0 ** -20
        # (the products' own difference, 128 terms of fp32, is far below)
        assert np.all(np.abs(x - y) <= near + 1e-5 * top)
