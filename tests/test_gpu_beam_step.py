"""A whole step of beam search -- append, attention, selection, reordering, over two layers --
captured once and replayed, against the same step run call by call."""
import pytest

from ligguf_amd import lib as L

pytestmark = pytest.mark.gpu
G, B, HEADS, KV, HD, PAGE, MOST, VOCAB, LAYERS = 3, 4, 8, 2, 64, 16, 6, 5000, 2


class State:
    def __init__(self, gpu, ctype, length):
        import torch
        from ligguf_amd import ops
        n = G * B * MOST
        self.table = torch.arange(n, dtype=torch.int32, device=gpu).view(G * B, MOST)
        full = min(length) // PAGE                    # pages that a group's beams hold together
        self.table.view(G, B, MOST)[:, :, :full] = self.table.view(G, B, MOST)[:, :1, :full].clone()
        self.caches = [ops.PagedKvCache.empty(ctype, n, PAGE, KV, HD, self.table) for _ in range(LAYERS)]
        self.layers = ops.PagedLayers(self.caches)
        g = torch.Generator(device=gpu).manual_seed(8)
        for c in self.caches:                         # the prompts' keys and values
            x = torch.randn(G * B, MOST * PAGE, 2 * KV * HD, generator=g, device=gpu)
            every = torch.arange(MOST * PAGE, dtype=torch.int32, device=gpu)[None].repeat(G * B, 1)
            flat = torch.arange(n, dtype=torch.int32, device=gpu).view(G * B, MOST)
            k, v = x.split(KV * HD, 2)
            own = ops.PagedKvCache(c.k, c.v, flat, KV, HD, ctype, PAGE)
            ops.qk_norm_rope_tokens(None, k, v, every, torch.ones(HD // 2, device=gpu), HD, cache=own)
        self.prefix = torch.full((G,), full * PAGE, dtype=torch.int32, device=gpu)
        self.length = torch.tensor(length, dtype=torch.int32, device=gpu)
        self.pos = self.length.repeat_interleave(B)[:, None].contiguous()
        self.scores = torch.zeros(G, B, device=gpu)
        self.done = torch.zeros(G, B, dtype=torch.int32, device=gpu)
        self.qkv = torch.zeros(LAYERS, G * B, 1, (HEADS + 2 * KV) * HD, device=gpu)
        self.logits = torch.zeros(G, B, VOCAB, device=gpu)
        self.freq = ops.rope_table(HD, 1e4)[0].to(gpu)
        self.out = torch.zeros(LAYERS, G * B, 1, HEADS * HD, device=gpu)

    def step(self):
        from ligguf_amd import ops
        for l, c in enumerate(self.caches):
            q, k, v = self.qkv[l].split([HEADS * HD, KV * HD, KV * HD], 2)
            q, _ = ops.qk_norm_rope_tokens(q, k, v, self.pos, self.freq, HD, cache=c)
            ops.attention_paged(q, c, self.pos, prefix=self.prefix, max_prefix=MOST * PAGE, out=self.out[l])
        r = ops.beam_select(self.logits, self.scores, B, done=self.done, end=2)
        self.length.add_(1)
        self.pos.add_(1)
        ops.beam_reorder(self.layers, r.parent, self.length)
        self.scores.copy_(r.score)
        self.done.copy_(r.token == 2)
        self.choice = r

    def all(self):
        return [self.out, self.table, self.scores, self.done, *self.choice] + [x for c in self.caches for x in (c.k, c.v)]


@pytest.mark.parametrize("ctype", [L.F16, L.KV4])
def test_captured_step_equals_the_calls(gpu, ctype):
    import torch
    length = [37, 48, 33]
    a, b, warm = (State(gpu, ctype, length) for _ in range(3))
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        warm.step()
        s.synchronize()
        with torch.cuda.graph(graph, stream=s):
            a.step()
    torch.cuda.synchronize()
    g = torch.Generator(device=gpu).manual_seed(9)
    for turn in range(30):
        qkv = torch.randn(a.qkv.shape, generator=g, device=gpu)
        logits = torch.randn(a.logits.shape, generator=g, device=gpu) * 3
        logits[:, :, 2] += 3.0 * (turn % 5 == 4)       # some beams end now and then
        for x in (a, b):
            x.qkv.copy_(qkv)
            x.logits.copy_(logits)
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        for i, (x, y) in enumerate(zip(a.all(), b.all())):
            same = torch.equal(x.view(torch.uint8), y.view(torch.uint8))
            assert same, (turn, i)
    assert b.table.unique().numel() > G and int(b.length.max()) == 78 and b.out.isfinite().all()
