"""lg_beam_reorder of pages that several workgroups copy, and lg_beam_select where scores,
vocabularies and parts lie at their borders."""
import numpy as np
import pytest

from ligguf_amd import lib as L
from test_gpu_beam import check, moved

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ctype", [L.F16, L.KV4])
@pytest.mark.parametrize("page,kv,hd,beams", [(128, 8, 128, 3), (1024, 2, 96, 2), (4096, 1, 64, 4), (16, 40, 256, 3)])
def test_large_pages(gpu, ctype, page, kv, hd, beams):
    """Rows up to a slice's border, one before and one behind, all but one of a page; rows behind stay."""
    import torch
    from ligguf_amd import ops
    row = kv * (hd * 2 if ctype == L.F16 else hd * 5 // 8)
    cut = min(max(65536 // row // 16 * 16, 16), page)
    for rows in sorted({min(n, page - 1) for n in (1, 15, 16, 17, cut - 1, cut, cut + 1, page)}):
        print(f"reorder type {ctype} page {page} of {kv} x {hd}, {rows} rows", flush=True)
        g = np.random.default_rng(rows)
        n = 2 * beams + 1
        table = torch.from_numpy(g.permutation(n)[:2 * beams].reshape(beams, 2).astype(np.int32)).to(gpu)
        c = ops.PagedKvCache.empty(ctype, n, page, kv, hd, table)
        for b in (c.k, c.v):
            b.view(torch.int32).random_(-2 ** 31, 2 ** 31 - 1)
        before = [b.clone() for b in (c.k, c.v)]
        parent, length = [[beams - 1] * beams], page + rows
        blank = [np.zeros((n, page, 1), np.int16) for _ in range(2)]
        want = moved(table.cpu().numpy(), blank, parent, [length], page, beams, n)
        old = table.cpu().numpy()
        ops.beam_reorder(ops.PagedLayers([c]), torch.tensor(parent, dtype=torch.int32, device=gpu), torch.tensor([length], dtype=torch.int32, device=gpu))
        assert np.array_equal(table.cpu().numpy(), want)
        src = int(old[beams - 1, 1])
        for a, b in zip((c.k, c.v), before):
            for p in range(n):
                x, y, z = (t.view(torch.uint8).reshape(n, -1) for t in (a, b, b))
                copied = p in want[:, 1] and p != src
                if ctype == L.F16:
                    parts = [(0, page * row, row)]
                else:
                    parts = [(h * page * hd // 2, page * hd // 2, hd // 2) for h in range(kv)]
                    parts += [(kv * page * hd // 2 + h * page * hd // 8, page * hd // 8, hd // 8) for h in range(kv)]
                for at, size, one in parts:
                    m = rows * one if copied else 0
                    assert torch.equal(x[p, at:at + m], z[src, at:at + m])
                    assert torch.equal(x[p, at + m:at + size], y[p, at + m:at + size])


@pytest.mark.parametrize("ng,nb,vocab,top", [(1, 1, 4095, 3), (1, 1, 4096, 3), (1, 2, 8191, 7), (1, 2, 8192, 7), (1, 3, 8193, 64), (1, 64, 8200, 64),
                                             (1, 1, 151936, 64), (300, 2, 5000, 4), (1, 16, 65537, 32), (513, 1, 3000, 1), (1, 3, 32767, 5),
                                             (1, 3, 32768, 5), (2, 3, 32769, 9), (1, 2, 49155, 64)])
def test_vocabularies_at_borders_of_parts(gpu, ng, nb, vocab, top):
    g = np.random.default_rng(vocab)
    x = (g.standard_normal((ng, nb, vocab)) * 3).astype(np.float32)
    s = -np.sort(g.random((ng, nb)).astype(np.float32) * 9, axis=1)
    # the best ones at the ends of rows and of parts
    for p in (0, vocab - 1, min(4095, vocab - 1), min(4096, vocab - 1), min(16384, vocab - 1), vocab // 2, vocab // 3):
        x[:, :, p] = 12 + g.random((ng, nb)).astype(np.float32)
    check(gpu, x, s, top)
