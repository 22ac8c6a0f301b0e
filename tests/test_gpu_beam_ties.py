"""lg_beam_select where candidates' scores are the same in double: by the lower beam, of one beam by the higher
logit, then the lower token -- also where a row's logits are looked through in several parts."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def choose(x, scores, top):
    """(parent, token) of a group whose candidates' scores are the same for all tokens of a beam, which the caller
    sees to: beams by score, then in order, tokens by logit, then in order."""
    out = []
    for b in np.lexsort((np.arange(len(scores)), -scores.astype(np.float64))):
        out += [(int(b), int(t)) for t in np.lexsort((np.arange(x.shape[1]), -x[b].astype(np.float64)))[:top]]
    return out[:top]


def check(gpu, x, scores, top):
    import torch
    from ligguf_amd import ops
    print(f"beam ties {x.shape}, top {top}", flush=True)
    r = ops.beam_select(torch.from_numpy(x).to(gpu), torch.from_numpy(scores).to(gpu), top)
    p, t = r.parent.cpu().numpy(), r.token.cpu().numpy()
    for g in range(len(x)):
        assert list(zip(p[g].tolist(), t[g].tolist())) == choose(x[g], scores[g], top), g
    return r


@pytest.mark.parametrize("vocab", [300, 20000, 32768, 40000, 151936])
@pytest.mark.parametrize("beams,top", [(1, 1), (1, 2), (1, 64), (3, 5), (8, 16), (64, 64)])
def test_logits_next_to_nothing(gpu, vocab, beams, top):
    """Logits of 0 and of 1e-20 and less: log sums of 5 and more take their differences away."""
    g = np.random.default_rng(vocab + top)
    x = np.zeros((2, beams, vocab), np.float32)
    for row in x.reshape(-1, vocab):
        row[g.integers(0, vocab, 40)] = (g.integers(-9, 10, 40) * 1e-21).astype(np.float32)
    x[0, 0, vocab // 3], x[0, 0, vocab - 3] = 1e-20, 2e-20
    check(gpu, x, np.full((2, beams), -1.5, np.float32), top)


@pytest.mark.parametrize("vocab", [1000, 50257, 151936])
@pytest.mark.parametrize("beams,top", [(1, 64), (4, 8), (6, 40)])
def test_scores_that_outweigh_all_logits(gpu, vocab, beams, top):
    """Beams of -10^30: their tokens' scores are all the same; logits rise, fall and repeat over the parts."""
    x = np.zeros((3, beams, vocab), np.float32)
    x[0] = np.arange(vocab) / vocab
    x[1] = -np.arange(vocab) / vocab
    x[2] = np.arange(vocab) % 7
    s = np.full((3, beams), -1e30, np.float32)
    s[:, 1:2] = -2e30
    check(gpu, x, s, top)


def test_the_same_alone_and_among_many(gpu):
    """Rows alone are looked through in parts, among many as a whole: the same choice."""
    g = np.random.default_rng(3)
    x = np.zeros((300, 2, 40000), np.float32)
    x[0, :, g.integers(0, 40000, 30)] = (g.integers(1, 9, (30, 1)) * 1e-20).astype(np.float32)
    x[1:] = x[:1]
    s = np.full((300, 2), -1.0, np.float32)
    one, all_ = check(gpu, x[:1], s[:1], 12), check(gpu, x, s, 12)
    for a, b in zip(one, all_):
        assert bool((a == b).all())
