"""p0pc0rn_amd.beam_search end to end: every beam that a search returns is scored again by itself, token after token in a sequence
that shares nothing, and its score has to be the sum of the logarithms of its tokens' probabilities. A wrong parent, page, copy or
row of the cache anywhere on the way would show. Both sides run the same kernels over the same cached values, but the split of a
row's work may differ: sums of up to 30 logarithms in fp32 of magnitude under 400 agree to 30 * 400 * 2^-23 = 1.5e-3."""
import numpy as np
import pytest

from p0pc0rn_amd import beam_search as B

pytestmark = pytest.mark.gpu


def rescore(model, prompt, text, **kw):
    s = B.Search(model, 1, 1, longest=len(prompt) + len(text) + 1, **kw)
    total = 0.0
    for i, t in enumerate(list(prompt) + list(text)):
        if i >= len(prompt):
            x = s.logits.read(np.float32, model.vocab).astype(np.float64)
            total += x[t] - (x.max() + np.log(np.exp(x - x.max()).sum()))
        s.sequences(1)
        s.forward(np.array([t]))
    return total


@pytest.mark.parametrize("kw", [{}, dict(window=9, sinks=2), dict(page=64)])
def test_every_beam_has_the_score_of_its_tokens(dev, kw):
    model = B.Decoder(vocab=1024)
    prompts = np.random.default_rng(3).integers(0, 1024, (2, 27))
    s = B.Search(model, 2, 4, longest=60, **kw)
    text, score = s.run(prompts, 30)
    assert np.all(np.diff(score, axis=1) <= 0)
    for n in range(2):
        assert len({tuple(t) for t in text[n].tolist()}) == 4
        for w in (0, 3):
            assert abs(rescore(model, prompts[n], text[n, w], **kw) - score[n, w]) <= 1.5e-3, (n, w)
    held = s.ref.read(np.int32, s.n_pages)
    assert held.max() > 1 or kw                            # beams of one prompt share its pages


def test_a_search_of_one_beam_is_greedy(dev):
    model = B.Decoder(vocab=512, seed=4)
    text, _ = B.Search(model, 1, 1, longest=30).run([[7, 3]], 12)
    s, tokens = B.Search(model, 1, 1, longest=30), []
    for t in [7, 3]:
        s.sequences(1)
        s.forward(np.array([t]))
    for _ in range(12):
        tokens.append(int(s.logits.read(np.float32, 512).argmax()))
        s.sequences(1)
        s.forward(np.array([tokens[-1]]))
    assert text[0, 0].tolist() == tokens


def test_a_pool_that_is_too_small_says_so(dev):
    s = B.Search(B.Decoder(vocab=512), 1, 2, longest=40)
    s.n_pages = 1
    with pytest.raises(RuntimeError, match="pages missing"):
        s.run([[1] * 33], 2)
