"""The example runs the paged cache's and beam search's calls together: every speculative token is a greedy choice, and
every beam's score is the sum of its tokens' log probabilities, both by runs of the plain chain over the whole text."""

import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def _logits(E, model, text):
    """Logits after every token of a text, in one chunk on a cache of its own."""
    cache = E.Cache(model, -(-len(text) // 16))
    tables = [[]]
    table = cache.grow(tables, [len(text)])
    return model.forward(torch.tensor(text, device="cuda"), cache, table, E.ints([0, len(text)]), E.ints([0])).double().cpu()


def test_speculative_tokens_are_greedy_choices(cuda):
    import paged_serving as E
    model = E.Model()
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(model.vocab, (n,), generator=g).tolist() for n in (1, 16, 45)]
    plain = E.greedy(model, E.Cache(model, 32), prompts, 16)

    def draft(b, so_far):
        ahead = plain[b][len(so_far):len(so_far) + 4]
        return [(i, t) for i, t in enumerate(ahead)] + [(0, 3), (1 if ahead else 0, 5)]

    fast, rounds = E.speculative(model, E.Cache(model, 32), prompts, 16, draft)
    assert rounds <= 8  # 15 tokens after the prompt's own, up to 5 a step
    for prompt, out in zip(prompts, fast):
        logits = _logits(E, model, prompt + out)
        for i, t in enumerate(out):
            row = logits[len(prompt) - 1 + i]
            # fp16 activations through two layers: logits of size 3 within 0.03
            assert row[t] >= row.max() - 0.06


def test_beam_scores_are_log_probabilities(cuda):
    import paged_serving as E
    model = E.Model(seed=4)
    g = torch.Generator().manual_seed(5)
    prompt = torch.randint(model.vocab, (30,), generator=g).tolist()
    scores, tokens = E.beams(model, E.Cache(model, 40), prompt, 10, 4)
    assert scores == sorted(scores, reverse=True) and len({tuple(t) for t in tokens}) == 4
    for s, out in zip(scores, tokens):
        lp = torch.log_softmax(_logits(E, model, prompt + out), -1)
        total = sum(lp[len(prompt) - 1 + i, t].item() for i, t in enumerate(out))
        assert abs(total - s) <= 0.06 * len(out), (total, s)
