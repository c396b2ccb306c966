"""The example's beam search returns every page that its hypotheses no longer hold."""

import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.parametrize("length,steps,width", [(30, 50, 4), (32, 20, 3), (7, 40, 5)])
def test_beams_return_dropped_pages(cuda, monkeypatch, length, steps, width):
    import paged_serving as E
    held = {}
    reorder = E.beam.reorder

    def recorded(*args, **kw):
        res = reorder(*args, **kw)
        held["table"] = res[0]
        return res

    monkeypatch.setattr(E.beam, "reorder", recorded)
    model = E.Model(seed=length)
    prompt = torch.randint(model.vocab, (length,), generator=torch.Generator().manual_seed(length)).tolist()
    pages = 60
    cache = E.Cache(model, pages)
    E.beams(model, cache, prompt, steps, width)
    used = {p for row in held["table"].tolist() for p in row if p >= 0}
    assert len(cache.free) == len(set(cache.free)) and not used & set(cache.free)
    assert sorted(used | set(cache.free)) == list(range(pages))
