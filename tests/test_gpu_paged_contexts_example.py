"""GPU test of the normed append, the weighted and the shared attention and the eviction together, as
examples/paged_long_contexts.py runs them.

Logits of the shared and of the plain attention differ by the roundings of fp16 activations (2^-11 of values of a few units, through two layers and
a head of three times unit variance): 0.05 covers them; a row too many or too few changes logits by their own size, 3."""

import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.fixture
def served(cuda):
    import paged_long_contexts as ex
    model = ex.LongModel()
    document, positions, questions = ex.make(model)
    cache = ex.Cache(model, 96)
    pages, weights = ex.read(model, cache, document, positions)
    return ex, model, document, positions, questions, cache, pages, weights


def test_every_weight_is_counted(served):
    """A token's weights add up to 1 for each of its heads, so those of a kv head's rows to its heads' tokens: to 2^-16 of the sum
    and 4e-5 a weight (test_gpu_paged_weighted.py)."""
    ex, model, document, _, _, _, _, weights = served
    total = weights.double().sum(-1)
    want = len(document) * model.heads // model.kv_heads
    assert ((total - want).abs() <= want * 6e-5).all(), total
    # the first row is seen by every token, the last by one
    assert (weights[..., len(document) - 1] <= model.heads // model.kv_heads).all() and (weights[..., len(document):] == 0).all()


def test_shared_pages_give_what_single_ones_do(served):
    ex, model, document, positions, questions, cache, pages, _ = served
    end = positions[0][-1] + 1
    _, one = ex.answer(model, cache, pages, len(document), end, questions, 2)
    _, two = ex.answer(model, cache, pages, len(document), end, questions, 2, share=False)
    assert ((one - two).abs() <= 0.05).all() and one.std() > 1


def test_a_cut_document(served):
    ex, model, document, positions, questions, cache, pages, weights = served
    end, n = positions[0][-1] + 1, len(document)
    _, whole = ex.answer(model, cache, pages, n, end, questions, 1)
    k, v = cache.k.clone(), cache.v.clone()
    same, rows, w = ex.cut(cache, pages, n, weights, keep=n)  # nothing to cut
    assert same == pages and rows == n and torch.equal(w[..., :n], weights[..., :n])
    kept, rows, w = ex.cut(cache, pages, n, weights, keep=80)
    assert rows == 80 and len(kept) == 5 and not set(kept) & set(pages)
    page = cache.page_size
    for layer in range(model.layers):
        for g in range(model.kv_heads):
            order = weights[layer, 0, g, 4:n - 16].sort(descending=True, stable=True).indices[:60] + 4
            stay = sorted([0, 1, 2, 3] + order.tolist() + list(range(n - 16, n)))
            assert torch.equal(w[layer, 0, g, :80], weights[layer, 0, g, stay])
            for d, j in enumerate(stay):
                for new, old in ((cache.k, k), (cache.v, v)):
                    assert torch.equal(new[layer, kept[d // page], g, d % page], old[layer, pages[j // page], g, j % page])
    out, less = ex.answer(model, cache, kept, rows, end, questions, 3)
    _, plain = ex.answer(model, cache, kept, rows, end, questions, 3, share=False)
    assert ((less - plain).abs() <= 0.05).all() and not torch.equal(less, whole) and all(len(o) == 3 for o in out)


def test_a_step_captured(served):
    """One layer's calls of a decoding step in a graph, replayed with other lengths between eager ones."""
    import paged
    ex, model, document, _, _, cache, pages, _ = served
    B, H, K, D = 3, model.heads, model.kv_heads, model.head_dim
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(B, H + 2 * K, D, generator=g, device="cuda").half()
    spare = [cache.free.pop() for _ in range(B)]
    for x in (cache.k, cache.v):  # rows that nothing has been written to would be whatever the allocator left
        x[:, spare] = torch.randn(x[:, spare].shape, generator=g, device="cuda").half()
    table, cu, ctx = ex.ints([pages[:10] + [p] for p in spare]), ex.ints([0, 1, 2, 3]), ex.ints([160, 165, 163])
    groups, shared, pos = ex.ints([0, 3]), ex.ints([160]), ex.ints([[70, 71, 72], [1, 2, 3], [4, 5, 6]])
    sums = torch.zeros(B, K, 176, device="cuda")
    new = torch.zeros_like(sums)

    def step():
        q = paged.append(qkv[:, H:H + K], qkv[:, H + K:], cache.k[0], cache.v[0], table, cu, ctx, q=qkv[:, :H], positions=pos, neox=True,
                         q_norm=model.q_norm, k_norm=model.k_norm, axes=model.axes)
        a = paged.shared_attention(q, cache.k[0], cache.v[0], table, cu, ctx, groups, shared, max_new=1)
        b, _ = paged.weighted_attention(q, cache.k[0], cache.v[0], table, cu, ctx, sums, weights_out=new, max_new=1)
        return q, a, b

    step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = step()
    for lens in ([160, 165, 163], [170, 160, 161], [162, 163, 175]):
        ctx.copy_(ex.ints(lens))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (*held, new)]
        want = [x.clone() for x in (*step(), new)]
        assert all(torch.equal(a, b) for a, b in zip(got, want))
