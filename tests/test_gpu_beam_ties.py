"""GPU tests of beam.select's order of equal totals: lower beam first, then the lower token, for zeros of either sign and for
beams that are out; where the totals of different logits round to one number, the larger logit."""

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
INF = float("inf")


def _order(logits, scores):
    """The call's parents and tokens, and the definition's."""
    import beam
    want = R.select(logits.double().cpu(), scores.double().cpu())
    got = beam.select(logits, scores)
    fin = want[0] > -INF
    assert torch.equal(got[0].cpu() > -INF, fin)
    assert ((got[0].double().cpu() - want[0]).abs()[fin] <= 2.0 ** -23 * want[0].abs()[fin] + 1e-6).all()
    assert got[1].tolist() == want[1].tolist()
    assert got[2].tolist() == want[2].tolist()


def _signs(seed, shape):
    g = torch.Generator().manual_seed(seed)
    return torch.where(torch.rand(shape, generator=g) < 0.5, -torch.zeros(shape), torch.zeros(shape))


@pytest.mark.parametrize("dtype", TYPES)
def test_zeros_of_either_sign_are_equal(cuda, dtype):
    _order(torch.tensor([[[-0.0, 0.0]]], device="cuda").to(dtype), torch.zeros(1, 1, device="cuda"))
    for V, W in ((40, 3), (5000, 1), (5000, 8), (70001, 4)):
        x = -1.0 - torch.rand(2, W, V, generator=torch.Generator().manual_seed(V))
        at = torch.randperm(V, generator=torch.Generator().manual_seed(W))[:min(V, 30)]
        x[:, :, at] = _signs(V + W, (2, W, len(at)))  # the maximum, in many places
        _order(x.to(dtype).cuda(), torch.zeros(2, W, device="cuda"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [33, 5000])
def test_zeros_of_either_sign_at_the_cut(cuda, dtype, V):
    """Nothing but zeros, and zeros below a few larger logits: which ones stay is the lowest tokens' matter."""
    x = _signs(V, (2, 6, V))
    _order(x.to(dtype).cuda(), torch.zeros(2, 6, device="cuda"))
    x[:, :, V - 3:] = 1.0
    x[0, 2, V // 2] = 2.0
    _order(x.to(dtype).cuda(), torch.zeros(2, 6, device="cuda"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), INF])
def test_a_beam_that_is_out_stands_for_its_lowest_tokens(cuda, dtype, bad):
    """One logit that is NaN or infinite puts its beam out: all of its totals are -inf, and equal."""
    g = torch.Generator().manual_seed(3)
    for W, V in ((1, 7), (1, 5000), (3, 40000), (8, 5), (64, 2100)):
        x = torch.randn(2, W, V, generator=g)
        x[:, :, V // 2] = bad
        _order(x.to(dtype).cuda(), torch.zeros(2, W, device="cuda"))
    # a sentence with too few finite totals: the beam that is out fills up in order with the masked tokens of the others
    x = torch.randn(1, 5, 6000, generator=g)
    x[0, 1, 4000] = bad
    x[0, 0, 2:] = x[0, 2:, 1:] = -INF
    s = torch.tensor([[0.5, 0.0, -INF, -INF, float("nan")]], device="cuda")
    _order(x.to(dtype).cuda(), s)


def test_nothing_but_nan(cuda):
    _order(torch.full((2, 3, 4000), float("nan"), device="cuda"), torch.zeros(2, 3, device="cuda"))


@pytest.mark.parametrize("score", [-1e30, 1e30, INF])
def test_totals_that_round_to_one_number(cuda, score):
    """A score beside which the logits vanish: within a beam the larger logit is still the better one."""
    import beam
    x = torch.randn(1, 3, 9000, generator=torch.Generator().manual_seed(4))
    x[0, 0, [5, 8000]] = 9.0  # equal logits: the lower token
    s, p, t = beam.select(x.cuda(), torch.full((1, 3), score, device="cuda"))
    assert (s == score).all() and p.tolist() == [[0, 0, 0]]
    assert t[0].tolist() == torch.sort(x[0, 0], descending=True, stable=True).indices[:3].tolist()
