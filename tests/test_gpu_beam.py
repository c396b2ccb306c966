"""GPU tests of beam.select against the 64-bit restatement: parents and tokens equal, scores within the rounding of the
total to fp32 (2^-24 of it) and 1e-6 for the logarithm's sum (terms within 2^-22 each)."""

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu


def _check(logits, scores):
    import beam
    want = R.select(logits.double().cpu(), scores.double().cpu())
    got = beam.select(logits, scores)
    assert got[0].dtype == torch.float32 and got[1].dtype == got[2].dtype == torch.int32
    assert got[1].tolist() == want[1].tolist()
    assert got[2].tolist() == want[2].tolist()
    g, w = got[0].double().cpu(), want[0]
    fin = w > -float("inf")
    assert torch.equal(fin, g > -float("inf"))
    assert ((g - w).abs()[fin] <= 2.0 ** -23 * w.abs()[fin] + 1e-6).all()
    again = beam.select(logits, scores)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,W,V", [(1, 1, 1), (1, 4, 5), (2, 3, 1), (3, 5, 2047), (1, 4, 32000), (2, 16, 31337), (1, 64, 4099), (5, 64, 70),
                                   (1, 2, 50257), (7, 1, 9000)])
def test_select(cuda, dtype, B, W, V):
    g = torch.Generator().manual_seed(V + W)
    x = (torch.randn(B, W, V, generator=g) * 3).to(dtype).cuda()
    _check(x, (torch.randn(B, W, generator=g) * 2).cuda())


def test_select_large(cuda):
    """Enough rows for 64 logits a thread."""
    g = torch.Generator().manual_seed(5)
    _check((torch.randn(16, 8, 128256, generator=g) * 2.5).half().cuda(), torch.randn(16, 8, generator=g).cuda())


@pytest.mark.parametrize("V", [33, 5000, 70001])
def test_select_equal_logits(cuda, V):
    """All equal: the lowest tokens of the lowest beams; two levels: the upper one first."""
    x = torch.zeros(2, 3, V, device="cuda")
    _check(x, torch.zeros(2, 3, device="cuda"))
    x[:, :, V // 2:] = 1.0
    _check(x.half(), torch.zeros(2, 3, device="cuda"))
    x[0, 1, -1] = 2.0
    _check(x, torch.tensor([[0.0, -1.0, 0.0], [1.0, 1.0, 1.5]], device="cuda"))


def test_select_equal_beams_many(cuda):
    """64 equal beams of equal logits overflow the candidate lists of both passes."""
    _check(torch.ones(2, 64, 3000, device="cuda"), torch.zeros(2, 64, device="cuda"))


def test_select_first_step(cuda):
    g = torch.Generator().manual_seed(6)
    x = torch.randn(2, 4, 6000, generator=g).cuda()
    s = torch.full((2, 4), -float("inf"), device="cuda")
    s[:, 0] = 0
    _check(x, s)
    _check(x[:, :, :3].contiguous(), s)  # fewer tokens than beams: -inf totals fill up in order
    s[1] = -float("inf")
    _check(x, s)


def test_select_masked_and_nan(cuda):
    g = torch.Generator().manual_seed(7)
    x = torch.randn(3, 4, 5001, generator=g).half().cuda()
    x[0, :, 2:] = -float("inf")     # constrained to two tokens
    x[1, 2] = float("nan")          # a beam that is not a number loses to the others
    x[2, 1, 77] = float("nan")
    x[2, 3, 78] = float("inf")
    _check(x, torch.randn(3, 4, generator=g).cuda())


def test_select_all_nan_is_in_range(cuda):
    import beam
    x = torch.full((1, 3, 4000), float("nan"), device="cuda")
    s, p, t = beam.select(x, torch.zeros(1, 3, device="cuda"))
    assert (s == -float("inf")).all() and ((p >= 0) & (p < 3)).all() and ((t >= 0) & (t < 4000)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_select_strides(cuda, dtype):
    """Rows that start at any element, and a vocabulary with padding behind it."""
    g = torch.Generator().manual_seed(8)
    wide = torch.randn(2, 5, 4111, generator=g).to(dtype).cuda()
    wide[..., 4001:] = 100.0
    _check(wide[:, 1:4, :4001], torch.randn(2, 3, generator=g).cuda())
    _check(wide[:, ::2, 3:4000], torch.randn(2, 3, generator=g).cuda())


def test_select_near_totals(cuda):
    """Totals 1e-5 apart on beams of different logarithms."""
    g = torch.Generator().manual_seed(9)
    x = torch.randn(1, 2, 40000, generator=g).cuda()
    x[0, 0, 11], x[0, 1, 22] = 9.0, 12.0
    lse = torch.logsumexp(x.double().cpu(), -1)[0]
    s0 = torch.tensor([-1.0], dtype=torch.float64)
    for d in (1e-5, -1e-5):
        s1 = s0 + (9.0 - lse[0]) - (12.0 - lse[1]) + d
        _check(x, torch.cat([s0, s1])[None].float().cuda())


def test_refusals(cuda):
    import beam
    x, s = torch.zeros(1, 2, 8, device="cuda"), torch.zeros(1, 2, device="cuda")
    for bad in (lambda: beam.select(x[0], s), lambda: beam.select(x.double(), s), lambda: beam.select(x, s.half()),
                lambda: beam.select(x, s[:, :1]), lambda: beam.select(x.transpose(1, 2), torch.zeros(1, 8, device="cuda")),
                lambda: beam.select(torch.zeros(1, 65, 8, device="cuda"), torch.zeros(1, 65, device="cuda")),
                lambda: beam.select(x, s.cpu()), lambda: beam.select(x[:, :, :0], s)):
        with pytest.raises(ValueError):
            bad()
