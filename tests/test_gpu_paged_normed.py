"""GPU tests of paged.append with norms and axes against the 64-bit restatement in paged_context_reference.py.

Tolerances: a stored value is rounded once, at most half a step (2^-11 f16, 2^-8 bf16, 2^-4 e4m3 of the value; subnormal steps
2^-24 / 2^-9).  In fp32 before it: the squares' sum (each square and 10 levels of additions, 2^-24 each: 1e-6, half of that after
the root), the root, the division and two products (3e-7), then the rotation as without norms, 1e-6 (|a| + |b|) of
the pair: below 2e-6 of the normed row's length in all."""

import random

import pytest
import torch

import paged_context_reference as C
import paged_reference as R
from test_gpu_paged import HALF, TINY, _bits, _garbage, _ints

pytestmark = pytest.mark.gpu

F16, BF16, E4, F32 = torch.float16, torch.bfloat16, torch.float8_e4m3fn, torch.float32
EPS = 1e-6


def _check(seed, heads, kv, D, page, ctx, new, dtype=F16, cache=None, rotary=None, neox=False, base=10000.0, weight=None, axes=0, which="qk",
           with_q=True, strided=False, ks=1.0, vs=1.0, far=False, odd=False):
    import paged
    cache = cache or dtype
    rng = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    B, T = len(ctx), sum(new)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    rd = D if rotary is None else rotary
    table, pages = R.make_pages(rng, [c + n for c, n in zip(ctx, new)], page, extra_pages=2)
    fused = (torch.randn(T, heads + 2 * kv, D, generator=g) * 3).to(dtype).cuda()
    fused[:, 0] *= 1e-3  # a head in which eps counts
    shift = (lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)) if odd else lambda t: t.contiguous()
    q, k, v = fused[:, :heads], fused[:, heads:heads + kv], fused[:, heads + kv:]
    if strided:
        both = _garbage((pages, 2, kv, page, D), cache)
        kc, vc = both[:, 0], both[:, 1]
    else:
        q, k, v = shift(q), shift(k), shift(v)
        kc, vc = _garbage((pages, kv, page, D), cache), _garbage((pages, kv, page, D), cache)
    before = _bits(kc).clone(), _bits(vc).clone()
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).to(weight or dtype).cuda() if c in which else None for c in "qk")
    rows = [[ctx[b] + i for b in range(B) for i in range(new[b])]]
    axis, given = [0] * (rd // 2), None
    if axes:
        rows = [[(2_000_000_011 if far else 7) * a + p * (a + 1) // 3 for p in rows[0]] for a in range(axes)]
        axis = [rng.randrange(axes) for _ in range(rd // 2)]
        given = torch.full((axes, T + 3), -9, dtype=torch.int32, device="cuda")[:, :T].copy_(_ints(rows))
    out = paged.append(k, v, kc, vc, _ints(table).reshape(B, -1), _ints(cu), _ints(ctx), q=q if with_q else None, positions=given, freq_base=base,
                       rotary_dim=rotary, neox=neox, k_scale=ks, v_scale=vs, q_norm=qw if with_q else None, k_norm=kw, norm_eps=EPS,
                       axes=axis if axes else None)
    torch.cuda.synchronize()
    wd = [None if w is None else w.double().cpu() for w in (qw, kw)]
    qd, kd, vd = q.double().cpu(), k.double().cpu(), v.double().cpu()
    kg, vg = kc.float().double().cpu() * ks, vc.float().double().cpu() * vs

    def close(got, x, w, t, pos, scale=1.0, limit=None):
        x = C.normed(x, w, EPS)
        want = C.rotate_axes(x, pos, base, rd, neox, axis)
        if limit:
            want = want.clamp(-limit, limit)
        lim = HALF[t] * want.abs() + TINY[t] * scale + 2e-6 * torch.linalg.vector_norm(x, dim=-1, keepdim=True)
        assert ((got - want).abs() <= lim).all(), ((got - want).abs() / lim).max()

    touched = set()
    for b in range(B):
        for i in range(new[b]):
            t, row = cu[b] + i, ctx[b] + i
            pos = [r[t] for r in rows]
            pg, slot = table[b][row // page], row % page
            touched.add((pg, slot))
            close(kg[pg, :, slot], kd[t], wd[1], cache, pos, ks, 448 * ks if cache == E4 else None)
            vw = vd[t].clamp(-448 * vs, 448 * vs) if cache == E4 else vd[t]
            lim = HALF[cache] * vw.abs() + TINY[cache] * vs if cache == E4 else 0.0 * vw
            assert ((vg[pg, :, slot] - vw).abs() <= lim).all()
            if with_q:
                close(out[t].double().cpu(), qd[t], wd[0], dtype, pos)
    for c, old in ((kc, before[0]), (vc, before[1])):  # nothing else is touched
        same = (_bits(c) == old).reshape(pages, kv, page, -1).all(-1).all(1).cpu()
        for pg in range(pages):
            for slot in range(page):
                assert same[pg, slot] or (pg, slot) in touched, (pg, slot)
    return out


@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("dtype,cache,weight", [(F16, F16, F16), (BF16, BF16, F32), (F16, E4, F32), (BF16, E4, BF16)])
def test_types(cuda, dtype, cache, weight, neox):
    e4 = cache == E4
    _check(1, 8, 2, 64, 16, [5, 0, 31], [1, 7, 3], dtype, cache, neox=neox, weight=weight, axes=3, ks=0.0625 if e4 else 1.0, vs=0.3 if e4 else 1.0)


@pytest.mark.parametrize("D,rotary,neox", [(96, None, True), (96, 48, True), (96, 48, False), (128, 64, True), (128, 128, True), (256, None, False),
                                           (256, 256, True), (256, 16, True), (64, 0, False), (64, 20, True), (64, 12, False), (40, 10, False),
                                           (8, 2, True), (200, 80, True), (240, None, False), (16, 16, True)])
def test_rotary_sizes(cuda, D, rotary, neox):
    _check(2, 3, 1, D, 32, [17, 2], [9, 1], rotary=rotary, neox=neox, axes=2)


@pytest.mark.parametrize("which", ["q", "k", ""])
@pytest.mark.parametrize("axes", [0, 1, 4])
def test_one_norm_or_axes_alone(cuda, which, axes):
    _check(3, 5, 3, 64, 16, [3, 40], [2, 6], which=which, axes=axes, neox=True)


@pytest.mark.parametrize("page", [1, 2, 16, 128])
def test_pages(cuda, page):
    _check(4, 4, 2, 64, page, [0, 15, 16, 40], [2, 1, 17, 0], BF16)


def test_far_positions(cuda):
    _check(5, 4, 2, 128, 16, [3], [6], neox=True, base=500000.0, axes=2, far=True)


@pytest.mark.parametrize("neox", [False, True])
def test_strided_views(cuda, neox):
    _check(6, 6, 3, 64, 16, [4, 9], [3, 5], neox=neox, axes=3, strided=True)
    _check(7, 6, 3, 64, 16, [4, 9], [3, 5], BF16, E4, neox=neox, strided=True)


@pytest.mark.parametrize("cache", [F16, E4])
def test_unaligned(cuda, cache):
    _check(8, 4, 2, 64, 16, [14], [5], cache=cache, axes=3, odd=True, ks=0.3 if cache == E4 else 1.0)


def test_without_queries_and_many_sequences(cuda):
    _check(9, 4, 2, 64, 16, [i % 19 for i in range(150)], [i % 3 for i in range(150)], with_q=False)


@pytest.mark.parametrize("heads,kv,D,neox", [(32, 8, 128, True), (7, 7, 96, False), (24, 1, 256, True), (1, 1, 64, False)])
def test_many_tokens(cuda, heads, kv, D, neox):
    """Enough tokens that a block takes every head of its token."""
    _check(10, heads, kv, D, 64, [0, 100], [700, 430], neox=neox, axes=3)


def test_in_place_and_zero_rows(cuda):
    """q_out may be q; a head of zeros stays zeros."""
    import paged
    g = torch.Generator().manual_seed(11)
    q, k, v = (torch.randn(5, h, 128, generator=g).half().cuda() for h in (4, 2, 2))
    q[2, 1] = 0
    w = torch.ones(128, dtype=F32, device="cuda")
    kc, vc = _garbage((2, 2, 16, 128), F16), _garbage((2, 2, 16, 128), F16)
    args = (kc, vc, _ints([[1, 0]]), _ints([0, 5]), _ints([13]))
    want = paged.append(k, v, *args, q=q.clone(), neox=True, q_norm=w, k_norm=w)
    got = paged.append(k, v, *args, q=q, q_out=q, neox=True, q_norm=w, k_norm=w)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want) and (got[2, 1] == 0).all() and not got.isnan().any()


def test_nan_stays_in_its_head_and_bad_pages_are_left(cuda):
    import paged
    q, k = torch.randn(40, 2, 64, device="cuda").half(), torch.randn(40, 1, 64, device="cuda").half()
    q[3, 1, 5], k[7, 0, 0] = float("nan"), float("inf")
    w = torch.ones(64, dtype=F16, device="cuda")
    kc, vc = _garbage((2, 1, 16, 64), F16), _garbage((2, 1, 16, 64), F16)
    out = paged.append(k, k, kc, vc, _ints([[1, 7]]), _ints([0, 40]), _ints([4]), q=q, q_norm=w, k_norm=w)
    bad = out.isnan().any(-1)
    assert bad[3, 1] and bad.sum() == 1
    rows = kc[1, 0, 4:].isnan().any(-1)  # rows 4..15 are tokens 0..11
    assert rows[7] and rows.sum() == 1 and kc[0].isnan().all() and kc[1, 0, :4].isnan().all()


def test_padding_tokens_are_passed_over(cuda):
    import paged
    q, k = torch.randn(6, 2, 64, device="cuda").half(), torch.randn(6, 1, 64, device="cuda").half()
    kc, vc = _garbage((1, 1, 16, 64), F16), _garbage((1, 1, 16, 64), F16)
    out = torch.full_like(q, 7.0)
    paged.append(k, k, kc, vc, _ints([[0]]), _ints([1, 4]), _ints([2]), q=q, q_out=out, k_norm=torch.ones(64, dtype=F16, device="cuda"))
    assert (out[0] == 7).all() and (out[4:] == 7).all() and (out[1:4] != 7).any() and kc[0, 0, 5:].isnan().all()


def test_refusals(cuda):
    import paged
    k, c = torch.zeros(2, 1, 64, dtype=F16, device="cuda"), torch.zeros(2, 1, 16, 64, dtype=F16, device="cuda")
    w = torch.ones(64, dtype=F16, device="cuda")
    args, pos = (k, k, c, c.clone(), _ints([[0]]), _ints([0, 2]), _ints([0])), _ints([[0, 1], [2, 3]])
    for kw in (dict(k_norm=w[:32]), dict(k_norm=w.cpu()), dict(k_norm=w.bfloat16()), dict(k_norm=torch.ones(128, dtype=F16, device="cuda")[::2]),
               dict(q_norm=w), dict(q=k, q_norm=w, k_norm=w.float()), dict(k_norm=w, norm_eps=-1.0), dict(axes=[0] * 32),
               dict(axes=[0] * 31, positions=pos), dict(axes=[2] * 32, positions=pos), dict(axes=[-1] * 32, positions=pos),
               dict(axes=[0] * 32, positions=pos[0]), dict(axes=[0] * 32, positions=pos[:, :1]), dict(positions=pos, k_norm=w)):
        with pytest.raises(ValueError):
            paged.append(*args, **kw)
