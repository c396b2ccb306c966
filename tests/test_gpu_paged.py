"""GPU tests of the paged cache's writes and moves: append (rotation, types, strides, pages), commit_path and
beam.reorder, against the 64-bit restatement in paged_reference.py.

Tolerances: a stored value is rounded once, at most half a step (2^-11 f16, 2^-8 bf16, 2^-4 e4m3 of the value; subnormal
steps 2^-24 / 2^-9).  The fp32 rotation before it: angle 1e-7, sine and cosine 2.4e-7, three roundings of 6e-8, below
1e-6 (|a| + |b|) of the pair in all."""

import random

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float8_e4m3fn: 2.0 ** -4}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float8_e4m3fn: 2.0 ** -10}


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _garbage(shape, dtype):
    """A cache full of NaN, so that whatever is not written shows."""
    if dtype == torch.float8_e4m3fn:
        return torch.full(shape, 0x7F, dtype=torch.uint8, device="cuda").view(dtype)
    return torch.full(shape, float("nan"), dtype=dtype, device="cuda")


def _bits(t):
    return t.contiguous().view(torch.uint8)


def _check_append(seed, heads, kv, D, page, ctx, new, dtype, cache, rotary, neox, base=10000.0, with_q=True, positions="tree",
                  strided=False, ks=1.0, vs=1.0):
    import paged
    rng = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    B, T = len(ctx), sum(new)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    table, pages = R.make_pages(rng, [c + n for c, n in zip(ctx, new)], page, extra_pages=2)
    fused = torch.randn(T, heads + 2 * kv, D, generator=g).to(dtype).cuda()
    if strided:  # slices of one projection, and K and V in one cache tensor
        q, k, v = fused[:, :heads], fused[:, heads:heads + kv], fused[:, heads + kv:]
        both = _garbage((pages, 2, kv, page, D), cache)
        kc, vc = both[:, 0], both[:, 1]
    else:
        q, k, v = (x.contiguous() for x in (fused[:, :heads], fused[:, heads:heads + kv], fused[:, heads + kv:]))
        kc, vc = _garbage((pages, kv, page, D), cache), _garbage((pages, kv, page, D), cache)
    before = _bits(kc).clone(), _bits(vc).clone()
    pos = [ctx[b] + i for b in range(B) for i in range(new[b])]
    given = None
    if positions == "tree":
        pos = [p // 2 + 3 for p in pos]
        given = _ints(pos)
    elif positions == "far":
        pos = [1_000_000_007 + 13 * i for i in range(T)]
        given = _ints(pos)
    out = paged.append(k, v, kc, vc, _ints(table).reshape(B, -1), _ints(cu), _ints(ctx), q=q if with_q else None, positions=given,
                       freq_base=base, rotary_dim=rotary, neox=neox, k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    rd = D if rotary is None else rotary
    kd, vd, qd = k.double().cpu(), v.double().cpu(), q.double().cpu()
    kg, vg = kc.float().double().cpu() * ks, vc.float().double().cpu() * vs

    def close(got, want, raw, t, scale=1.0):
        # |a| + |b| of the pair a value comes from
        size = torch.linalg.vector_norm(raw, dim=-1, keepdim=True)
        lim = HALF[t] * want.abs() + TINY[t] * scale + 1e-6 * size
        assert ((got - want).abs() <= lim).all(), ((got - want).abs() - lim).max()

    touched = set()
    for b in range(B):
        for i in range(new[b]):
            t, row = cu[b] + i, ctx[b] + i
            pg, slot = table[b][row // page], row % page
            touched.add((pg, slot))
            want = R.rotate(kd[t], pos[t], base, rd, neox)
            if cache == torch.float8_e4m3fn:
                want = want.clamp(-448 * ks, 448 * ks)
            close(kg[pg, :, slot], want, kd[t], cache, ks)
            vw = vd[t].clamp(-448 * vs, 448 * vs) if cache == torch.float8_e4m3fn else vd[t]
            lim = (HALF[cache] * vw.abs() + TINY[cache] * vs) if cache == torch.float8_e4m3fn else 0.0 * vw
            assert ((vg[pg, :, slot] - vw).abs() <= lim).all()
            if with_q:
                close(out[t].double().cpu(), R.rotate(qd[t], pos[t], base, rd, neox), qd[t], dtype)
    for c, old in ((kc, before[0]), (vc, before[1])):  # nothing else is touched
        same = (_bits(c) == old).reshape(pages, kv, page, -1).all(-1).all(1).cpu()
        for pg in range(pages):
            for slot in range(page):
                assert same[pg, slot] or (pg, slot) in touched, (pg, slot)


F16, BF16, E4 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F16, E4), (BF16, E4)])
def test_append_types(cuda, dtype, cache, neox):
    _check_append(1, 8, 2, 64, 16, [5, 0, 31], [1, 7, 3], dtype, cache, None, neox, ks=0.0625 if cache == E4 else 1.0,
                  vs=0.3 if cache == E4 else 1.0)


@pytest.mark.parametrize("D,rotary,neox", [(96, None, True), (96, 48, True), (96, 48, False), (128, 64, True), (256, None, False),
                                           (256, 256, True), (64, 0, False), (64, 20, True), (64, 12, False), (40, 10, False), (8, 2, True)])
def test_append_rotary_sizes(cuda, D, rotary, neox):
    _check_append(2, 3, 1, D, 32, [17, 2], [9, 1], F16, F16, rotary, neox)


@pytest.mark.parametrize("page", [1, 2, 8, 16, 128])
def test_append_pages(cuda, page):
    _check_append(3, 4, 2, 64, page, [0, 15, 16, 40], [2, 1, 17, 0], BF16, BF16, None, False, positions=None)


def test_append_far_positions_and_base(cuda):
    _check_append(4, 4, 2, 128, 16, [3], [6], F16, F16, None, True, base=500000.0, positions="far")


def test_append_strided_views(cuda):
    _check_append(5, 6, 3, 64, 16, [4, 9], [3, 5], F16, F16, None, False, strided=True)
    _check_append(6, 6, 3, 64, 16, [4, 9], [3, 5], BF16, E4, None, True, strided=True)


def test_append_without_queries_and_many_sequences(cuda):
    _check_append(7, 4, 2, 64, 16, [i % 19 for i in range(150)], [i % 3 for i in range(150)], F16, F16, None, False, with_q=False)


def test_append_many_tokens(cuda):
    """Enough tokens that a block takes every head of its token."""
    _check_append(8, 32, 8, 64, 64, [0, 100], [900, 300], F16, F16, None, False, positions=None)


@pytest.mark.parametrize("cache", [F16, E4])
def test_append_unaligned(cuda, cache):
    """Operands at odd elements take the element-wise kernel and give the aligned call's bits."""
    import paged
    g = torch.Generator().manual_seed(9)
    T, heads, kv, D, page = 5, 4, 2, 64, 16
    cu, ctx, table = _ints([0, 5]), _ints([14]), _ints([[2, 0]])
    x = torch.randn(T, heads + 2 * kv, D, generator=g).half().cuda()
    q, k, v = (t.contiguous() for t in x.split([heads, kv, kv], 1))

    def odd(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        return buf[1:].view(t.shape).copy_(t)

    res = []
    for shift in (lambda t: t, odd):
        kc, vc = _garbage((3, kv, page, D), cache), _garbage((3, kv, page, D), cache)
        o = paged.append(shift(k), shift(v), kc, vc, table, cu, ctx, q=shift(q), k_scale=0.3 if cache == E4 else 1.0)
        res.append((o, _bits(kc), _bits(vc)))
    for a, b in zip(*res):
        assert torch.equal(a, b)


def test_append_in_place_saturation_and_nan(cuda):
    import paged
    D, page = 64, 16
    kc, vc = _garbage((1, 1, page, D), E4), _garbage((1, 1, page, D), E4)
    k = torch.full((1, 1, D), 3000.0, dtype=F16, device="cuda")
    v = k.clone()
    v[0, 0, 0], v[0, 0, 1], v[0, 0, 2] = float("inf"), float("-inf"), float("nan")
    q = torch.randn(1, 4, D, device="cuda").half()
    want = paged.append(k, v, kc, vc, _ints([[0]]), _ints([0, 1]), _ints([3]), q=q.clone(), neox=True)
    got = paged.append(k, v, kc, vc, _ints([[0]]), _ints([0, 1]), _ints([3]), q=q, q_out=q, neox=True, rotary_dim=None)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)
    row = vc[0, 0, 3].float().cpu()
    assert row[0] == 448 and row[1] == -448 and row[2].isnan() and (row[3:] == 448).all()


def test_append_skips_bad_pages(cuda):
    """Pages outside the pool and rows past the table are not written; the others are."""
    import paged
    D, page = 64, 16
    kc, vc = _garbage((2, 1, page, D), F16), _garbage((2, 1, page, D), F16)
    k = torch.ones(40, 1, D, dtype=F16, device="cuda")
    q = torch.randn(40, 2, D, device="cuda").half()
    out = paged.append(k, k, kc, vc, _ints([[1, 7]]), _ints([0, 40]), _ints([4]), q=q, rotary_dim=0)
    assert torch.equal(out, q)
    assert kc[0].isnan().all() and (kc[1, 0, 4:] == 1).all() and kc[1, 0, :4].isnan().all() and (vc[1, 0, 4:] == 1).all()


@pytest.mark.parametrize("dtype,D,page", [(F16, 128, 16), (BF16, 96, 32), (E4, 64, 1), (E4, 8, 16)])
def test_commit_path(cuda, dtype, D, page):
    import paged
    rng = random.Random(11)
    layers, kv = 3, 2
    ctx, new = [0, 13, 30, 7, 2], [9, 80, 4, 0, 100]
    paths = [[0, 2, 3, 8], [0, 1, 2, 40], [1, 2], [], list(range(0, 100, 2)) + list(range(99, 100))]
    steps = max(map(len, paths))
    table, pages = R.make_pages(rng, [c + n for c, n in zip(ctx, new)], page, 1)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    k, v = (torch.randn(layers, pages, kv, page, D, device="cuda").to(dtype) for _ in range(2))
    wk, wv = _bits(k).clone(), _bits(v).clone()
    for b, path in enumerate(paths):
        for w, src in ((wk, _bits(k).clone()), (wv, _bits(v).clone())):
            for j, node in enumerate(path):
                d, s = ctx[b] + j, ctx[b] + node
                w[:, table[b][d // page], :, d % page] = src[:, table[b][s // page], :, s % page]
    lens = paged.commit_path(k, v, _ints(table), _ints(cu), _ints(ctx), _ints([p + [-1] * (steps - len(p)) for p in paths]))
    assert lens.tolist() == [c + len(p) for c, p in zip(ctx, paths)]
    assert torch.equal(_bits(k), wk) and torch.equal(_bits(v), wv)


def test_commit_path_bad_entries(cuda):
    """Nodes that the sequence does not have are skipped and not counted; bad pages are left alone."""
    import paged
    k = torch.randn(1, 2, 1, 16, 64, device="cuda").half()
    want = k.clone()
    want[0, 0, 0, 2] = want[0, 0, 0, 3]
    lens = paged.commit_path(k, k, _ints([[0, 9]]), _ints([0, 20]), _ints([1]), _ints([[0, 2, 20, -5, 18]]))
    assert lens.tolist() == [4] and torch.equal(k, want)


@pytest.mark.parametrize("dtype,page,D", [(F16, 16, 128), (E4, 32, 96), (BF16, 2, 64), (E4, 1, 8)])
def test_reorder(cuda, dtype, page, D):
    import beam
    rng = random.Random(12)
    layers, kv, S, W = 2, 3, 3, 4
    lens = [rng.randint(0, 50) for _ in range(S * W)]
    lens[0], lens[1] = 16, 0
    table, pages = R.make_pages(rng, [n + 1 for n in lens], page, S * W)
    used = {p for row in table for p in row}
    free = [p for p in range(pages) if p not in used]
    parents = [[rng.randrange(W) for _ in range(W)] for _ in range(S)]
    parents[0] = [1, 0, 0, 3]
    fresh = [free[i * W:(i + 1) * W] for i in range(S)]
    k, v = (torch.randn(layers, pages, kv, page, D, device="cuda").to(dtype) for _ in range(2))
    wk, wv = _bits(k).clone(), _bits(v).clone()
    wt, wl = [], []
    for i in range(S * W):
        src = i // W * W + parents[i // W][i % W]
        full, held = divmod(lens[src], page)
        wt.append([table[src][p] if p < full else fresh[i // W][i % W] if p == full else -1 for p in range(len(table[0]))])
        wl.append(lens[src])
        for w in (wk, wv):
            w[:, fresh[i // W][i % W], :, :held] = w[:, table[src][full], :, :held]
    nt, nl = beam.reorder(k, v, _ints(table), _ints(lens), _ints(parents), _ints(fresh))
    assert nt.tolist() == wt and nl.tolist() == wl
    assert torch.equal(_bits(k), wk) and torch.equal(_bits(v), wv)


def test_reorder_strided_cache(cuda):
    """K and V interleaved in one tensor, a table with room behind it."""
    import beam
    both = torch.randn(2, 6, 2, 1, 16, 64, device="cuda").half()
    k, v = both[:, :, 0], both[:, :, 1]
    want = both.clone()
    want[:, 4, :, :, :5], want[:, 5, :, :, :5] = both[:, 3, :, :, :5], both[:, 3, :, :, :5]
    wide = torch.full((2, 8), 77, dtype=torch.int32, device="cuda")
    wide[:, :2] = _ints([[0, 2], [1, 3]])
    nt, nl = beam.reorder(k, v, wide[:, :2], _ints([18, 21]), _ints([[1, 1]]), _ints([[4, 5]]))
    assert nt.tolist() == [[1, 4], [1, 5]] and nl.tolist() == [21, 21] and torch.equal(both, want)
