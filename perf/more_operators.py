"""Performance cases of serving long, shared and growing contexts over the paged key/value cache, through the
framework's public entry points.

  append  queries and keys normalised head by head and rotated, by one position or by one of several axes
          for each pair, and keys and values written into their pages, in one pass (paged.append);
  shared  attention of a batch whose groups of sequences share their first rows, which are read once for a
          group (paged.shared_attention);
  weigh   attention that also sums the softmax weights which every cached row gets, over the tokens and the
          heads of a kv head (paged.weighted_attention);
  evict   the rows of the largest sums kept, with the first and the last ones, and copied into fresh pages,
          for every layer, sequence and kv head (paged.evict).

With `own` false, `run` computes the same with elementary torch operations in 32 bits (angles in 64);
`exact` recomputes a case in float64, sequence by sequence.

A cache is [pages, kv heads, page size, head dim] for K and for V (with a leading layer axis where every
layer is touched); a block table is [sequences, pages of the longest], int32.
"""

import math
import os
import random
import sys

import torch

own = False

_REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4, "e4m3": 1}
_E4M3_MAX = 448.0
_EPS = 1e-6


def _package():
    """The framework's module (imported where `own` is true only)."""
    path = os.path.join(_REPO, "gfx1150-inference_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import paged

    return paged


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------


def listed():
    return [
        # one decode step of an 8B model for eight users: one token each, queries and keys normalised
        {"name": "append_norm_b8_n1", "kind": "append", "B": 8, "n": 1, "ctx": 1500, "heads": 32, "kv": 8, "D": 128, "page": 16,
         "type": "f16", "cache": "f16", "rotary": 128, "neox": True, "base": 1000000.0, "axes": 1, "mixed": False, "ragged": True},
        # prompts with images, positions of three axes in runs of pairs, an fp8 cache
        {"name": "append_axes3_b3_n700_e4m3", "kind": "append", "B": 3, "n": 700, "ctx": 90, "heads": 16, "kv": 4, "D": 128, "page": 32,
         "type": "bf16", "cache": "e4m3", "rotary": 128, "neox": True, "base": 1000000.0, "axes": 3, "mixed": False, "ragged": True},
        # video prompts of a 70B model: four chunks of up to 2048 tokens, the axes in turn from pair to pair
        {"name": "append_axes3_b4_n2048", "kind": "append", "B": 4, "n": 2048, "ctx": 0, "heads": 64, "kv": 8, "D": 128, "page": 64,
         "type": "bf16", "cache": "bf16", "rotary": 128, "neox": False, "base": 500000.0, "axes": 3, "mixed": True, "ragged": True},
        # eight users of an 8B model behind one system prompt
        {"name": "shared_b8_p1024", "kind": "shared", "B": 8, "G": 1, "n": 1, "P": 1024, "ctx": 200, "heads": 32, "kv": 8, "D": 128, "page": 16,
         "type": "f16", "cache": "f16", "tree": False, "ragged": True},
        # sixty-four users of a 70B model who ask about one long document
        {"name": "shared_b64_p16384", "kind": "shared", "B": 64, "G": 1, "n": 1, "P": 16384, "ctx": 1500, "heads": 64, "kv": 8, "D": 128,
         "page": 16, "type": "bf16", "cache": "bf16", "tree": False, "ragged": True},
        # beam search: sixteen sentences of eight beams, each sentence's beams behind its own prompt
        {"name": "shared_beams_g16_b128_p1000", "kind": "shared", "B": 128, "G": 16, "n": 1, "P": 1000, "ctx": 60, "heads": 32, "kv": 8,
         "D": 128, "page": 16, "type": "f16", "cache": "f16", "tree": False, "ragged": True},
        # drafted trees of users in three groups, each group behind its own documents in an fp8 cache
        {"name": "shared_trees21_g3_b12_p32768_e4m3", "kind": "shared", "B": 12, "G": 3, "n": 21, "P": 32768, "ctx": 700, "heads": 32,
         "kv": 8, "D": 128, "page": 64, "type": "f16", "cache": "e4m3", "tree": True, "ragged": True},
        # one decode step of an 8B model for one user whose cache is kept short by its weights
        {"name": "weigh_b1_n1_ctx4096", "kind": "weigh", "B": 1, "n": 1, "ctx": 4095, "heads": 32, "kv": 8, "D": 128, "page": 16,
         "type": "f16", "cache": "f16", "tree": False, "ragged": False},
        # batched decode of a 70B model at contexts of very different lengths
        {"name": "weigh_b16_n1_ctx16384", "kind": "weigh", "B": 16, "n": 1, "ctx": 16384, "heads": 64, "kv": 8, "D": 128, "page": 32,
         "type": "bf16", "cache": "bf16", "tree": False, "ragged": True},
        # chunks of two prompts: every token of a chunk adds its weights
        {"name": "weigh_b2_n600_ctx1500", "kind": "weigh", "B": 2, "n": 600, "ctx": 1500, "heads": 32, "kv": 8, "D": 128, "page": 16,
         "type": "f16", "cache": "f16", "tree": False, "ragged": True},
        # one user's cache cut to a third, in all 32 layers of an 8B model
        {"name": "evict_b1_ctx3000_keep1024", "kind": "evict", "B": 1, "ctx": 3000, "keep": 1024, "recent": 256, "sinks": 4, "kv": 8, "D": 128,
         "page": 16, "cache": "f16", "layers": 32, "ragged": False},
        # twelve users of very different contexts, eight layers at a time; some are short enough to keep all
        {"name": "evict_b12_ctx8192_keep2048", "kind": "evict", "B": 12, "ctx": 8192, "keep": 2048, "recent": 1024, "sinks": 4, "kv": 8,
         "D": 128, "page": 32, "cache": "bf16", "layers": 8, "ragged": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["append", "shared", "shared", "weigh", "weigh", "evict"])
    heads, kv = rng.choice([(32, 8), (64, 8), (32, 32), (16, 2), (12, 4), (8, 1)])
    D = rng.choice([64, 96, 128, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    typ = rng.choice(["f16", "bf16"])
    cache = rng.choice([typ, typ, "e4m3"])
    case = {"kind": kind, "kv": kv, "D": D, "page": page, "cache": cache, "ragged": rng.random() < 0.7}
    if kind == "evict":
        ctx, layers, B = _log(rng, 200, 16384), _log(rng, 1, 32), _log(rng, 1, 24)
        keep = max(64, round(ctx * rng.uniform(0.1, 0.7)))
        while B * layers * ctx * kv * D > 12 * 8 * 8192 * 8 * 128:
            B, layers = (B + 1) // 2, max(1, layers // 2)
            if B * layers == 1:
                ctx, keep = ctx // 2, max(64, keep // 2)
        return case | {"B": B, "ctx": ctx, "layers": layers, "keep": keep, "recent": rng.randint(0, keep // 2), "sinks": rng.randint(0, 8)}
    case |= {"heads": heads, "type": typ}
    if kind == "append":
        n, B = rng.choice([1, _log(rng, 1, 64), _log(rng, 1, 2048)]), _log(rng, 1, 64)
        limit = 4 * 2048 * 80 * 128  # values of q, k and v of the largest listed case
        while B > 1 and B * n * (heads + 2 * kv) * D > limit:
            B = (B + 1) // 2
        n = min(n, limit // (B * (heads + 2 * kv) * D))
        return case | {"B": B, "n": n, "ctx": _log(rng, 1, 8000), "neox": rng.random() < 0.5, "rotary": rng.choice([D, D, D // 2]),
                       "base": rng.choice([10000.0, 500000.0]), "axes": rng.choice([1, 2, 3, 3]), "mixed": rng.random() < 0.5}
    n, tree = rng.choice([(1, False), (1, False), (_log(rng, 2, 40), True), (_log(rng, 2, 512), False)])
    most = 64 * 17900 * 64 * 128  # products of the largest listed case of decoding, a quarter of them
    if kind == "shared":
        n = min(n, 64)
        G = rng.choice([1, 1, 2, _log(rng, 1, 16)])
        B, P, ctx = G * _log(rng, 2, 32), _log(rng, 64, 32768), _log(rng, 16, 2000)
        while B * n * (P + ctx + n) * heads * D > most or (G * P + B * ctx) * kv * D > 64 * 2000 * 8 * 128:
            B, P, ctx = max(G, B // 2 // G * G), P // 2 + 1, ctx // 2 + 1
        return case | {"B": B, "G": G, "n": n, "P": max(P, page), "ctx": ctx, "tree": tree}
    ctx, B = _log(rng, 16, 32768), _log(rng, 1, 32)
    while B * n * (ctx + n) * heads * D > most // 4 or B * ctx * kv * D > 16 * 16384 * 8 * 128:
        B, ctx = (B + 1) // 2, ctx // 2 + 1 if B <= 2 else ctx
    return case | {"B": B, "n": n, "ctx": ctx, "tree": tree}


def _lens(case):
    """(context lengths, counts of new tokens) of a case's sequences: its sizes decide them, not the seed.  With
    shared rows the context is what a sequence has behind them."""
    B, n, ctx = case["B"], case.get("n", 1), case["ctx"]
    if not case.get("ragged"):
        return [ctx] * B, [n] * B
    r = random.Random(B * 1000003 + n * 10007 + ctx)
    c = [ctx] + [r.randint(ctx // 16, ctx) for _ in range(B - 1)]
    m = [n] + [r.randint((n + 1) // 2, n) for _ in range(B - 1)]
    return c, m


def _groups(case):
    """(first sequence of each group and the end, shared rows of each group)"""
    B, G, P = case["B"], case["G"], case["P"]
    members = -(-B // G)
    r = random.Random(B * 10007 + P)
    return [min(g * members, B) for g in range(G + 1)], [P] + [r.randint(P // 3, P) for _ in range(G - 1)]


def _axes(case):
    """The axis that each pair turns by: runs of pairs, the first axis the shortest, or the axes in turn."""
    half, A = case["rotary"] // 2, case["axes"]
    if case["mixed"]:
        return [i % A for i in range(half)]
    first = half // 4 if A > 1 else half
    return [0 if i < first else 1 + (i - first) * (A - 1) // (half - first) for i in range(half)]


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------


def _tree(r, n):
    """Parents of a random drafted tree (node 0 is its root; parents come before their children)."""
    return [-1] + [r.randint(max(0, i - 1 - i // 2), max(0, i // 2)) if i > 1 else 0 for i in range(1, n)]


def _ancestors(parents, words):
    """One row of 32-bit words per node: the bits of the node itself and of its ancestors."""
    rows = []
    for i, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else 0) | (1 << i))
    signed = lambda w: w - (1 << 32) if w >> 31 else w  # noqa: E731
    return [[signed((x >> (32 * w)) & 0xFFFFFFFF) for w in range(words)] for x in rows]


def _random_cache(g, shape, name):
    x = torch.empty(shape, dtype=torch.float16, device="cuda").normal_(generator=g)
    return x if name == "f16" else x.to(_TYPES[name])


def prepare(case, seed):
    r = random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    normal = lambda shape, t: torch.empty(shape, dtype=torch.float32, device="cuda").normal_(generator=g).to(_TYPES[t])  # noqa: E731
    kv, D, page, kind = case["kv"], case["D"], case["page"], case["kind"]
    ctx, new = _lens(case)
    B, T = case["B"], sum(new)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    shared = [0] * B  # pages that a sequence shares
    s = {"case": case}
    if kind == "shared":
        first, rows = _groups(case)
        for i, p in enumerate(rows):
            for b in range(first[i], first[i + 1]):
                ctx[b] += p
                shared[b] = p // page  # as a server shares: whole pages; the rows of the open one are the sequence's own
        s |= {"groups": ints(first), "shared": ints([p // page * page for p in rows])}
    # block tables over pages in random order; -1 past a sequence's own
    rows = ctx if kind == "evict" else [c + n for c, n in zip(ctx, new)]
    need = [max(1, -(-x // page)) for x in rows]
    width, kept = max(need), -(-case.get("keep", 0) // page)
    lead = [b if kind != "shared" else max(f for f in first[:-1] if f <= b) for b in range(B)]
    ids = list(range(sum(k - (p if f != b else 0) for b, (k, p, f) in enumerate(zip(need, shared, lead))) + B * kept))
    r.shuffle(ids)
    table, at = [], 0
    for b in range(B):
        head = table[lead[b]][:shared[b]] if lead[b] != b else []
        own_pages = need[b] - len(head)
        table.append(head + ids[at:at + own_pages] + [-1] * (width - need[b]))
        at += own_pages
    s |= {"cu": ints(cu), "ctx": ints(ctx), "table": ints(table), "T": T, "max_new": max(new)}
    shape = (len(ids), kv, page, D)
    if kind == "evict":
        shape = (case["layers"],) + shape
        s["fresh"] = ints(ids[at:]).reshape(B, kept)
        # sums of attention weights: a few rows hold most, many hold next to nothing, some nothing at all
        w = normal((case["layers"], B, kv, width * page), "f32").mul_(2.5).exp_()
        s["weights"] = torch.where(w < 0.01, torch.zeros_like(w), w)
    else:
        heads = case["heads"]
        s["q"] = normal((T, heads, D), case["type"]) * 2
        if kind == "append":
            s |= {"k": normal((T, kv, D), case["type"]) * 3, "v": normal((T, kv, D), case["type"]), "q_out": torch.empty_like(s["q"]),
                  "q_norm": (1 + 0.2 * normal((D,), "f32")).to(_TYPES[case["type"]]), "k_norm": (1 + 0.2 * normal((D,), "f32")).to(_TYPES[case["type"]])}
            # frames of 24 x 18 patches behind each other: time, height and width of every token
            place = [c + i for c, n in zip(ctx, new) for i in range(n)]
            grid = [place, [p // 24 % 18 + p // 432 for p in place], [p % 24 + p // 432 for p in place]]
            s["positions"] = ints([[p // 432 for p in place]] + grid[1:case["axes"]]) if case["axes"] > 1 else ints(place)
            s["axes"] = _axes(case) if case["axes"] > 1 else None
        else:
            s |= {"out": torch.empty_like(s["q"]), "mask": None}
            if case["tree"]:
                words = -(-max(new) // 32)
                s["mask"] = ints([row for n in new for row in _ancestors(_tree(r, n), words)])
            if kind == "weigh":
                s["weights"] = normal((B, kv, width * page), "f32").abs_()
                s["weights_out"] = torch.zeros_like(s["weights"])
    # the scales of an fp8 cache are the model's constants; powers of two here
    s |= {"k_scale": 0.0625 if case["cache"] == "e4m3" else 1.0, "v_scale": 0.03125 if case["cache"] == "e4m3" else 1.0}
    return s | {"k_cache": _random_cache(g, shape, case["cache"]), "v_cache": _random_cache(g, shape, case["cache"])}


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------


def run(s):
    return {"append": _append, "shared": _shared, "weigh": _weigh, "evict": _evict}[s["case"]["kind"]](s)


def _sequence_of(cu, T):
    """(sequence, place within its new tokens) of every token."""
    t = torch.arange(T, device=cu.device)
    seq = torch.searchsorted(cu[1:].long(), t, right=True)
    return seq, t - cu.long()[seq]


def _bits(t):
    """The tensor whose indexing moves whole elements (fp8 as bytes)."""
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _stored(x, scale, dtype):
    return (x / scale).clamp(-_E4M3_MAX, _E4M3_MAX).to(dtype) if dtype == torch.float8_e4m3fn else x.to(dtype)


def _append(s):
    c = s["case"]
    if own:
        _package().append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["ctx"], q=s["q"], q_out=s["q_out"],
                          positions=s["positions"], freq_base=c["base"], rotary_dim=c["rotary"], neox=c["neox"], k_scale=s["k_scale"],
                          v_scale=s["v_scale"], q_norm=s["q_norm"], k_norm=s["k_norm"], norm_eps=_EPS, axes=s["axes"])
        return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    rotary, half = c["rotary"], c["rotary"] // 2
    inv = c["base"] ** (-torch.arange(0, rotary, 2, device=s["q"].device, dtype=torch.float64) / rotary)
    if s["axes"] is None:
        pos = s["positions"].double()[:, None]
    else:
        pos = s["positions"].double()[torch.tensor(s["axes"], device=s["q"].device)].T
    angle = pos * inv
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x, weight):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * weight.float()
        a, b = (x[..., :half], x[..., half:rotary]) if c["neox"] else (x[..., 0:rotary:2], x[..., 1:rotary:2])
        u, w = a * cos - b * sin, a * sin + b * cos
        y = torch.cat([u, w], -1) if c["neox"] else torch.stack([u, w], -1).flatten(-2)
        return torch.cat([y, x[..., rotary:]], -1)

    seq, off = _sequence_of(s["cu"], s["T"])
    at = s["ctx"].long()[seq] + off
    page, slot = s["table"].long()[seq, at // c["page"]], at % c["page"]
    head = torch.arange(c["kv"], device=at.device)
    where = (page[:, None], head[None], slot[:, None])
    _bits(s["k_cache"])[where] = _bits(_stored(turned(s["k"], s["k_norm"]), s["k_scale"], s["k_cache"].dtype))
    _bits(s["v_cache"])[where] = _bits(_stored(s["v"].float(), s["v_scale"], s["v_cache"].dtype))
    s["q_out"].copy_(turned(s["q"], s["q_norm"]))
    return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _gathered(s, cache, scale, table):
    """[batch, kv heads, rows, D] in 32 bits: the rows of each row of a table."""
    x = _bits(cache)[table.long().clamp(min=0)].view(cache.dtype).float() * scale
    return x.transpose(1, 2).reshape(table.shape[0], s["case"]["kv"], -1, s["case"]["D"])


def _new_rows(s):
    """Queries [batch, kv heads, new tokens * group, D] of every sequence, padded, and the token of each."""
    c = s["case"]
    cu, group = s["cu"].long(), c["heads"] // c["kv"]
    token = (cu[:-1, None] + torch.arange(s["max_new"], device=cu.device)).clamp(max=s["T"] - 1)
    q = s["q"][token].float().reshape(c["B"], s["max_new"], c["kv"], group, c["D"]).transpose(1, 2)
    return q.reshape(c["B"], c["kv"], -1, c["D"]), token


def _seen(s, rows, token):
    """[batch, new tokens, rows]: the rows of its sequence that a new token sees."""
    n, cu = s["max_new"], s["cu"].long()
    i = torch.arange(n, device=cu.device)
    j = torch.arange(rows, device=cu.device) - s["ctx"].long()[:, None]  # place among the new tokens
    if s["mask"] is None:
        seen = j[:, None] <= i[:, None]
    else:
        word = s["mask"][token].gather(2, (j.clamp(min=0) // 32).clamp(max=s["mask"].shape[1] - 1)[:, None].expand(-1, n, -1))
        seen = (j[:, None] < 0) | (((word >> (j.clamp(min=0) % 32)[:, None]) & 1) == 1)
    return seen & (j < (cu[1:] - cu[:-1])[:, None])[:, None]


def _per_head(x, group):
    """[batch, new tokens, rows] for the rows of queries [batch, 1, new tokens * group, rows]."""
    return x[:, None, :, None].expand(-1, 1, -1, group, -1).reshape(x.shape[0], 1, -1, x.shape[2])


def _outputs(s, out):
    c = s["case"]
    out = out.reshape(c["B"], c["kv"], s["max_new"], -1, c["D"]).transpose(1, 2).reshape(c["B"], s["max_new"], c["heads"], c["D"])
    return s["out"].copy_(out[_sequence_of(s["cu"], s["T"])])


def _shared(s):
    c = s["case"]
    if own:
        return _package().shared_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["ctx"], s["groups"], s["shared"],
                                           mask=s["mask"], max_new=s["max_new"], k_scale=s["k_scale"], v_scale=s["v_scale"], out=s["out"])
    B, G, page, kv, D, group = c["B"], c["G"], c["page"], c["kv"], c["D"], c["heads"] // c["kv"]
    q, token = _new_rows(s)
    scale = 1.0 / math.sqrt(D)
    members, rows = -(-B // G), q.shape[2]
    first = s["groups"].long()[:-1].clamp(max=B - 1)
    lead = torch.arange(B, device=q.device) // members  # the group of a sequence
    member = (first[:, None] + torch.arange(members, device=q.device)).clamp(max=B - 1)
    full = (c["P"] // page) * page
    limit = s["shared"].long()
    # the shared rows once for a group, for all of its sequences' queries
    common = s["table"][first][:, :full // page]
    k = _gathered(s, s["k_cache"], s["k_scale"], common)
    qg = q[member].transpose(1, 2).reshape(G, kv, members * rows, D)
    hidden = torch.arange(full, device=q.device) >= limit[:, None]
    score = (qg @ k.transpose(2, 3)).mul_(scale).masked_fill_(hidden[:, None, None], -math.inf)
    score = score.reshape(G, kv, members, rows, full).transpose(1, 2)
    score = score.reshape(G * members, kv, rows, full)[:B]
    # the other rows of every sequence
    width = s["table"].shape[1]
    start = limit[lead] // page
    column = start[:, None] + torch.arange(-(-(c["ctx"] + page + c["n"]) // page), device=q.device)
    tail = s["table"].gather(1, column.clamp(max=width - 1))
    ko = _gathered(s, s["k_cache"], s["k_scale"], tail)
    # a tail's rows count from `start`: those of the whole sequence, picked out
    seen = _seen(s, width * page, token)
    at = (column[:, :, None] * page + torch.arange(page, device=q.device)).flatten(1)
    inside = (column < width)[:, :, None].expand(-1, -1, page).flatten(1)
    seen = seen.gather(2, at.clamp(max=width * page - 1)[:, None].expand(-1, seen.shape[1], -1)) & inside[:, None]
    tail_score = (q @ ko.transpose(2, 3)).mul_(scale).masked_fill_(~_per_head(seen, group), -math.inf)
    top = torch.maximum(score.amax(-1, keepdim=True), tail_score.amax(-1, keepdim=True))
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p, pt = score.sub(top).exp_(), tail_score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True) + pt.sum(-1, keepdim=True)
    v = _gathered(s, s["v_cache"], s["v_scale"], common)
    if G * members > B:
        p = torch.cat([p, p.new_zeros((G * members - B,) + p.shape[1:])])
    pg = p.reshape(G, members, kv, rows, full).transpose(1, 2).reshape(G, kv, members * rows, full)
    out = (pg @ v).reshape(G, kv, members, rows, D).transpose(1, 2).reshape(G * members, kv, rows, D)[:B]
    out = out + pt @ _gathered(s, s["v_cache"], s["v_scale"], tail)
    return _outputs(s, torch.where(total > 0, out / total, torch.zeros_like(out)))


def _weigh(s):
    c = s["case"]
    if own:
        out, weights = _package().weighted_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["ctx"], s["weights"],
                                                     weights_out=s["weights_out"], mask=s["mask"], max_new=s["max_new"],
                                                     k_scale=s["k_scale"], v_scale=s["v_scale"], out=s["out"])
        return {"out": out, "weights": weights}
    q, token = _new_rows(s)
    k = _gathered(s, s["k_cache"], s["k_scale"], s["table"])
    live = torch.arange(s["max_new"], device=q.device) < (s["cu"][1:] - s["cu"][:-1])[:, None]
    seen = _seen(s, k.shape[2], token) & live[:, :, None]
    score = (q @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(c["D"])).masked_fill_(~_per_head(seen, c["heads"] // c["kv"]), -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total > 0, total, torch.ones_like(total))
    # a new row's sum starts, a cached one's goes on; nothing behind a sequence's rows is touched
    j, ctx = torch.arange(k.shape[2], device=q.device), s["ctx"][:, None, None]
    sums = p.sum(2) + torch.where(j < ctx, s["weights"], torch.zeros_like(s["weights"]))
    held = ctx + (s["cu"][1:] - s["cu"][:-1])[:, None, None]
    s["weights_out"].copy_(torch.where(j < held, sums, s["weights_out"]))
    return {"out": _outputs(s, p @ _gathered(s, s["v_cache"], s["v_scale"], s["table"])), "weights": s["weights_out"]}


def _evict(s):
    c = s["case"]
    if own:
        table, lens, weights = _package().evict(s["k_cache"], s["v_cache"], s["table"], s["ctx"], s["weights"], s["fresh"], c["keep"],
                                                recent=c["recent"], sinks=c["sinks"])
        return {"table": table, "lens": lens, "weights": weights, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    keep, page, ctx, w = c["keep"], c["page"], s["ctx"].long(), s["weights"]
    width = s["table"].shape[1]
    j = torch.arange(w.shape[3], device=w.device)
    cut = ctx > keep
    last = ctx[:, None, None]
    # the first and the last rows come before every weight; a stable sort leaves equal ones in their order
    rank = torch.where((j < c["sinks"]) | (j >= last - c["recent"]), math.inf, w).masked_fill(j >= last, -math.inf)
    rows = rank.sort(dim=-1, descending=True, stable=True).indices[..., :keep].sort(dim=-1).values
    if rows.shape[-1] < keep:  # no context reaches `keep`
        rows = torch.cat([rows, rows.new_zeros(rows.shape[:-1] + (keep - rows.shape[-1],))], -1)
    rows = torch.where(cut[:, None, None], rows, torch.arange(keep, device=w.device))
    lens = ctx.clamp(max=keep)
    place = torch.arange(keep, device=w.device)
    kept = w.gather(3, rows.clamp(max=w.shape[3] - 1)).masked_fill(place >= lens[:, None, None], 0.0)
    weights = torch.zeros_like(w)
    weights[..., :min(keep, w.shape[3])] = kept[..., :w.shape[3]]
    fresh = torch.cat([s["fresh"], s["fresh"].new_full((c["B"], width), -1)], 1)[:, :width]
    table = torch.where(cut[:, None], fresh, s["table"])
    which = cut.nonzero().squeeze(1)
    rows = rows[:, which]
    layer = torch.arange(c["layers"], device=w.device)[:, None, None, None]
    head = torch.arange(c["kv"], device=w.device)[:, None]
    source = s["table"].long()[which][:, None].expand(-1, c["kv"], -1)[None].expand(c["layers"], -1, -1, -1).gather(3, rows // page)
    target = s["fresh"].long()[which][:, place // page][None, :, None].expand_as(rows)
    for cache in (s["k_cache"], s["v_cache"]):
        x = _bits(cache)
        x[layer, target, head, (place % page).expand_as(rows)] = x[layer, source, head, rows % page]
    return {"table": table, "lens": lens.int(), "weights": weights, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------


def work(case):
    kv, D, page, eb = case["kv"], case["D"], case["page"], _BYTES[case["cache"]]
    ctx, new = _lens(case)
    T = sum(new)
    if case["kind"] == "evict":
        kept = sum(case["keep"] for c in ctx if c > case["keep"])
        weights = case["layers"] * kv * (sum(ctx) + sum(min(c, case["keep"]) for c in ctx)) * 4
        return {"bytes": 2 * 2 * kept * case["layers"] * kv * D * eb + weights, "flops": 0}
    heads, qb = case["heads"], _BYTES[case["type"]]
    if case["kind"] == "append":
        return {"bytes": T * D * (2 * heads * qb + 2 * kv * (qb + eb)) + 4 * T * case["axes"], "flops": T * (heads + kv) * (3 * case["rotary"] + 4 * D)}
    words = -(-max(new) // 32) if case["tree"] else 0
    inner = sum(n if case["tree"] else n * (n + 1) // 2 for n in new)
    pairs = sum(n * c for c, n in zip(ctx, new)) + inner
    rows, extra = sum(ctx) + T, 0
    if case["kind"] == "shared":
        first, shared = _groups(case)
        pairs += sum(p * sum(new[a:b]) for p, a, b in zip(shared, first, first[1:]))
        whole = [p // page * page for p in shared]
        rows += sum(whole) + sum((p - w) * (b - a) for p, w, a, b in zip(shared, whole, first, first[1:]))
    else:
        extra = 4 * kv * (2 * sum(ctx) + T)
    return {"bytes": 2 * rows * kv * D * eb + 2 * T * heads * D * qb + 4 * T * words + extra, "flops": 4 * pairs * heads * D}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits, one sequence at a time
# ---------------------------------------------------------------------------------------------


def _rows(cache, table, page, upto):
    """[upto, kv heads, D] in float64: the first rows of one sequence."""
    pages = torch.tensor([table[i // page] for i in range(upto)], device="cuda")
    slots = torch.arange(upto, device="cuda") % page
    return _bits(cache)[pages, :, slots].view(cache.dtype).double()


def exact(case, seed):
    s = prepare(case, seed)
    kind, page, D, kv = case["kind"], case["page"], case["D"], case["kv"]
    table, ctx = s["table"].tolist(), s["ctx"].tolist()
    if kind == "evict":
        k, v = s["k_cache"].double(), s["v_cache"].double()
        weights = torch.zeros_like(s["weights"], dtype=torch.float64)
        fresh = s["fresh"].tolist()
        for b in range(case["B"]):
            if ctx[b] <= case["keep"]:
                weights[:, b, :, :ctx[b]] = s["weights"][:, b, :, :ctx[b]].double()
                continue
            a, z = case["sinks"], ctx[b] - case["recent"]
            pages = torch.tensor(table[b], device="cuda")
            to = torch.arange(case["keep"], device="cuda")
            target = torch.tensor(fresh[b], device="cuda")[to // page]
            for layer in range(case["layers"]):
                for h in range(kv):
                    w = s["weights"][layer, b, h, :ctx[b]].double()
                    order = torch.argsort(-w[a:z], stable=True)[:case["keep"] - a - case["recent"]]
                    keep = torch.zeros(ctx[b], dtype=torch.bool, device="cuda")
                    keep[:a] = keep[z:] = True
                    keep[a + order] = True
                    rows = keep.nonzero()[:, 0]
                    weights[layer, b, h, :case["keep"]] = w[rows]
                    for x, old in ((k, s["k_cache"]), (v, s["v_cache"])):
                        x[layer, target, h, to % page] = _bits(old)[layer, pages[rows // page], h, rows % page].view(old.dtype).double()
        return {"table": None, "lens": None, "weights": weights, "k_cache": k, "v_cache": v}
    _, new = _lens(case)
    starts = s["cu"].tolist()
    if kind == "append":
        k, v = s["k_cache"].double(), s["v_cache"].double()
        half = case["rotary"] // 2
        freq = torch.tensor([case["base"] ** (-2.0 * i / case["rotary"]) for i in range(half)], device="cuda", dtype=torch.float64)
        place = s["positions"].double().reshape(-1, s["T"])
        turn = torch.stack([place[s["axes"][i] if s["axes"] else 0] * freq[i] for i in range(half)], 1)
        unit = torch.polar(torch.ones_like(turn), turn)[:, None]

        def rotate(x, weight):
            x = x.double()
            x = x / ((x ** 2).sum(-1, keepdim=True) / D + _EPS) ** 0.5 * weight.double()
            first = slice(0, half) if case["neox"] else slice(0, 2 * half, 2)
            second = slice(half, 2 * half) if case["neox"] else slice(1, 2 * half, 2)
            z = torch.complex(x[..., first], x[..., second]) * unit
            x[..., first], x[..., second] = z.real, z.imag
            return x

        limit = _E4M3_MAX if case["cache"] == "e4m3" else math.inf
        kr, vr = (rotate(s["k"], s["k_norm"]) / s["k_scale"]).clamp(-limit, limit), (s["v"].double() / s["v_scale"]).clamp(-limit, limit)
        for b in range(case["B"]):
            at = range(ctx[b], ctx[b] + new[b])
            pages = torch.tensor([table[b][i // page] for i in at], device="cuda")
            slots = torch.tensor([i % page for i in at], device="cuda")
            k[pages, :, slots] = kr[starts[b]:starts[b + 1]]
            v[pages, :, slots] = vr[starts[b]:starts[b + 1]]
        return {"q": rotate(s["q"], s["q_norm"]), "k_cache": k, "v_cache": v}
    out = torch.zeros(s["T"], case["heads"], D, dtype=torch.float64, device="cuda")
    group = case["heads"] // kv
    weights = s["weights_out"].double() if kind == "weigh" else None
    for b in range(case["B"]):
        n, total = new[b], ctx[b] + new[b]
        k, v = _rows(s["k_cache"], table[b], page, total) * s["k_scale"], _rows(s["v_cache"], table[b], page, total) * s["v_scale"]
        hidden = torch.zeros(n, total, dtype=torch.bool, device="cuda")
        if s["mask"] is None:
            hidden[:, ctx[b]:] = ~torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        else:
            words = s["mask"][starts[b]:starts[b + 1]].tolist()
            hidden[:, ctx[b]:] = torch.tensor([[not (row[j // 32] >> (j % 32)) & 1 for j in range(n)] for row in words], device="cuda")
        for g in range(kv):
            q = s["q"][starts[b]:starts[b + 1], g * group:(g + 1) * group].double().transpose(0, 1).reshape(group * n, D)
            score = q @ k[:, g].T.contiguous() / math.sqrt(D)
            score = torch.softmax(score.reshape(group, n, total).masked_fill(hidden, -math.inf), -1)
            out[starts[b]:starts[b + 1], g * group:(g + 1) * group] = (score.reshape(group * n, total) @ v[:, g].contiguous()).reshape(group, n, D).transpose(0, 1)
            if weights is not None:
                weights[b, g, :total] = score.sum((0, 1))
                weights[b, g, :ctx[b]] += s["weights"][b, g, :ctx[b]].double()
    return {"out": out, "weights": weights} if kind == "weigh" else out
