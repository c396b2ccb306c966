"""Performance cases of the paged key/value cache's operators, through the framework's public entry points.

Four operators of serving over a cache that is cut into pages:
  append  new keys and values rotated by their positions and written into their pages, the queries
          rotated in the same pass (paged.append);
  attn    attention of each sequence's new tokens over its cached ones and over those of the new
          tokens that a bit mask lets each see: a drafted tree, or a plain chain without a mask
          (paged.tree_attention);
  commit  the rows of the accepted path of a drafted tree moved to the front, in every layer
          (paged.commit_path);
  beam    one step of beam search: selection over beams and vocabulary (beam.select), then block
          tables and open pages reordered by the chosen parents (beam.reorder).

With `own` false, `run` computes the same with elementary torch operations in 32 bits (angles and
the beams' scores in 64); `exact` recomputes a case in float64, sequence by sequence.

A cache is [pages, kv heads, page size, head dim] for K and for V (with a leading layer axis where
every layer is touched); a block table is [sequences, pages of the longest], int32.
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


def _package():
    """The framework's modules (imported where `own` is true only)."""
    path = os.path.join(_REPO, "gfx1150-inference_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import beam
    import paged

    return paged, beam


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------


def listed():
    return [
        # one decode step of an 8B model for eight users: the cache write of one token each
        {"name": "append_8b_b8_n1", "kind": "append", "B": 8, "n": 1, "ctx": 1500, "heads": 32, "kv": 8, "D": 128, "page": 16,
         "type": "f16", "cache": "f16", "rotary": 128, "neox": False, "base": 500000.0, "ragged": True},
        # drafted trees of an fp8 cache: sixteen users, 24 nodes each
        {"name": "append_8b_b16_n24_e4m3", "kind": "append", "B": 16, "n": 24, "ctx": 4100, "heads": 32, "kv": 8, "D": 128, "page": 32,
         "type": "bf16", "cache": "e4m3", "rotary": 128, "neox": True, "base": 500000.0, "ragged": True},
        # prompts of a 70B model: four chunks of up to 2048 tokens
        {"name": "append_70b_b4_n2048", "kind": "append", "B": 4, "n": 2048, "ctx": 0, "heads": 64, "kv": 8, "D": 128, "page": 64,
         "type": "f16", "cache": "f16", "rotary": 128, "neox": False, "base": 10000.0, "ragged": True},
        # single-user decode of an 8B model: one token against a context of 1024
        {"name": "attn_8b_b1_n1_ctx1024", "kind": "attn", "B": 1, "n": 1, "ctx": 1023, "heads": 32, "kv": 8, "D": 128, "page": 16,
         "type": "f16", "cache": "f16", "tree": False, "ragged": False},
        # batched decode of a 70B model: contexts of very different lengths
        {"name": "attn_70b_b32_n1_ctx16384", "kind": "attn", "B": 32, "n": 1, "ctx": 16384, "heads": 64, "kv": 8, "D": 128, "page": 16,
         "type": "bf16", "cache": "bf16", "tree": False, "ragged": True},
        # a drafted tree of 63 nodes for each of eight users of a 70B model
        {"name": "attn_70b_b8_tree63_ctx8191", "kind": "attn", "B": 8, "n": 63, "ctx": 8191, "heads": 64, "kv": 8, "D": 128, "page": 32,
         "type": "f16", "cache": "f16", "tree": True, "ragged": True},
        # small trees against long contexts in an fp8 cache
        {"name": "attn_8b_b4_tree13_ctx32768_e4m3", "kind": "attn", "B": 4, "n": 13, "ctx": 32768, "heads": 32, "kv": 8, "D": 128,
         "page": 64, "type": "f16", "cache": "e4m3", "tree": True, "ragged": True},
        # chunks of a prompt (a chain, no mask) of a model of head_dim 64
        {"name": "attn_d64_b3_n500_ctx1700", "kind": "attn", "B": 3, "n": 500, "ctx": 1700, "heads": 32, "kv": 8, "D": 64, "page": 128,
         "type": "f16", "cache": "f16", "tree": False, "ragged": True},
        # one user's accepted path through the 80 layers of a 70B model
        {"name": "commit_70b_b1_n26", "kind": "commit", "B": 1, "n": 26, "ctx": 700, "kv": 8, "D": 128, "page": 16, "cache": "f16",
         "layers": 80, "path": 5, "ragged": False},
        # the same for 48 users of an 8B model with an fp8 cache
        {"name": "commit_8b_b48_n40_e4m3", "kind": "commit", "B": 48, "n": 40, "ctx": 90, "kv": 8, "D": 128, "page": 32, "cache": "e4m3",
         "layers": 32, "path": 7, "ragged": True},
        # beam search of one sentence: four beams, a small vocabulary, fp32 logits
        {"name": "beam_b1_w4_v32000", "kind": "beam", "B": 1, "W": 4, "V": 32000, "logits": "f32", "ctx": 77, "kv": 8, "D": 128, "page": 16,
         "cache": "f16", "layers": 4},
        # sixteen sentences of eight beams over the 8B vocabulary, all 32 layers' open pages
        {"name": "beam_b16_w8_v128256", "kind": "beam", "B": 16, "W": 8, "V": 128256, "logits": "f16", "ctx": 230, "kv": 8, "D": 128,
         "page": 16, "cache": "f16", "layers": 32},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["append", "attn", "attn", "attn", "commit", "beam"])
    heads, kv = rng.choice([(32, 8), (64, 8), (32, 32), (16, 2), (12, 4), (8, 1)])
    D = rng.choice([64, 96, 128, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    typ = rng.choice(["f16", "bf16"])
    cache = rng.choice([typ, typ, "e4m3"])
    case = {"kind": kind, "kv": kv, "D": D, "page": page, "cache": cache}
    if kind in ("append", "attn"):
        case |= {"heads": heads, "type": typ, "ragged": rng.random() < 0.7}
    if kind == "append":
        n = rng.choice([1, _log(rng, 1, 64), _log(rng, 1, 2048)])
        B = _log(rng, 1, 64)
        limit = 4 * 2048 * 80 * 128  # values of q, k and v of the largest listed case
        while B > 1 and B * n * (heads + 2 * kv) * D > limit:
            B = (B + 1) // 2
        n = min(n, limit // (B * (heads + 2 * kv) * D))
        return case | {"B": B, "n": n, "ctx": _log(rng, 1, 8000), "neox": rng.random() < 0.5, "rotary": rng.choice([D, D, D // 2]),
                       "base": rng.choice([10000.0, 500000.0])}
    if kind == "attn":
        n, tree = rng.choice([(1, False), (_log(rng, 2, 16), True), (_log(rng, 8, 128), True), (_log(rng, 2, 512), False)])
        ctx, B = _log(rng, 16, 32768), _log(rng, 1, 48)
        # no more cached values, and no more products, than the largest listed cases
        while B > 1 and (B * ctx * kv * D > 32 * 16384 * 8 * 128 or B * n * (ctx + n) * heads * D > 8 * 63 * 8191 * 64 * 128):
            B = (B + 1) // 2
        while B * n * (ctx + n) * heads * D > 8 * 63 * 8191 * 64 * 128 or B * ctx * kv * D > 32 * 16384 * 8 * 128:
            ctx = ctx // 2 + 1
        return case | {"B": B, "n": n, "ctx": ctx, "tree": tree}
    if kind == "commit":
        n = _log(rng, 4, 64)
        B, layers = _log(rng, 1, 48), _log(rng, 4, 80)
        while B > 1 and B * layers * kv * D * _BYTES[cache] > 48 * 32 * 8 * 128:
            B = (B + 1) // 2
        while layers * B * kv * D * _BYTES[cache] > 48 * 32 * 8 * 128:
            layers = (layers + 1) // 2
        return case | {"B": B, "n": n, "ctx": _log(rng, 1, 200), "layers": layers, "path": rng.randint(2, min(n // 2, 9)), "ragged": rng.random() < 0.7}
    W = rng.choice([1, 2, 3, 4, 5, 8, 16])
    B, V = _log(rng, 1, 16), _log(rng, 1000, 128256)
    while B * W > 128:
        B = (B + 1) // 2
    layers = _log(rng, 1, 32)
    while layers > 1 and B * W * layers * kv * D * page * _BYTES[cache] > 128 * 32 * 8 * 128 * 16 * 2:
        layers = (layers + 1) // 2
    return case | {"B": B, "W": W, "V": V, "logits": rng.choice(["f16", "bf16", "f32"]), "ctx": _log(rng, 1, 300), "layers": layers}


def _lens(case):
    """(context lengths, counts of new tokens) of a case's sequences: its sizes decide them, not the seed."""
    B, n, ctx = case["B"], case.get("n", 1), case["ctx"]
    if not case.get("ragged"):
        return [ctx] * B, [n] * B
    r = random.Random(B * 1000003 + n * 10007 + ctx)
    c = [ctx] + [r.randint(ctx // 16, ctx) for _ in range(B - 1)]
    m = [n] + [r.randint((n + 1) // 2, n) for _ in range(B - 1)]
    return c, m


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


def _pages(r, lens, page, width):
    """Block tables over pages in random order; -1 past a sequence's own."""
    need = [max(1, -(-x // page)) for x in lens]
    ids = list(range(sum(need)))
    r.shuffle(ids)
    table, at = [], 0
    for k in need:
        table.append(ids[at:at + k] + [-1] * (width - k))
        at += k
    return torch.tensor(table, dtype=torch.int32, device="cuda"), at


def prepare(case, seed):
    r = random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    normal = lambda shape, t: torch.empty(shape, dtype=torch.float32, device="cuda").normal_(generator=g).to(_TYPES[t])  # noqa: E731
    kv, D, page = case["kv"], case["D"], case["page"]
    s = {"case": case}
    if case["kind"] == "beam":
        B, W, V, layers = case["B"], case["W"], case["V"], case["layers"]
        # every sentence's beams share the full pages of its prompt; each has its own open page and a spare one
        ctx = [case["ctx"] + (5 * b) % page for b in range(B)]
        full = [c // page for c in ctx]
        total = sum(full) + 2 * B * W
        ids = list(range(total))
        r.shuffle(ids)
        width = max(full) + 2
        rows, at, fresh = [], 0, []
        for b in range(B):
            shared = ids[at:at + full[b]]
            at += full[b]
            for _ in range(W):
                rows.append(shared + [ids[at]] + [-1] * (width - full[b] - 1))
                fresh.append(ids[at + 1])
                at += 2
        logits = normal((B, W, V), "f32") * 2.5
        logits[:, :, ::997] += 4.0
        s |= {"logits": logits.to(_TYPES[case["logits"]]), "scores": normal((B, W), "f32").abs() * -3.0,
              "table": ints(rows), "lens": ints([c for c in ctx for _ in range(W)]), "fresh": ints(fresh).reshape(B, W)}
        shape = (layers, total, kv, page, D)
        return s | {"k_cache": _random_cache(g, shape, case["cache"]), "v_cache": _random_cache(g, shape, case["cache"])}
    ctx, new = _lens(case)
    B, T = case["B"], sum(new)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    width = max(-(-(c + n) // page) for c, n in zip(ctx, new))
    table, pages = _pages(r, [c + n for c, n in zip(ctx, new)], page, width)
    s |= {"cu": ints(cu), "ctx": ints(ctx), "table": table, "T": T, "max_new": max(new)}
    shape = (pages, kv, page, D)
    if case["kind"] == "commit":
        paths = []
        for n in new:
            # an ascending path whose targets are no sources of later steps' rows, so that a pass can be repeated
            k = min(case["path"], n)
            tail = sorted(r.sample(range(k, n), min(k - 1, n - k))) if n > k else []
            path = [0] + tail
            paths.append(path + [-1] * (case["path"] - len(path)))
        s["path"] = ints(paths)
        shape = (case["layers"],) + shape
    else:
        heads = case["heads"]
        s["q"] = normal((T, heads, D), case["type"]) * 2
        if case["kind"] == "append":
            s |= {"k": normal((T, kv, D), case["type"]), "v": normal((T, kv, D), case["type"]), "q_out": torch.empty_like(s["q"])}
            depth = [c + min(i, 6 + i % 3) if case["n"] <= 64 else c + i for c, n in zip(ctx, new) for i in range(n)]
            s["positions"] = ints(depth)
        else:
            s |= {"out": torch.empty_like(s["q"]), "mask": None}
            if case["tree"]:
                words = -(-max(new) // 32)
                s["mask"] = ints([row for n in new for row in _ancestors(_tree(r, n), words)])
    # the scales of an fp8 cache are the model's constants; powers of two here
    s |= {"k_scale": 0.0625 if case["cache"] == "e4m3" else 1.0, "v_scale": 0.03125 if case["cache"] == "e4m3" else 1.0}
    return s | {"k_cache": _random_cache(g, shape, case["cache"]), "v_cache": _random_cache(g, shape, case["cache"])}


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------


def run(s):
    return {"append": _append, "attn": _attention, "commit": _commit, "beam": _beam}[s["case"]["kind"]](s)


def _sequence_of(cu, T):
    """(sequence, place within its new tokens) of every token."""
    t = torch.arange(T, device=cu.device)
    seq = torch.searchsorted(cu[1:].long(), t, right=True)
    return seq, t - cu.long()[seq]


def _rotated(x, positions, rotary, base, neox):
    inv = base ** (-torch.arange(0, rotary, 2, device=x.device, dtype=torch.float64) / rotary)
    angle = positions.double()[:, None] * inv
    c, sn = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = x.float()
    a, b = (x[..., :rotary // 2], x[..., rotary // 2:rotary]) if neox else (x[..., 0:rotary:2], x[..., 1:rotary:2])
    u, w = a * c - b * sn, a * sn + b * c
    r = torch.cat([u, w], -1) if neox else torch.stack([u, w], -1).flatten(-2)
    return torch.cat([r, x[..., rotary:]], -1)


def _bits(t):
    """The tensor whose indexing moves whole elements (fp8 as bytes)."""
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _stored(x, scale, dtype):
    return (x / scale).clamp(-_E4M3_MAX, _E4M3_MAX).to(dtype) if dtype == torch.float8_e4m3fn else x.to(dtype)


def _append(s):
    c = s["case"]
    if own:
        paged, _ = _package()
        paged.append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["ctx"], q=s["q"], q_out=s["q_out"],
                     positions=s["positions"], freq_base=c["base"], rotary_dim=c["rotary"], neox=c["neox"], k_scale=s["k_scale"],
                     v_scale=s["v_scale"])
        return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    seq, off = _sequence_of(s["cu"], s["T"])
    at = s["ctx"].long()[seq] + off
    page, slot = s["table"].long()[seq, at // c["page"]], at % c["page"]
    head = torch.arange(c["kv"], device=at.device)
    where = (page[:, None], head[None], slot[:, None])
    k = _rotated(s["k"], s["positions"], c["rotary"], c["base"], c["neox"])
    _bits(s["k_cache"])[where] = _bits(_stored(k, s["k_scale"], s["k_cache"].dtype))
    _bits(s["v_cache"])[where] = _bits(_stored(s["v"].float(), s["v_scale"], s["v_cache"].dtype))
    s["q_out"].copy_(_rotated(s["q"], s["positions"], c["rotary"], c["base"], c["neox"]))
    return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attention(s):
    c = s["case"]
    if own:
        paged, _ = _package()
        return paged.tree_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["ctx"], mask=s["mask"],
                                    max_new=s["max_new"], k_scale=s["k_scale"], v_scale=s["v_scale"], out=s["out"])
    B, n, heads, kv, D = c["B"], s["max_new"], c["heads"], c["kv"], c["D"]
    cu, ctx, group = s["cu"].long(), s["ctx"].long(), heads // kv
    new = cu[1:] - cu[:-1]
    gather = lambda cache, scale: (_bits(cache)[s["table"].long().clamp(min=0)].view(cache.dtype).float() * scale).transpose(1, 2).reshape(B, kv, -1, D)  # noqa: E731
    k, v = gather(s["k_cache"], s["k_scale"]), gather(s["v_cache"], s["v_scale"])
    i = torch.arange(n, device=cu.device)
    token = (cu[:-1, None] + i).clamp(max=s["T"] - 1)  # [B, n]
    q = s["q"][token].float().reshape(B, n, kv, group, D).transpose(1, 2).reshape(B, kv, n * group, D)
    j = torch.arange(k.shape[2], device=cu.device) - ctx[:, None]  # [B, keys]: place among the new tokens
    if s["mask"] is None:
        seen = j[:, None] <= i[:, None]
    else:
        word = s["mask"][token].gather(2, (j.clamp(min=0) // 32).clamp(max=s["mask"].shape[1] - 1)[:, None].expand(B, n, -1))
        seen = (j[:, None] < 0) | (((word >> (j.clamp(min=0) % 32)[:, None]) & 1) == 1)
    seen = (seen & (j < new[:, None])[:, None])[:, None, :, None].expand(B, 1, n, group, -1).reshape(B, 1, n * group, -1)
    score = (q @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(D)).masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.where(total > 0, (p @ v) / total, torch.zeros_like(total))
    out = out.reshape(B, kv, n, group, D).transpose(1, 2).reshape(B, n, heads, D)
    seq, off = _sequence_of(s["cu"], s["T"])
    return s["out"].copy_(out[seq, off])


def _commit(s):
    c = s["case"]
    if own:
        paged, _ = _package()
        lens = paged.commit_path(s["k_cache"], s["v_cache"], s["table"], s["cu"], s["ctx"], s["path"])
        return {"lens": lens, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    path, ctx = s["path"].long(), s["ctx"].long()
    B, A = path.shape
    live = path >= 0
    step = torch.arange(A, device=path.device).expand(B, A)
    src = ctx[:, None] + torch.where(live, path, step)  # a step past the path's end keeps its own row
    dst = ctx[:, None] + step
    last = s["table"].shape[1] * c["page"] - 1
    src, dst = src.clamp(max=last), dst.clamp(max=last)
    place = lambda at: (s["table"].long().gather(1, at // c["page"]).clamp(min=0).reshape(-1), (at % c["page"]).reshape(-1))  # noqa: E731
    (sp, ss), (dp, ds) = place(src), place(torch.where(live, dst, src))
    for cache in (s["k_cache"], s["v_cache"]):
        x = _bits(cache)
        x[:, dp, :, ds] = x[:, sp, :, ss]
    return {"lens": (ctx + live.sum(1)).int(), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _beam(s):
    c = s["case"]
    if own:
        _, beam = _package()
        scores, parents, tokens = beam.select(s["logits"], s["scores"])
        table, lens = beam.reorder(s["k_cache"], s["v_cache"], s["table"], s["lens"], parents, s["fresh"])
    else:
        B, W, V = s["logits"].shape
        x = s["logits"].double()
        x = x - x.amax(-1, keepdim=True)
        x = s["scores"].double()[..., None] + x - x.exp().sum(-1, keepdim=True).log()
        scores, flat = x.reshape(B, W * V).sort(stable=True, dim=-1, descending=True)
        scores, flat = scores[:, :W].float(), flat[:, :W]
        parents, tokens = (flat // V).int(), (flat % V).int()
        source = (torch.arange(B, device=flat.device)[:, None] * W + parents).reshape(-1)
        lens = s["lens"][source]
        full = lens.long() // c["page"]
        old = s["table"][source]
        column = torch.arange(old.shape[1], device=old.device)
        fresh = s["fresh"].reshape(-1)
        table = torch.where(column < full[:, None], old, torch.where(column == full[:, None], fresh[:, None], -torch.ones_like(old)))
        tail = old.long().gather(1, full[:, None])[:, 0]
        held = (torch.arange(c["page"], device=old.device) < (lens.long() % c["page"])[:, None])[None, :, None, :, None]
        for cache in (s["k_cache"], s["v_cache"]):
            b = _bits(cache)
            b[:, fresh.long()] = torch.where(held, b[:, tail], b[:, fresh.long()])
    return {"scores": scores, "parents": parents, "tokens": tokens, "table": table, "lens": lens, "k_cache": s["k_cache"],
            "v_cache": s["v_cache"]}


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------


def work(case):
    kv, D, page, eb = case["kv"], case["D"], case["page"], _BYTES[case["cache"]]
    if case["kind"] == "beam":
        B, W, V = case["B"], case["W"], case["V"]
        held = sum((case["ctx"] + (5 * b) % page) % page for b in range(B)) * W
        moved = 2 * 2 * held * case["layers"] * kv * D * eb
        return {"bytes": B * W * V * _BYTES[case["logits"]] + moved + B * W * (4 + 12), "flops": 3 * B * W * V}
    ctx, new = _lens(case)
    T = sum(new)
    if case["kind"] == "commit":
        steps = sum(min(case["path"], n, 1 + max(0, n - case["path"])) - 1 for n in new)
        return {"bytes": 2 * 2 * max(1, steps) * case["layers"] * kv * D * eb, "flops": 0}
    heads, qb = case["heads"], _BYTES[case["type"]]
    if case["kind"] == "append":
        return {"bytes": T * D * (2 * heads * qb + 2 * kv * (qb + eb)) + 4 * T, "flops": 3 * T * (heads + kv) * case["rotary"]}
    words = -(-max(new) // 32) if case["tree"] else 0
    pairs = sum(n * c + (n if case["tree"] else n * (n + 1) // 2) for c, n in zip(ctx, new))
    return {"bytes": 2 * (sum(ctx) + T) * kv * D * eb + 2 * T * heads * D * qb + 4 * T * words, "flops": 4 * pairs * heads * D}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits, one sequence at a time
# ---------------------------------------------------------------------------------------------


def _rows(cache, table, page, upto):
    """[upto, kv heads, D] in float64: the first rows of one sequence."""
    at = range(upto)
    pages = torch.tensor([table[i // page] for i in at], device="cuda")
    slots = torch.tensor([i % page for i in at], device="cuda")
    if cache.dtype == torch.float8_e4m3fn:
        return cache.view(torch.uint8)[pages, :, slots].view(torch.float8_e4m3fn).double()
    return cache[pages, :, slots].double()


def exact(case, seed):
    s = prepare(case, seed)
    kind, page, D, kv = case["kind"], case["page"], case["D"], case["kv"]
    table = s["table"].tolist()
    if kind == "beam":
        W, V = case["W"], case["V"]
        scores, parents = [], []
        for b in range(case["B"]):
            rows = torch.stack([s["scores"][b, w].double() + torch.log_softmax(s["logits"][b, w].double(), -1) for w in range(W)])
            best, at = rows.reshape(-1).topk(W)
            scores.append(best)
            parents.append([i // V for i in at.tolist()])
        k, v = s["k_cache"].double(), s["v_cache"].double()
        fresh, lens = s["fresh"].tolist(), s["lens"].tolist()
        for b in range(case["B"]):
            for w in range(W):
                src = b * W + parents[b][w]
                full, held = divmod(lens[src], page)
                for new, old in ((k, s["k_cache"]), (v, s["v_cache"])):
                    new[:, fresh[b][w], :, :held] = old[:, table[src][full], :, :held].double()
        return {"scores": torch.stack(scores), "parents": None, "tokens": None, "table": None, "lens": None, "k_cache": k, "v_cache": v}
    ctx, new = _lens(case)
    starts = s["cu"].tolist()
    if kind == "commit":
        k, v = s["k_cache"].double(), s["v_cache"].double()
        for b, path in enumerate(s["path"].tolist()):
            for j, node in enumerate(p for p in path if p >= 0):
                (dp, ds), (sp, ss) = ((table[b][i // page], i % page) for i in (ctx[b] + j, ctx[b] + node))
                for x, old in ((k, s["k_cache"]), (v, s["v_cache"])):
                    x[:, dp, :, ds] = old[:, sp, :, ss].double()
        return {"lens": None, "k_cache": k, "v_cache": v}
    if kind == "append":
        k, v = s["k_cache"].double(), s["v_cache"].double()
        half = case["rotary"] // 2
        turn = s["positions"].double()[:, None] * torch.tensor([case["base"] ** (-2.0 * i / case["rotary"]) for i in range(half)], device="cuda", dtype=torch.float64)
        unit = torch.polar(torch.ones_like(turn), turn)[:, None]

        def rotate(x):
            x = x.double().clone()
            first = slice(0, half) if case["neox"] else slice(0, 2 * half, 2)
            second = slice(half, 2 * half) if case["neox"] else slice(1, 2 * half, 2)
            z = torch.complex(x[..., first], x[..., second]) * unit
            x[..., first], x[..., second] = z.real, z.imag
            return x

        limit = _E4M3_MAX if case["cache"] == "e4m3" else math.inf
        kr, vr = (rotate(s["k"]) / s["k_scale"]).clamp(-limit, limit), (s["v"].double() / s["v_scale"]).clamp(-limit, limit)
        for b in range(case["B"]):
            at = range(ctx[b], ctx[b] + new[b])
            pages = torch.tensor([table[b][i // page] for i in at], device="cuda")
            slots = torch.tensor([i % page for i in at], device="cuda")
            k[pages, :, slots] = kr[starts[b]:starts[b + 1]]
            v[pages, :, slots] = vr[starts[b]:starts[b + 1]]
        return {"q": rotate(s["q"]), "k_cache": k, "v_cache": v}
    out = torch.zeros(s["T"], case["heads"], D, dtype=torch.float64, device="cuda")
    group = case["heads"] // kv
    for b in range(case["B"]):
        n, total = new[b], ctx[b] + new[b]
        k, v = _rows(s["k_cache"], table[b], page, total) * s["k_scale"], _rows(s["v_cache"], table[b], page, total) * s["v_scale"]
        hidden = torch.zeros(n, total, dtype=torch.bool, device="cuda")
        if s["mask"] is None:
            hidden[:, ctx[b]:] = ~torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        else:
            words = s["mask"][starts[b]:starts[b + 1]].tolist()
            hidden[:, ctx[b]:] = torch.tensor([[not (row[j // 32] >> (j % 32)) & 1 for j in range(n)] for row in words], device="cuda")
        for h in range(case["heads"]):
            score = s["q"][starts[b]:starts[b + 1], h].double() @ k[:, h // group].T.contiguous() / math.sqrt(D)
            score[hidden] = -math.inf
            out[starts[b]:starts[b + 1], h] = torch.softmax(score, -1) @ v[:, h // group].contiguous()
    return out
