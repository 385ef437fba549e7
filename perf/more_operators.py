"""What a language model's server runs around the attention of drafted tokens, as measurable cases.

Five kinds of pass, each an operator of fusedkernellibrary_amd.attention:

  tables  a step's tables from its requests' lengths: page table, slots, positions and, of trees, what sees what
  axes    RMS norm of query and key heads and rotation by positions of several axes (time, height, width); with "cache" into the
          pages of a cache, from where the new tokens' keys and values are read back
  attend  attention over the cache's pages whose scores are capped by a tanh or get a bias by distance, or whose rows see
          no key in front of a window or of their document, or all of a prefix
  verify  drafted tokens against the target's probabilities, by given random numbers, and the token behind them
  keep    the cache rows of the accepted tokens, moved to where the sequence goes on

The cache: keys [pages, kv_heads, page, dim] and values [pages, kv_heads, page / 4, dim, 4] as int8 or e4m3 codes, one float32
scale per token and head ([pages, kv_heads, page]); a value is code * scale, scale = max |x| of the row / 127 (448 for e4m3).
Sequence b has context[b] tokens in the cache before its new ones; token j of it lives in page page_table[b, j // page], and
its new tokens are rows q_start[b] to q_start[b + 1]. parents[row] is the new token that a new token follows, counted from the
sequence's first (which has -1). Lengths are spread evenly between "lo" and "hi" and dealt to the sequences by the seed.
"""
import functools
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
EPS = 1e-6


def listed():
    return [
        # the step of a few conversations, one token each, in a batch that is padded to 20 rows
        {"name": "tables_16x1", "kind": "tables", "batch": 16, "new_lo": 1, "new": 1, "lo": 10, "hi": 4000, "page": 64, "tree": False, "padding": 4},
        # 200 requests with trees of up to 61 drafted tokens
        {"name": "tables_200_trees_61", "kind": "tables", "batch": 200, "new_lo": 13, "new": 61, "lo": 500, "hi": 4100, "page": 32, "tree": True, "padding": 0},
        # one frame's tokens of one conversation, seven query heads to a key head
        {"name": "axes_64", "kind": "axes", "cache": False, "tokens": 64, "hq": 28, "hkv": 4, "dim": 128, "rot": 128, "layout": "sections", "pairs": False, "type": "bf16", "table": 4096},
        # a prompt with a video, odd length, the axes' frequencies dealt out in turn
        {"name": "axes_8191", "kind": "axes", "cache": False, "tokens": 8191, "hq": 32, "hkv": 8, "dim": 128, "rot": 128, "layout": "cycle", "pairs": False, "type": "bf16", "table": 8192},
        # 64 conversations with one token each, contexts of all lengths, capped scores
        {"name": "attend_64x8k_cap", "kind": "attend", "batch": 64, "new_lo": 1, "new": 1, "lo": 900, "hi": 8191, "hq": 32, "hkv": 8, "dim": 128, "page": 64, "codes": "int8", "type": "bf16", "tree": False, "cap": 50.0, "bias": False, "window": 0, "documents": 0, "prefix": 0},
        # small trees behind long contexts, of which a window is seen, scores biased by distance
        {"name": "attend_16_trees_window_bias", "kind": "attend", "batch": 16, "new_lo": 3, "new": 13, "lo": 30000, "hi": 65003, "hq": 32, "hkv": 8, "dim": 128, "page": 64, "codes": "e4m3", "type": "bf16", "tree": True, "cap": 0.0, "bias": True, "window": 4096, "documents": 0, "prefix": 0},
        # a chunk of a prompt behind a prefix that sees itself whole, three documents one behind the other, capped scores, half precision
        {"name": "attend_prompt_2048", "kind": "attend", "batch": 1, "new_lo": 2048, "new": 2048, "lo": 1500, "hi": 1500, "hq": 32, "hkv": 8, "dim": 128, "page": 64, "codes": "e4m3", "type": "f16", "tree": False, "cap": 30.0, "bias": False, "window": 0, "documents": 3, "prefix": 1777},
        # four tokens drafted for one conversation, a small vocabulary
        {"name": "verify_1x5_32000", "kind": "verify", "batch": 1, "new_lo": 5, "new": 5, "vocab": 32000, "draft": True, "tree": False, "type": "f32"},
        # trees of drafted tokens without probabilities of their own, an odd vocabulary, 16 bits
        {"name": "verify_24_trees_29_100003", "kind": "verify", "batch": 24, "new_lo": 13, "new": 29, "vocab": 100003, "draft": False, "tree": True, "type": "bf16"},
        # 64 conversations with up to seven drafted tokens each, a large vocabulary
        {"name": "verify_64x8_131072", "kind": "verify", "batch": 64, "new_lo": 4, "new": 8, "vocab": 131072, "draft": True, "tree": False, "type": "f32"},
        # one layer's cache, a few trees
        {"name": "keep_8_trees_13", "kind": "keep", "batch": 8, "new_lo": 5, "new": 13, "lo": 100, "hi": 900, "hkv": 2, "dim": 64, "page": 16, "codes": "int8", "layers": 1},
        # the caches of 16 layers, trees of up to 29
        {"name": "keep_48_trees_29_layers_16", "kind": "keep", "batch": 48, "new_lo": 13, "new": 29, "lo": 50, "hi": 300, "hkv": 8, "dim": 128, "page": 32, "codes": "e4m3", "layers": 16},
    ]


HEADS = [(8, 2), (16, 16), (16, 2), (32, 8), (28, 4), (20, 20), (64, 8), (12, 4)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        # not above the largest listed cases, in traffic, in products of many rows or in what the inputs take
        if w["bytes"] <= 5.6e8 and w["flops"] <= 2.2e10 and _held(case) <= 1.1e9:
            return case


def _held(case):
    """About how many bytes the inputs, or the plain form's rows, have."""
    if case["kind"] == "verify":
        size = 4 if case["type"] == "f32" else 2
        return case["batch"] * (case["new_lo"] + case["new"]) / 2 * case["vocab"] * size * (2 if case["draft"] else 1)
    if case["kind"] == "keep":
        return case["layers"] * case["batch"] * ((case["lo"] + case["hi"]) / 2 + case["new"] + case["page"]) * case["hkv"] * 2 * (case["dim"] + 4)
    if case["kind"] == "attend":
        return case["batch"] * (case["hi"] + case["new"]) * case["hkv"] * case["dim"] * 2
    return 0


def _draw(rng):
    kind = rng.choice(["tables", "axes", "attend", "attend", "verify", "keep"])
    hq, hkv = rng.choice(HEADS)
    dim = rng.choice([64, 96, 128, 128, 192, 256])
    case = {"kind": kind}
    if kind == "axes":
        rot = rng.choice([dim, dim, dim // 2])
        case |= {"cache": rng.random() < 0.4, "tokens": _log(rng, 1, 8192), "hq": hq, "hkv": hkv, "dim": dim, "rot": rot, "layout": rng.choice(["sections", "cycle", "two"])}
        case |= {"pairs": rng.random() < 0.3, "type": rng.choice(["bf16", "f16"]), "table": 8192}
        return case | ({"page": rng.choice([16, 32, 64, 128]), "codes": rng.choice(["int8", "e4m3"])} if case["cache"] else {})
    if kind == "verify":
        chain = rng.random() < 0.6
        new = rng.randint(1, 9) if chain else rng.randint(2, 64)
        return case | {"batch": _log(rng, 1, 128), "new_lo": rng.randint(1, new), "new": new, "vocab": _log(rng, 1000, 160000), "draft": chain and rng.random() < 0.7, "tree": not chain,
                       "type": rng.choice(["f32", "f32", "bf16", "f16"])}
    page = rng.choice([16, 32, 64, 128])
    if kind == "tables":
        new = rng.choice([1, rng.randint(2, 64), _log(rng, 64, 2048)])
        return case | {"batch": _log(rng, 1, 1024 if new <= 16 else 256 if new <= 64 else 16), "new_lo": rng.randint(0, new), "new": new, "lo": rng.randint(0, 500), "hi": _log(rng, 500, 32768),
                       "page": page, "tree": 1 < new <= 64 and rng.random() < 0.7, "padding": rng.choice([0, 0, rng.randint(1, 40)])}
    if kind == "keep":
        new = rng.randint(2, 64)
        return case | {"batch": _log(rng, 1, 64), "new_lo": rng.randint(1, new), "new": new, "lo": rng.randint(0, 200), "hi": rng.randint(200, 1000), "hkv": hkv, "dim": dim, "page": page,
                       "codes": rng.choice(["int8", "e4m3"]), "layers": _log(rng, 1, 32)}
    new = rng.choice([1, 1, rng.randint(2, 64), _log(rng, 64, 2048)])
    tree = 1 < new <= 64 and rng.random() < 0.7
    hi = _log(rng, 16, 65536 if new <= 64 else 4096)
    documents = 0 if tree or rng.random() < 0.6 else rng.randint(2, 6)
    return case | {"batch": _log(rng, 1, 64) if new <= 64 else rng.randint(1, 3), "new_lo": rng.randint(1, new), "new": new, "lo": rng.randint(0, hi), "hi": hi, "hq": hq, "hkv": hkv, "dim": dim,
                   "page": page, "codes": rng.choice(["int8", "e4m3"]), "type": rng.choice(["bf16", "f16"]), "tree": tree, "cap": rng.choice([0.0, 30.0, 50.0, rng.uniform(5.0, 100.0)]),
                   "bias": rng.random() < 0.5, "window": 0 if documents or rng.random() < 0.5 else _log(rng, 16, 8192), "documents": documents,
                   "prefix": 0 if tree or rng.random() < 0.6 else _log(rng, 1, hi + new)}


def _spread(lo, hi, n):
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]


def _lengths(case):
    """(context, new tokens) of each sequence, before the seed deals them."""
    return list(zip(_spread(case.get("lo", 0), case.get("hi", 0), case["batch"]), reversed(_spread(case["new_lo"], case["new"], case["batch"]))))


def _first_seen(case, context, new):
    """The first key that a sequence's rows see, row by row, where nothing is drafted as a tree."""
    rows = range(context, context + new)
    if case["documents"]:
        starts = [(context + new) * i // case["documents"] for i in range(case["documents"])]
        return [max(s for s in starts if s <= j) for j in rows]
    return [max(0, j + 1 - case["window"]) if case["window"] else 0 for j in rows]


def _axes(case):
    """The axis of each pair's position: three runs of pairs, three axes in turn, or two halves."""
    pairs = case["rot"] // 2
    if case["layout"] == "two":
        return [int(i >= pairs // 2) for i in range(pairs)]
    if case["layout"] == "cycle":
        return [i % 3 if i < pairs - pairs // 8 else 0 for i in range(pairs)]
    return [0 if 4 * i < pairs else 1 if 8 * i < 5 * pairs else 2 for i in range(pairs)]


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _quantised(shape, codes, gen):
    """Rows of random keys or values, some elements of a head larger than the others, as codes and scales."""
    kind, top = CODES[codes]
    x = torch.randn(shape, device="cuda", generator=gen)
    x *= 1.0 + 3.0 * (torch.rand(shape[1], 1, shape[-1], device="cuda", generator=gen) > 0.96)
    scale = x.abs().amax(-1) / top
    x /= scale.unsqueeze(-1)
    return (x.round_() if codes == "int8" else x).to(kind), scale


def _cache(pages, hkv, page, dim, codes, gen):
    k, k_scale = _quantised((pages, hkv, page, dim), codes, gen)
    v, v_scale = _quantised((pages, hkv, page, dim), codes, gen)
    v = v.view(torch.int8).view(pages, hkv, page // 4, 4, dim).transpose(3, 4).contiguous().view(v.dtype)
    return k, v, k_scale, v_scale


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _page_table(needs, width, gen):
    """Rows of the pages that sequences have, in any order, and how many pages there are."""
    pages = sum(needs) + 3
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    table = torch.zeros((len(needs), width), dtype=torch.int32, device="cuda")
    row = torch.repeat_interleave(torch.arange(len(needs)), torch.tensor(needs)).cuda()
    starts = torch.tensor([sum(needs[:i]) for i in range(len(needs))]).cuda()
    table[row, torch.arange(sum(needs), device="cuda") - starts[row]] = order[: sum(needs)]
    return table, pages


def _trees(new, rng):
    """Parents of each sequence's new tokens, row by row: every one but the first continues one of those before it."""
    return [[-1] + [rng.randint(max(0, t - 5), t - 1) for t in range(1, n)] if n else [] for n in new]


def _depths(parents):
    depth = []
    for p in parents:
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return depth


def _mask_words(parents, words):
    """What each token of a tree sees, itself and its ancestors, as signed 64-bit words."""
    seen = []
    for t, p in enumerate(parents):
        seen.append((seen[p] if p >= 0 else 0) | 1 << t)
    return [[(s >> 64 * w & (1 << 64) - 1) - (1 << 64 if s >> 64 * w + 63 & 1 else 0) for w in range(words)] for s in seen]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 2654435761 % (1 << 40))
    rng = random.Random(seed)
    kind = case["kind"]

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    state = {"kind": kind}
    if kind == "axes":
        dtype, dim, hkv, hq, tokens, axes = TYPES[case["type"]], case["dim"], case["hkv"], case["hq"], case["tokens"], _axes(case)
        packed = randn(tokens, (hq + 2 * hkv) * dim).to(dtype).view(tokens, hq + 2 * hkv, dim)
        angle = torch.arange(case["table"], device="cuda").double()[:, None] * 10000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda").double() / case["rot"])
        state |= {"type": dtype, "pairs": case["pairs"], "q": packed[:, :hq], "k": packed[:, hq:hq + hkv], "v": packed[:, hq + hkv:], "axes": axes, "cos": angle.cos().float(), "sin": angle.sin().float(),
                  "positions": torch.randint(0, case["table"], (max(axes) + 1, tokens), dtype=torch.int32, device="cuda", generator=gen), "weights": [(1.0 + 0.2 * randn(dim)).to(dtype) for _ in range(2)]}
        if case["cache"]:
            page = case["page"]
            pages = -(-tokens // page) + 2
            state |= {"cache": _cache(pages, hkv, page, dim, case["codes"], gen), "slots": torch.randperm(pages * page, device="cuda", generator=gen)[:tokens].to(torch.int32)}
        return state
    lengths = _lengths(case)
    rng.shuffle(lengths)
    new, tokens = [n for _, n in lengths], sum(n for _, n in lengths)
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    parents = _trees(new, rng) if kind == "keep" or case["tree"] else None
    if kind == "tables":
        page, rows = case["page"], tokens + case["padding"]
        have, needs = [-(-c // page) for c, _ in lengths], [-(-(c + n) // page) for c, n in lengths]
        # (some hold a page more than their tokens fill: drafts that were refused had been in it)
        held = [h + (rng.random() < 0.2) for h in have]
        table, pages = _page_table(held, max(max(needs), max(have) + 1) + 2, gen)
        spare = sum(max(0, n - h) for n, h in zip(needs, held)) + rng.randint(0, 9)
        state |= {"page": page, "rows": rows, "most": max(1, max(new)), "page_table": table, "held": _ints(held), "context": _ints([c for c, _ in lengths]), "new": _ints(new)}
        state |= {"free": (pages + torch.randperm(spare + 7, device="cuda", generator=gen)).to(torch.int32), "available": _ints([spare])}
        if parents:
            state["parents"] = _ints([p for tree in parents for p in tree] + [-1] * case["padding"])
        return state
    if kind == "verify":
        return _to_verify(case, gen, rng, new, starts, parents)
    page, dim, hkv, batch = case["page"], case["dim"], case["hkv"], case["batch"]
    needs = [-(-(c + n) // page) for c, n in lengths]
    table, pages = _page_table(needs, max(needs), gen)
    state |= {"page_table": table, "context": _ints([c for c, _ in lengths]), "q_start": _ints(starts), "max_new": max(new), "max_context": max(c for c, _ in lengths)}
    if kind == "keep":
        # The accepted tokens: the first ones in order, as the likeliest continuation is drafted first, then some of the last.
        # (So none of the rows that move is where another goes, and a pass may be repeated.)
        path = torch.full((batch, max(new)), -1, dtype=torch.int32)
        count = []
        for b, n in enumerate(new):
            kept = rng.randint(1, min(n, 8))
            straight = rng.randint(1, kept)
            rest = sorted(rng.sample(range(kept, n), min(kept - straight, n - kept)))
            row = list(range(straight)) + rest
            count.append(len(row))
            path[b, : len(row)] = torch.tensor(row, dtype=torch.int32)
        return state | {"caches": [_cache(pages, hkv, page, dim, case["codes"], gen) for _ in range(case["layers"])], "path": path.cuda(), "count": _ints(count)}
    dtype, hq = TYPES[case["type"]], case["hq"]
    state |= {"type": dtype, "cache": _cache(pages, hkv, page, dim, case["codes"], gen), "q": (1.5 * randn(tokens, hq, dim)).to(dtype), "cap": case["cap"] or None}
    depths = [_depths(p) for p in parents] if parents else [list(range(n)) for n in new]
    if parents:
        words = -(-max(new) // 64)
        state["mask"] = torch.tensor([w for p in parents for w in _mask_words(p, words)], dtype=torch.int64, device="cuda").view(tokens, words)
        state["positions"] = _ints([c + d for (c, _), tree in zip(lengths, depths) for d in tree])
    if case["bias"]:
        state["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], dtype=torch.float32, device="cuda")
    if case["window"] and parents:
        state["first"] = _ints([max(0, c + d + 1 - case["window"]) for (c, _), tree in zip(lengths, depths) for d in tree])
    elif case["window"] or case["documents"]:
        state["first"] = _ints([f for c, n in lengths for f in _first_seen(case, c, n)])
    if case["prefix"]:
        state["prefix"] = _ints([min(case["prefix"], c + n) for c, n in lengths])
    return state


def _to_verify(case, gen, rng, new, starts, parents):
    """Probabilities of a target and of a model that resembles it, and tokens which that one drafted."""
    tokens, vocab, dtype = starts[-1], case["vocab"], TYPES[case["type"]]

    def randn():
        return torch.randn((tokens, vocab), device="cuda", generator=gen)

    logits = randn().mul_(3.0)
    target = torch.softmax(logits, -1).to(dtype)
    state = {"kind": "verify", "q_start": _ints(starts), "max_new": max(new), "target": target, "uniforms": torch.rand(tokens, device="cuda", generator=gen)}
    # a drafted row's distribution is like that of its parent's row
    tree = [[t - 1 for t in range(n)] for n in new] if parents is None else parents
    before = torch.tensor([starts[b] + max(p, 0) for b, row in enumerate(tree) for p in row], device="cuda")
    nth = []                                       # which of its parent's children a row is
    for row in tree:
        nth += [row[:t].count(p) for t, p in enumerate(row)]
    if case["draft"]:
        q = torch.softmax(logits[before].add_(randn().mul_(0.4)), -1)
        state["tokens"] = torch.multinomial(q, 1, generator=gen)[:, 0].to(torch.int32)
        state["draft"] = q.to(dtype)
    else:
        guess = logits.add_(randn().mul_(0.4)).topk(max(nth) + 1, -1).indices
        state["tokens"] = guess[before, torch.tensor(nth, device="cuda")].to(torch.int32)
    if parents is not None:
        state["parents"] = _ints([p for row in parents for p in row])
    return state


# ---- the operators in their plain form, in 32 bits (64 where a border has to be met) ----------------------------------

def _ancestors(parents):
    """Of each sequence's tokens [batch, n], which they come behind, themselves among them: [batch, n, n] of truth values."""
    n = parents.shape[1]
    step = (parents[..., None] == torch.arange(n, device="cuda")).float() + torch.eye(n, device="cuda")
    for _ in range((n - 1).bit_length()):                         # (paths of twice the length each time)
        step = (step @ step).clamp(max=1.0)
    return step > 0


def _plain_tables(s):
    table, held, context, new, page, rows, most = s["page_table"], s["held"].long(), s["context"].long(), s["new"].long(), s["page"], s["rows"], s["most"]
    start = torch.zeros(len(new) + 1, dtype=torch.long, device="cuda")
    start[1:] = new.cumsum(0)
    need = ((context + new + page - 1) // page - held).clamp(min=0) * (new > 0)
    ahead = need.cumsum(0) - need
    width = table.shape[1]
    column = torch.arange(width, device="cuda")
    taken = (column >= held[:, None]) & (column < (held + need)[:, None])
    which = s["available"].long() - 1 - (ahead[:, None] + column - held[:, None])
    table.copy_(torch.where(taken, s["free"][which.clamp(0, len(s["free"]) - 1)], table))
    row = torch.arange(rows, device="cuda")
    of = torch.bucketize(row, start[1:], right=True)
    there = of < len(new)
    of = of.clamp(max=len(new) - 1)
    nth = row - start[of]
    at = context[of] + nth
    slots = torch.where(there, table[of, (at // page).clamp(max=width - 1)].long() * page + at % page, -1)
    depth, mask = nth, None
    if "parents" in s:
        inside, row = nth.clamp(0, most - 1), (start[:-1, None] + torch.arange(most, device="cuda")).clamp(max=rows - 1)
        above = _ancestors(torch.where(torch.arange(most, device="cuda") < new[:, None], s["parents"].long()[row], -1))
        depth = above.sum(-1)[of, inside] - 1
        bits = torch.nn.functional.pad(above.long(), (0, -most % 64)).view(len(new), most, -1, 64) << torch.arange(64, device="cuda")
        mask = torch.where(there[:, None], bits.sum(-1)[of, inside], 0)
    positions = torch.where(there, context[of] + depth, 0)
    out = [start, slots, positions, held + need, s["available"] - need.sum()]
    return [x.to(torch.int32) for x in out] + [table] + ([mask] if mask is not None else [])


def _norm_rotate(x, weight, state):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    axes = torch.tensor(state["axes"], device="cuda")
    at, pair = state["positions"].long()[axes].t(), torch.arange(len(axes), device="cuda")
    cos, sin = state["cos"][at, pair].unsqueeze(1), state["sin"][at, pair].unsqueeze(1)
    half = cos.shape[-1]
    x, rest = x[..., : 2 * half], x[..., 2 * half:]
    if state["pairs"]:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _quantise(x, codes):
    top = 127.0 if codes.dtype == torch.int8 else 448.0
    scale = x.abs().amax(-1) / top
    x = x / torch.where(scale > 0, scale, 1.0).unsqueeze(-1)
    return (x.round() if codes.dtype == torch.int8 else x).to(codes.dtype).view(torch.int8), scale


def _plain_axes(s):
    q, k = (_norm_rotate(x, w, s) for x, w in zip((s["q"], s["k"]), s["weights"]))
    if "cache" not in s:
        return [q.to(s["type"]), k.to(s["type"])]
    kc, vc, ks, vs = s["cache"]
    page = kc.shape[2]
    at, off = s["slots"].long() // page, s["slots"].long() % page
    for_k, ks[at, :, off] = _quantise(k, kc)
    for_v, vs[at, :, off] = _quantise(s["v"].float(), vc)
    # (codes are moved as bytes: not every type of 8 bits has an indexed copy)
    kc.view(torch.int8)[at, :, off] = for_k
    vc.view(torch.int8)[at, :, off // 4, :, off % 4] = for_v
    k = kc.view(torch.int8)[at, :, off].view(kc.dtype).float() * ks[at, :, off].unsqueeze(-1)
    v = vc.view(torch.int8)[at, :, off // 4, :, off % 4].view(vc.dtype).float() * vs[at, :, off].unsqueeze(-1)
    return [q.to(s["type"]), k.to(s["type"]), v.to(s["type"])]


def _plain_attend(s):
    q, (kc, vc, ks, vs) = s["q"], s["cache"]
    table, context, start = s["page_table"].long(), s["context"].long(), s["q_start"].long()
    batch, hkv, page, dim = table.shape[0], kc.shape[1], kc.shape[2], kc.shape[3]
    most, length = s["max_new"], table.shape[1] * page

    def rows(x):
        return x.transpose(1, 2).reshape(batch, hkv, length, -1)

    k = rows(kc.view(torch.int8)[table].view(kc.dtype).float() * ks[table].unsqueeze(-1))
    v = rows((vc.view(torch.int8)[table].view(vc.dtype).float() * vs[table].view(batch, -1, hkv, page // 4, 1, 4)).transpose(-1, -2).reshape(batch, -1, hkv, page, dim))
    # every sequence's rows padded to the longest
    tokens, hq = q.shape[0], q.shape[1]
    nth, new = torch.arange(most, device="cuda"), start[1:] - start[:-1]
    row = (start[:-1, None] + nth).clamp(max=tokens - 1)
    qp = q.float()[row].view(batch, most, hkv, hq // hkv, dim).permute(0, 2, 3, 1, 4).reshape(batch, hkv, -1, dim)
    sc = (qp @ k.transpose(-1, -2) * dim ** -0.5).view(batch, hkv, hq // hkv, most, length)
    if s["cap"]:
        sc = s["cap"] * torch.tanh(sc / s["cap"])
    j = torch.arange(length, device="cuda")
    at = j - context[:, None]                                     # keys counted from the first new one
    fresh = at.clamp(0, most - 1)
    if "slopes" in s:
        where = s["positions"].long()[row] if "positions" in s else context[:, None] + nth
        key_at = torch.where(at < 0, j, where.gather(1, fresh))
        sc = sc - s["slopes"].view(hkv, hq // hkv, 1, 1) * (where[:, :, None] - key_at[:, None]).float()[:, None, None]
    if "mask" in s:
        seen = (s["mask"][row][..., nth // 64] >> (nth % 64)) & 1 != 0
        seen = seen.gather(2, fresh[:, None].expand(batch, most, length))
    else:
        upto = nth + 1 if "prefix" not in s else torch.maximum(nth + 1, (s["prefix"].long() - context)[:, None])
        seen = at[:, None] < (upto if upto.dim() == 2 else upto[None])[..., None]
    seen = ((at < 0)[:, None] | seen) & (at < new[:, None])[:, None]
    if "first" in s:
        seen &= j >= s["first"].long()[row][..., None]
    sc = sc.masked_fill(~seen[:, None, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    p = (sc - torch.where(top > -math.inf, top, 0.0)).exp()
    total = p.sum(-1, keepdim=True)
    o = (p.view(batch, hkv, -1, length) @ v).view(batch, hkv, hq // hkv, most, dim) / torch.where(total > 0, total, 1.0)
    here = torch.arange(tokens, device="cuda")
    of = torch.bucketize(here, start[1:], right=True)
    return o.permute(0, 3, 1, 2, 4).reshape(batch, most, hq, dim)[of, here - start[of]].to(s["type"])


def _plain_verify(s):
    target, tokens, start, u, most = s["target"], s["tokens"].long(), s["q_start"].long(), s["uniforms"].double(), s["max_new"]
    batch, nth, every = len(start) - 1, torch.arange(most, device="cuda"), torch.arange(len(start) - 1, device="cuda")
    new = start[1:] - start[:-1]
    row = (start[:-1, None] + nth).clamp(max=len(u) - 1)
    asked = (nth > 0) & (nth < new[:, None])
    parents = torch.where(asked, s["parents"].long()[row] if "parents" in s else nth - 1, -1)
    p = torch.where(asked, target[start[:-1, None] + parents.clamp(min=0), tokens[row]].double(), 0.0)
    # the children of a row in front of each, and what is left to it if they are refused
    elder = (parents[:, :, None] == parents[:, None]) & (nth[:, None] > nth) & asked[:, :, None] & asked[:, None]
    if "draft" in s:
        yes = asked & (p > u[row] * s["draft"][row, tokens[row]].double())
    else:
        yes = asked & (p > u[row] * (1.0 - (elder * p[:, None]).sum(-1)))
    yes = yes & ~(elder & yes[:, None]).any(-1) | (nth == 0)
    reached = (nth < new[:, None]) & ~(_ancestors(parents) & ~yes[:, None]).any(-1)
    count = reached.sum(-1)
    path = torch.where(reached, nth, most).sort(-1).values
    here = path[every, count - 1]
    last, refused = target[start[:-1] + here].double(), asked & (parents == here[:, None])
    if "draft" in s:
        q = s["draft"][start[:-1] + (here + 1).clamp(max=most - 1).minimum(new - 1)].double()
        weight = torch.where(refused.any(-1, keepdim=True), (last - q).clamp(min=0.0), last)
    else:
        weight = last.clone()
        b, t = refused.nonzero(as_tuple=True)
        weight[b, tokens[row[b, t]]] = 0.0
    weight = torch.where(weight.sum(-1, keepdim=True) > 0, weight, last)
    upto = weight.cumsum(-1)
    chosen = ((upto > u[start[:-1], None] * weight.sum(-1, keepdim=True)) & (weight > 0)).int().argmax(-1)
    out = torch.where(path < most, tokens[row.gather(1, path.clamp(max=most - 1))], -1).roll(-1, 1)
    out[:, -1] = -1
    out[every, count - 1] = chosen
    return [x.to(torch.int32) for x in (torch.where(path < most, path, -1), count, out)]


def _plain_keep(s):
    table, context, path, count = s["page_table"].long(), s["context"].long(), s["path"].long(), s["count"].long()
    page = s["caches"][0][0].shape[2]
    nth = torch.arange(path.shape[1], device="cuda")
    b, i = ((nth < count[:, None]) & (path > nth)).nonzero(as_tuple=True)
    source, to = context[b] + path[b, i], context[b] + i
    (sp, so), (tp, to_) = ((table[b, j // page], j % page) for j in (source, to))
    for k, v, ks, vs in s["caches"]:
        kb, vb = k.view(torch.int8), v.view(torch.int8)
        kb[tp, :, to_], vb[tp, :, to_ // 4, :, to_ % 4] = kb[sp, :, so], vb[sp, :, so // 4, :, so % 4]
        ks[tp, :, to_], vs[tp, :, to_] = ks[sp, :, so], vs[sp, :, so]
    return _moved(s)


def _moved(s):
    # (a move changes no code: bytes are compared, of whatever type they are the codes)
    return [x if x.dtype == torch.float32 else x.view(torch.int8) for cache in s["caches"] for x in cache]


PLAIN = {"tables": _plain_tables, "axes": _plain_axes, "attend": _plain_attend, "verify": _plain_verify, "keep": _plain_keep}


# ---- the framework's operators ----------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _module():
    from fusedkernellibrary_amd import attention
    return attention


def _own(s):
    ops, kind = _module(), s["kind"]
    if kind == "tables":
        t = ops.step_tables(s["page_table"], s["held"], s["context"], s["new"], s["free"], s["available"], page_tokens=s["page"], tokens=s["rows"], max_new=s["most"], parents=s.get("parents"))
        return [t.q_start, t.slots, t.positions, t.held, t.available, s["page_table"]] + ([t.mask] if "parents" in s else [])
    if kind == "verify":
        return list(ops.verify_drafts(s["target"], s["tokens"], s["q_start"], s["uniforms"], max_new=s["max_new"], draft=s.get("draft"), parents=s.get("parents")))
    if kind == "keep":
        ops.kv_keep([ops.KvCache(*c) for c in s["caches"]], s["page_table"], s["context"], s["path"], s["count"])
        return _moved(s)
    if kind == "axes":
        tables = (*s["weights"], s["cos"], s["sin"], s["positions"])
        if "cache" not in s:
            return ops.qk_norm_rope(s["q"], s["k"], *tables, eps=EPS, pairs=s["pairs"], axes=s["axes"])
        cache = ops.KvCache(*s["cache"])
        q = ops.qkv_to_cache(cache, s["q"], s["k"], s["v"], s["slots"], *tables, eps=EPS, pairs=s["pairs"], axes=s["axes"])
        return [q, *ops.kv_read(cache, s["slots"], dtype=s["type"])]
    return ops.tree_attention(s["q"], ops.KvCache(*s["cache"]), s["page_table"], s["context"], s["q_start"], max_new=s["max_new"], max_context=s["max_context"], mask=s.get("mask"), cap=s["cap"],
                              slopes=s.get("slopes"), positions=s.get("positions"), first=s.get("first"), prefix=s.get("prefix"))


def run(state):
    return _own(state) if own else PLAIN[state["kind"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "axes":
        dim, hkv, hq = case["dim"], case["hkv"], case["hq"]
        token = 4.0 * hq * dim + 4.0 * hkv * dim + 4 * (max(_axes(case)) + 1)
        if case["cache"]:  # values too; written, and read back
            token += 2.0 * hkv * dim + 4.0 * hkv * (dim + 4) + 2.0 * hkv * dim + 8
        token += 4.0 * case["rot"] * min(1.0, case["table"] / case["tokens"])
        return {"bytes": case["tokens"] * token, "flops": case["tokens"] * 8.0 * (hq + hkv) * dim}
    lengths = _lengths(case)
    tokens = sum(n for _, n in lengths)
    if kind == "tables":
        rows, words = tokens + case["padding"], -(-max(1, case["new"]) // 64)
        pages = sum(-(-(c + n) // case["page"]) - -(-c // case["page"]) for c, n in lengths)
        return {"bytes": 20.0 * len(lengths) + 8.0 * rows + 8.0 * pages + (4.0 + 8.0 * words) * rows * case["tree"] + 8.0, "flops": 10.0 * rows}
    if kind == "verify":
        size = 4.0 if case["type"] == "f32" else 2.0
        return {"bytes": case["batch"] * case["vocab"] * size * (2 if case["draft"] else 1) + tokens * (8.0 + 2 * size) + case["batch"] * 8.0 * case["new"], "flops": case["batch"] * case["vocab"] * 3.0}
    row = case["dim"] + 4  # a cached key or value of one head: codes and scale
    if kind == "keep":
        moved = sum(min(n, 8) for _, n in lengths) / 4.0  # (about: how many are accepted, and move, is the seed's)
        return {"bytes": case["layers"] * max(1.0, moved) * 4.0 * case["hkv"] * row + case["batch"] * 4.0 * (case["new"] + 2), "flops": 0.0}
    keys = pairs = 0
    for c, n in lengths:
        first = _first_seen(case, c, n)
        upto = [min(c + n, max(j + 1, case["prefix"])) for j in range(c, c + n)]
        seen = [max(0, b - a) for a, b in zip(first, upto)]
        if case["tree"]:
            seen = [s - t // 2 for t, s in enumerate(seen)]
        keys += c + n - min(first, default=0)
        pairs += sum(seen)
    return {"bytes": keys * 2.0 * case["hkv"] * row + tokens * 4.0 * case["hq"] * case["dim"], "flops": max(1, pairs) * 4.0 * case["hq"] * case["dim"]}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------

def _exact_heads(x, weight, state):
    """RMS norm and rotation of [tokens, heads, dim] as one complex product per pair."""
    x = x.double()
    n = x.shape[-1]
    x = x / (x.pow(2).sum(-1, keepdim=True) / n + EPS).sqrt() * weight.double()
    table = torch.complex(state["cos"].double(), state["sin"].double())
    turn = torch.stack([table[state["positions"][a].long(), i] for i, a in enumerate(state["axes"])], -1)[:, None]
    half = turn.shape[-1]
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if state["pairs"] else (slice(0, half), slice(half, 2 * half))
    turned = torch.complex(x[..., first], x[..., second]) * turn
    y = x.clone()
    y[..., first], y[..., second] = turned.real, turned.imag
    return y


def _exact_stored(x, codes):
    """What rows of [tokens, heads, dim] are worth once they are held in 8 bits."""
    top = x.abs().max(-1, keepdim=True).values
    if codes == torch.int8:
        step = top / 127
        return torch.where(top > 0, torch.round(x / step) * step, 0.0)
    # e4m3: three bits after the leading one, no exponent below -6
    step = top / 448
    y = torch.where(top > 0, x / step, 0.0)
    unit = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / unit) * unit * step


def _exact_rows(state, slots):
    """(keys, values) [slots, heads, dim] of the cache, one page slot after another."""
    kc, vc, ks, vs = state["cache"]
    page = kc.shape[2]
    at, off = torch.div(slots, page, rounding_mode="floor").long(), torch.remainder(slots, page).long()
    k = kc.view(torch.int8)[at, :, off].view(kc.dtype).double() * ks[at, :, off].double()[..., None]
    v = torch.stack([vc.view(torch.int8)[..., i][at, :, torch.div(off, 4, rounding_mode="floor")].view(vc.dtype).double() for i in range(4)])
    v = v[off % 4, torch.arange(len(slots), device=slots.device)] * vs[at, :, off].double()[..., None]
    return k, v


def _exact_attend(case, state):
    q = state["q"].double()
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    page, dim, group = case["page"], case["dim"], case["hq"] // case["hkv"]
    for b, (lo, hi, context) in enumerate(zip(state["q_start"].tolist(), state["q_start"].tolist()[1:], state["context"].tolist())):
        j = torch.arange(context + hi - lo, device="cuda")
        k, v = _exact_rows(state, state["page_table"][b][j // page] * page + j % page)
        index = j[context:]
        if case["tree"]:
            bits = torch.stack([torch.bitwise_and(torch.bitwise_right_shift(state["mask"][lo:hi, i // 64], i % 64), 1) for i in range(hi - lo)], 1) == 1
            seen = torch.cat([torch.ones((hi - lo, context), dtype=torch.bool, device="cuda"), bits], 1)
            index, j_at = state["positions"][lo:hi].long(), torch.cat([j[:context], state["positions"][lo:hi].long()])
        else:
            seen, j_at = j[None] <= index[:, None], j
        if "prefix" in state:
            seen = seen | (j < state["prefix"][b])[None]
        if "first" in state:
            seen = seen & (j[None] >= state["first"][lo:hi, None])
        none = ~seen.any(1)
        for h in range(case["hkv"]):
            s = torch.matmul(q[lo:hi, h * group:(h + 1) * group], k[:, h].t().contiguous()) / math.sqrt(dim)
            if case["cap"]:
                s = torch.tanh(s / case["cap"]) * case["cap"]
            if "slopes" in state:
                s = s + state["slopes"][h * group:(h + 1) * group].double()[None, :, None] * (j_at[None] - index[:, None]).double()[:, None]
            p = torch.softmax(s.masked_fill(~seen[:, None], -math.inf), -1)
            p[none] = 0.0
            out[lo:hi, h * group:(h + 1) * group] = torch.matmul(p, v[:, h])
    return out


def _exact_tables(state):
    table, held, context, new = (state[n].tolist() for n in ("page_table", "held", "context", "new"))
    free, left, page, rows, most = state["free"].tolist(), int(state["available"]), state["page"], state["rows"], state["most"]
    start, slots, positions, mask, words = [0], [], [], [], -(-most // 64)
    for b, (c, n) in enumerate(zip(context, new)):
        while n and held[b] * page < c + n:
            left -= 1
            table[b][held[b]] = free[left]
            held[b] += 1
        slots += [table[b][j // page] * page + j % page for j in range(c, c + n)]
        if "parents" in state:
            parents = state["parents"][start[-1]:start[-1] + n].tolist()
            positions += [c + d for d in _depths(parents)]
            mask += _mask_words(parents, words)
        else:
            positions += range(c, c + n)
        start.append(start[-1] + n)
    behind = rows - start[-1]
    out = [start, slots + [-1] * behind, positions + [0] * behind, held, [left], table]
    if "parents" in state:
        out.append(mask + [[0] * words] * behind)
    return [torch.tensor(x, dtype=torch.int64) for x in out]


def _exact_verify(state):
    """One sequence after the other, as the rule says it."""
    starts, ids, u, vocab = state["q_start"].tolist(), state["tokens"].tolist(), state["uniforms"].tolist(), state["target"].shape[1]
    most = state["max_new"]
    paths, counts, outs = [], [], []
    for lo, hi in zip(starts, starts[1:]):
        parents = state["parents"][lo:hi].tolist() if "parents" in state else [t - 1 for t in range(hi - lo)]
        path = [0]
        while True:
            weight = state["target"][lo + path[-1]].double()
            children, rest, at = [t for t, p in enumerate(parents) if t and p == path[-1]], 1.0, None
            for t in children:
                x = ids[lo + t]
                p = float(state["target"][lo + path[-1], x])
                if "draft" in state:
                    if p > u[lo + t] * float(state["draft"][lo + t, x]):
                        at = t
                        break
                    weight = (weight - state["draft"][lo + t].double()).clamp_(min=0.0)
                else:
                    if p > u[lo + t] * rest:
                        at = t
                        break
                    rest -= p
                    weight[x] = 0.0
            if at is None:
                break
            path.append(at)
        if not float(weight.sum()) > 0:
            weight = state["target"][lo + path[-1]].double()
        # what is in front of an element, in runs of 1000
        whole = torch.nn.functional.pad(weight, (0, -vocab % 1000)).view(-1, 1000)
        border, run, before = u[lo] * float(whole.sum()), 0, 0.0
        sums = whole.sum(1).tolist()
        while run + 1 < len(sums) and not before + sums[run] > border:
            before += sums[run]
            run += 1
        token = -1
        for i, w in enumerate(whole[run].tolist()):
            before += w
            if w > 0:
                token = run * 1000 + i
                if before > border:
                    break
        outs.append([ids[lo + t] for t in path[1:]] + [token] + [-1] * (most - len(path)))
        paths.append(path + [-1] * (most - len(path)))
        counts.append(len(path))
    return [torch.tensor(x, dtype=torch.int64) for x in (paths, counts, outs)]


def _exact_keep(state):
    page = state["caches"][0][0].shape[2]
    table, context, path, count = (state[n].tolist() for n in ("page_table", "context", "path", "count"))
    where = [(table[b][(context[b] + j) // page], (context[b] + j) % page) for b in range(len(count)) for i in range(count[b]) for j in (path[b][i], i)]
    source, to = [torch.tensor(where[i::2], device="cuda").unbind(1) for i in range(2)]
    out = []
    for k, v, ks, vs in state["caches"]:
        for x in (k.view(torch.int8), v.view(torch.int8).transpose(-1, -2).flatten(2, 3), ks, vs):     # (values as [pages, heads, page, dim])
            y = x.clone()
            y[to[0], :, to[1]] = x[source[0], :, source[1]]
            out.append(y)
        out[-3] = out[-3].view(v.shape[:3] + (4, -1)).transpose(-1, -2).contiguous()
    return out


def exact(case, seed):
    state = prepare(case, seed)
    kind = state["kind"]
    if kind == "axes":
        q, k = (_exact_heads(x, w, state) for x, w in zip((state["q"], state["k"]), state["weights"]))
        return [q, k] if "cache" not in state else [q] + [_exact_stored(x, state["cache"][0].dtype) for x in (k, state["v"].double())]
    return {"tables": _exact_tables, "verify": _exact_verify, "keep": _exact_keep}[kind](state) if kind != "attend" else _exact_attend(case, state)
