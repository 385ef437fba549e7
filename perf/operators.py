"""One step of a language model that verifies drafted tokens against a quantised key-value cache, as measurable cases.

Four kinds of pass, each an operator (or the two that a serving step chains) of fusedkernellibrary_amd.attention:

  rope    RMS norm of every query and key head and the rotation by the token's position, in one pass over packed rows
  cache   new tokens' keys and values quantised into the pages of a cache, then a stretch of the cache read back as 16 bits
          (what a chunk of a prompt does: its tokens are written, the whole context is handed to a dense attention)
  attend  attention of a tree of drafted tokens (or of one new token per sequence) over the cache's pages
  step    norm, rotation and quantising write in one launch, attention over the cache, the new tokens' cache rows read back

The cache: keys [pages, kv_heads, page, dim] and values [pages, kv_heads, page / 4, dim, 4] as int8 or e4m3 codes, one float32
scale per token and head ([pages, kv_heads, page]); a value is code * scale, scale = max |x| of the row / 127 (448 for e4m3).
Sequence b has context[b] tokens in the cache before its new ones; token j of it lives in page page_table[b, j // page], and
its new tokens' queries are rows q_start[b] to q_start[b + 1]. Bit u of mask[row] says that the row sees drafted token u.
Context lengths are spread evenly between "lo" and "hi" and dealt to the sequences by the seed, as are the pages.
"""
import functools
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
EPS = 1e-6


def listed():
    return [
        # norm and rotation where latency counts: the one new token of one sequence
        {"name": "rope_1", "kind": "rope", "tokens": 1, "hq": 32, "hkv": 8, "dim": 128, "rot": 128, "pairs": False, "type": "bf16", "table": 4096},
        # a prompt of odd length, seven query heads to a key head
        {"name": "rope_4099", "kind": "rope", "tokens": 4099, "hq": 28, "hkv": 4, "dim": 128, "rot": 128, "pairs": False, "type": "bf16", "table": 8192},
        # several prompts packed together, half of each head rotated, neighbouring elements as pairs, half precision
        {"name": "rope_16384_partial", "kind": "rope", "tokens": 16384, "hq": 16, "hkv": 8, "dim": 64, "rot": 32, "pairs": True, "type": "f16", "table": 32768},
        # 32 sequences with one new token each, written and checked back
        {"name": "cache_32_tokens", "kind": "cache", "batch": 32, "new": 1, "read": 1, "hkv": 8, "dim": 128, "page": 64, "codes": "int8", "type": "bf16"},
        # a 2048-token chunk of one prompt written, its 30011-token context read back
        {"name": "cache_chunk_2048", "kind": "cache", "batch": 1, "new": 2048, "read": 30011, "hkv": 8, "dim": 128, "page": 64, "codes": "e4m3", "type": "bf16"},
        # the smallest attention: one token of one sequence over a short context
        {"name": "attend_1x301", "kind": "attend", "batch": 1, "new_lo": 1, "new": 1, "lo": 300, "hi": 300, "hq": 8, "hkv": 2, "dim": 64, "page": 16, "codes": "int8", "type": "bf16", "tree": False},
        # ordinary serving: 64 sequences with one new token each, contexts of all lengths
        {"name": "attend_64x8k", "kind": "attend", "batch": 64, "new_lo": 1, "new": 1, "lo": 900, "hi": 8191, "hq": 32, "hkv": 8, "dim": 128, "page": 64, "codes": "int8", "type": "bf16", "tree": False},
        # verification of large trees: up to 61 drafted tokens for each of 16 sequences
        {"name": "attend_16_trees_61", "kind": "attend", "batch": 16, "new_lo": 33, "new": 61, "lo": 500, "hi": 4100, "hq": 32, "hkv": 8, "dim": 128, "page": 32, "codes": "e4m3", "type": "bf16", "tree": True},
        # one long document, a small tree, eight query heads to a key head
        {"name": "attend_long_131k", "kind": "attend", "batch": 1, "new_lo": 7, "new": 7, "lo": 131003, "hi": 131003, "hq": 64, "hkv": 8, "dim": 128, "page": 128, "codes": "int8", "type": "bf16", "tree": True},
        # the largest: 48 long contexts, four drafted tokens each
        {"name": "attend_48x32k", "kind": "attend", "batch": 48, "new_lo": 4, "new": 4, "lo": 4000, "hi": 32700, "hq": 32, "hkv": 8, "dim": 128, "page": 64, "codes": "e4m3", "type": "bf16", "tree": True},
        # a whole step for a few short conversations, one token each
        {"name": "step_4x1", "kind": "step", "batch": 4, "new_lo": 1, "new": 1, "lo": 200, "hi": 1500, "hq": 16, "hkv": 2, "dim": 64, "rot": 64, "pairs": False, "page": 16, "codes": "int8", "type": "bf16", "tree": False},
        # a whole step with trees of up to 29 drafted tokens
        {"name": "step_24_trees_29", "kind": "step", "batch": 24, "new_lo": 13, "new": 29, "lo": 150, "hi": 5000, "hq": 28, "hkv": 4, "dim": 128, "rot": 128, "pairs": False, "page": 64, "codes": "e4m3", "type": "f16", "tree": True},
    ]


HEADS = [(8, 2), (16, 16), (16, 2), (32, 8), (28, 4), (20, 20), (64, 8), (12, 4)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        case = _draw(rng)
        sizes = [v for v in case.values() if isinstance(v, int)] + [case["dim"] * (case.get("hq", 0) + n * case["hkv"]) for n in (0, 1, 2)] + [case.get("hq", 0) * case["dim"]]
        # not above the largest listed case, in traffic or in the products of many rows
        if work(case)["bytes"] <= 1.8e9 and work(case)["flops"] <= 8e10 and 3072 not in sizes:
            return case


def _draw(rng):
    kind = rng.choice(["rope", "cache", "attend", "attend", "step", "step"])
    hq, hkv = rng.choice(HEADS)
    dim = rng.choice([64, 96, 128, 128, 256])
    case = {"kind": kind, "hkv": hkv, "dim": dim, "type": rng.choice(["bf16", "f16"])}
    if kind != "cache":
        case["hq"] = hq
    if kind in ("rope", "step"):
        case |= {"rot": rng.choice([dim, dim, dim // 2]), "pairs": rng.random() < 0.3}
    if kind == "rope":
        return case | {"tokens": _log(rng, 1, 16384), "table": 32768}
    case |= {"page": rng.choice([16, 32, 64, 128]), "codes": rng.choice(["int8", "e4m3"])}
    if kind == "cache":
        new = rng.choice([1, _log(rng, 2, 2048)])
        return case | {"batch": _log(rng, 1, 64) if new < 64 else rng.randint(1, 4), "new": new, "read": max(new, _log(rng, 1, 30000) if rng.random() < 0.7 else new)}
    new = rng.choice([1, 1, rng.randint(2, 64)])
    hi = _log(rng, 16, 65536)
    return case | {"batch": _log(rng, 1, 96), "new_lo": rng.randint(1, new), "new": new, "lo": rng.randint(0, hi), "hi": hi, "tree": new > 1 and rng.random() < 0.8}


def _spread(lo, hi, n):
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]


def _lengths(case):
    """(context, new tokens) of each sequence, before the seed deals them."""
    if case["kind"] == "cache":
        return [(case["read"] - case["new"], case["new"])] * case["batch"]
    return list(zip(_spread(case["lo"], case["hi"], case["batch"]), reversed(_spread(case["new_lo"], case["new"], case["batch"]))))


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _quantised(shape, codes, gen):
    """Rows of random keys or values, some elements of a head larger than the others, as codes and scales."""
    kind, top = CODES[codes]
    x = torch.randn(shape, device="cuda", generator=gen)
    x *= 1.0 + 3.0 * (torch.rand(shape[1], 1, shape[-1], device="cuda", generator=gen) > 0.96)
    scale = x.abs().amax(-1) / top
    x /= scale.unsqueeze(-1)
    return (x.round_() if codes == "int8" else x).to(kind), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 2654435761 % (1 << 40))
    rng = random.Random(seed)
    kind, dtype, dim, hkv, hq = case["kind"], TYPES[case["type"]], case["dim"], case["hkv"], case.get("hq", 0)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    state = {"kind": kind, "type": dtype, "pairs": case.get("pairs", False)}
    if kind == "rope":
        tokens, table = case["tokens"], case["table"]
        state["positions"] = torch.randint(0, table, (tokens,), dtype=torch.int32, device="cuda", generator=gen)
    else:
        lengths = _lengths(case)
        rng.shuffle(lengths)
        page, batch = case["page"], len(lengths)
        needs = [-(-(c + n) // page) for c, n in lengths]
        pages = sum(needs) + 3
        order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
        page_table = torch.zeros((batch, max(needs)), dtype=torch.int32, device="cuda")
        row = torch.repeat_interleave(torch.arange(batch), torch.tensor(needs)).cuda()
        starts = torch.tensor([sum(needs[:i]) for i in range(batch)]).cuda()
        page_table[row, torch.arange(sum(needs), device="cuda") - starts[row]] = order[: sum(needs)]
        k, k_scale = _quantised((pages, hkv, page, dim), case["codes"], gen)
        v, v_scale = _quantised((pages, hkv, page, dim), case["codes"], gen)
        v = v.view(torch.int8).view(pages, hkv, page // 4, 4, dim).transpose(3, 4).contiguous().view(v.dtype)
        state |= {"cache": (k, v, k_scale, v_scale), "page_table": page_table}
        context, new = ints([c for c, _ in lengths]), [n for _, n in lengths]
        tokens = sum(new)
        state |= {"context": context, "q_start": ints([sum(new[:i]) for i in range(batch + 1)]), "max_new": max(new), "max_context": max(c for c, _ in lengths)}
        of = torch.repeat_interleave(torch.arange(batch), torch.tensor(new)).cuda()
        nth = torch.arange(tokens, device="cuda") - state["q_start"][of]

        def slots(b, at):
            return (page_table[b, at // page] * page + at % page).to(torch.int32)

        state["slots"] = slots(of, context[of] + nth)
        depth = nth
        if kind == "cache":
            state["read"] = slots(torch.arange(batch, device="cuda").repeat_interleave(case["read"]), torch.arange(case["read"], device="cuda").repeat(batch))
        elif case["tree"]:
            # every drafted token but the first continues one of those before it
            words, far = -(-max(new) // 64), torch.zeros((batch, max(new)), dtype=torch.int64, device="cuda")
            seen = torch.zeros((batch, max(new), words), dtype=torch.int64, device="cuda")
            for t in range(max(new)):
                parent = (torch.rand(batch, device="cuda", generator=gen) * t).long()
                if t:
                    seen[:, t], far[:, t] = seen[torch.arange(batch), parent], far[torch.arange(batch), parent] + 1
                seen[:, t, t // 64] |= -(1 << 63) if t % 64 == 63 else 1 << t % 64
            state["mask"], depth = seen[of, nth].contiguous(), far[of, nth]
        state["positions"] = (context[of] + depth).to(torch.int32)
        table = state["max_context"] + max(new)
    if kind == "attend":
        state["q"] = (1.5 * randn(tokens, hq, dim)).to(dtype)
    else:
        # one row per token, as a projection leaves it: query heads, key heads, value heads
        packed = randn(tokens, (hq + 2 * hkv) * dim).to(dtype).view(tokens, hq + 2 * hkv, dim)
        state |= {"q": packed[:, :hq], "k": packed[:, hq:hq + hkv], "v": packed[:, hq + hkv:]}
    if kind in ("rope", "step"):
        state["weights"] = [(1.0 + 0.2 * randn(dim)).to(dtype) for _ in range(2)]
        angle = torch.arange(table, device="cuda").double()[:, None] * 10000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda").double() / case["rot"])
        state |= {"cos": angle.cos().float(), "sin": angle.sin().float()}
    return state


# ---- the operators in their plain form, in 32 bits --------------------------------------------------------------------

def _norm_rotate(x, weight, state):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    at = state["positions"].long()
    cos, sin = state["cos"][at].unsqueeze(1), state["sin"][at].unsqueeze(1)
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


def _write(state, k, v):
    """float32 rows into the state's cache. (Codes are moved as bytes: not every type of 8 bits has an indexed copy.)"""
    kc, vc, ks, vs = state["cache"]
    page = kc.shape[2]
    at, off = state["slots"].long() // page, state["slots"].long() % page
    for_k, ks[at, :, off] = _quantise(k, kc)
    for_v, vs[at, :, off] = _quantise(v, vc)
    kc.view(torch.int8)[at, :, off] = for_k
    vc.view(torch.int8)[at, :, off // 4, :, off % 4] = for_v


def _read(state, slots):
    kc, vc, ks, vs = state["cache"]
    page = kc.shape[2]
    at, off = slots.long() // page, slots.long() % page
    k = kc.view(torch.int8)[at, :, off].view(kc.dtype).float() * ks[at, :, off].unsqueeze(-1)
    v = vc.view(torch.int8)[at, :, off // 4, :, off % 4].view(vc.dtype).float() * vs[at, :, off].unsqueeze(-1)
    return k.to(state["type"]), v.to(state["type"])


def _attend(state, q):
    kc, vc, ks, vs = state["cache"]
    table, context, start = state["page_table"].long(), state["context"], state["q_start"]
    batch, hkv, page, dim = table.shape[0], kc.shape[1], kc.shape[2], kc.shape[3]
    most, length = state["max_new"], table.shape[1] * page

    def rows(x):
        return x.transpose(1, 2).reshape(batch, hkv, length, -1)

    k = rows(kc.view(torch.int8)[table].view(kc.dtype).float() * ks[table].unsqueeze(-1))
    v = rows((vc.view(torch.int8)[table].view(vc.dtype).float() * vs[table].view(batch, -1, hkv, page // 4, 1, 4)).transpose(-1, -2).reshape(batch, -1, hkv, page, dim))
    # every sequence's rows padded to the longest
    tokens, hq = q.shape[0], q.shape[1]
    nth = torch.arange(most, device=q.device)
    row = (start[:-1, None] + nth).clamp(max=tokens - 1).long()
    qp = q.float()[row].view(batch, most, hkv, hq // hkv, dim).permute(0, 2, 3, 1, 4).reshape(batch, hkv, -1, dim)
    s = (qp @ k.transpose(-1, -2) * dim ** -0.5).view(batch, hkv, hq // hkv, most, length)
    if "mask" in state:
        seen = (state["mask"][row][..., nth // 64] >> (nth % 64)) & 1 != 0
    else:
        seen = (nth[:, None] >= nth).expand(batch, most, most)
    at = torch.arange(length, device=q.device) - context[:, None]
    drafted = (at >= 0) & (at < (start[1:] - start[:-1])[:, None])
    seen = (at < 0)[:, None] | drafted[:, None] & seen.gather(2, at.clamp(0, most - 1).long()[:, None].expand(batch, most, length))
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = (s - torch.where(top > -math.inf, top, 0.0)).exp()
    total = p.sum(-1, keepdim=True)
    o = (p.view(batch, hkv, -1, length) @ v).view(batch, hkv, hq // hkv, most, dim) / torch.where(total > 0, total, 1.0)
    here = torch.arange(tokens, device=q.device)
    of = torch.bucketize(here, start[1:].long(), right=True)
    return o.permute(0, 3, 1, 2, 4).reshape(batch, most, hq, dim)[of, here - start[of]].to(state["type"])


def _plain(state):
    kind, dtype = state["kind"], state["type"]
    if kind == "rope":
        return [_norm_rotate(x, w, state).to(dtype) for x, w in zip((state["q"], state["k"]), state["weights"])]
    if kind == "cache":
        _write(state, state["k"].float(), state["v"].float())
        return _read(state, state["read"])
    if kind == "attend":
        return _attend(state, state["q"])
    q = _norm_rotate(state["q"], state["weights"][0], state).to(dtype)
    _write(state, _norm_rotate(state["k"], state["weights"][1], state), state["v"].float())
    return [q, _attend(state, q), *_read(state, state["slots"])]


# ---- the framework's operators ----------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _module():
    from fusedkernellibrary_amd import attention
    return attention


def _own(state):
    ops, kind = _module(), state["kind"]
    if kind == "rope":
        return ops.qk_norm_rope(state["q"], state["k"], *state["weights"], state["cos"], state["sin"], state["positions"], eps=EPS, pairs=state["pairs"])
    cache = ops.KvCache(*state["cache"])
    if kind == "cache":
        ops.kv_write(cache, state["k"], state["v"], state["slots"])
        return ops.kv_read(cache, state["read"], dtype=state["type"])
    q, outputs = state["q"], []
    if kind == "step":
        q = ops.qkv_to_cache(cache, q, state["k"], state["v"], state["slots"], *state["weights"], state["cos"], state["sin"], state["positions"], eps=EPS, pairs=state["pairs"])
    o = ops.tree_attention(q, cache, state["page_table"], state["context"], state["q_start"], max_new=state["max_new"], max_context=state["max_context"], mask=state.get("mask"))
    return o if kind == "attend" else [q, o, *ops.kv_read(cache, state["slots"], dtype=state["type"])]


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    dim, hkv, hq = case["dim"], case["hkv"], case.get("hq", 0)
    row = dim + 4  # a cached key or value of one head: codes and scale
    rotated = 8 * case.get("rot", 0)  # a token's cosines and sines
    if case["kind"] == "rope":
        return {"bytes": case["tokens"] * (4.0 * (hq + hkv) * dim + rotated + 4), "flops": case["tokens"] * 8.0 * (hq + hkv) * dim}
    lengths = _lengths(case)
    tokens = sum(n for _, n in lengths)
    written = tokens * (2.0 * hkv * (2 * dim + row) + 4)
    if case["kind"] == "cache":
        read = case["batch"] * case["read"] * (2.0 * hkv * (row + 2 * dim) + 4)
        return {"bytes": written + read, "flops": 4.0 * hkv * dim * (tokens + case["batch"] * case["read"])}
    bytes_ = sum(c + n for c, n in lengths) * 2.0 * hkv * row + tokens * 4.0 * hq * dim
    flops = sum(n * (c + (n + 1) / 2) for c, n in lengths) * 4.0 * hq * dim
    if case["kind"] == "step":
        bytes_ += written + tokens * (4.0 * hq * dim + rotated + 4) + tokens * (2.0 * hkv * (row + 2 * dim) + 4)
        flops += tokens * 8.0 * (hq + 2 * hkv) * dim
    return {"bytes": bytes_, "flops": flops}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------

def _exact_heads(x, weight, state):
    """RMS norm and rotation of [tokens, heads, dim] as one complex product per pair."""
    x = x.double()
    n = x.shape[-1]
    x = x / (x.pow(2).sum(-1, keepdim=True) / n + EPS).sqrt() * weight.double()
    turn = torch.complex(state["cos"].double(), state["sin"].double())[state["positions"].long()][:, None]
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


def exact(case, seed):
    state = prepare(case, seed)
    kind = state["kind"]
    q = state["q"].double()
    if kind in ("rope", "step"):
        q, k = (_exact_heads(x, w, state) for x, w in zip((state["q"], state["k"]), state["weights"]))
        if kind == "rope":
            return [q, k]
        q = q.to(state["type"]).double()  # attention's input is held in 16 bits
    codes = state["cache"][0].dtype
    if kind != "attend":
        new = [_exact_stored(x, codes) for x in (k if kind == "step" else state["k"].double(), state["v"].double())]
    if kind == "cache":
        read = list(_exact_rows(state, state["read"]))
        place = torch.full((int(state["read"].max()) + 1,), -1, dtype=torch.long, device="cuda")
        place[state["read"].long()] = torch.arange(len(state["read"]), device="cuda")
        for have, x in zip(read, new):
            have[place[state["slots"].long()]] = x
        return read
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    page, dim = case["page"], case["dim"]
    for b, (lo, hi, context) in enumerate(zip(state["q_start"].tolist(), state["q_start"].tolist()[1:], state["context"].tolist())):
        j = torch.arange(context + hi - lo, device="cuda")
        slots = state["page_table"][b][j // page] * page + j % page
        k, v = _exact_rows(state, slots)
        if kind == "step":
            k[context:], v[context:] = new[0][lo:hi], new[1][lo:hi]
        u = torch.arange(hi - lo, device="cuda")
        if case["tree"]:
            tree = torch.stack([torch.bitwise_and(torch.bitwise_right_shift(state["mask"][lo:hi, i // 64], i % 64), 1) for i in range(hi - lo)], 1) == 1
        else:
            tree = u[None] <= u[:, None]
        seen = torch.cat([torch.ones((hi - lo, context), dtype=torch.bool, device="cuda"), tree], 1)
        group = case["hq"] // case["hkv"]
        for h in range(case["hkv"]):
            s = torch.matmul(q[lo:hi, h * group:(h + 1) * group], k[:, h].t().contiguous()) / math.sqrt(dim)
            p = torch.softmax(s.masked_fill(~seen[:, None], -math.inf), -1)
            out[lo:hi, h * group:(h + 1) * group] = torch.matmul(p, v[:, h])
    return out if kind == "attend" else [q, out, *new]
