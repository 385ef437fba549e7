"""A server's attention layer, from a prompt to drafted tokens that are verified as a tree, on the operators of
fusedkernellibrary_amd.attention:

    python examples/verify_drafts.py [--dim 128] [--heads 32] [--kv-heads 8] [--codes int8|e4m3]

Some sequences' prompts go through the layer in chunks. Then each sequence has a tree of drafted tokens, all of which one
call verifies; the tokens of one path through each tree are fed one by one as well, and both ways have to agree.
Then a small model of some layers goes on with its prompts by drafted tokens: `generate` is a server's loop. Weights, prompts
and drafts are random.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from fusedkernellibrary_amd import attention as ops  # noqa: E402


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def turns(positions, dim):
    angle = torch.arange(positions, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, dim, 2, device="cuda") / dim)
    return angle.cos(), angle.sin()


class Pages:
    """Which pages of the caches are whose, and how many tokens each sequence has: all of it on the device."""

    def __init__(self, batch, pages, entries, page, g):
        self.page = page
        self.table = torch.full((batch, entries), -1, dtype=torch.int32, device="cuda")
        self.held, self.context, self.available = ints([0] * batch), ints([0] * batch), ints([pages])
        self.free = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)

    def step(self, new, tokens, max_new, parents=None):
        t = ops.step_tables(self.table, self.held, self.context, new, self.free, self.available, page_tokens=self.page, tokens=tokens, max_new=max_new, parents=parents)
        self.held, self.available = t.held, t.available
        return t


class Layer:
    """Norm, rotation, cache and attention of one layer; what a model projects its tokens to comes in as packed rows."""

    def __init__(self, batch, longest, heads, kv_heads, dim, codes, page=32, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.page = heads, kv_heads, dim, page
        pages = -(-longest // page)
        self.cache = ops.KvCache.allocate(batch * pages, kv_heads, page, dim, codes=codes)
        self.pages = Pages(batch, batch * pages, pages, page, g)
        self.weights = [(1 + 0.1 * torch.randn(dim, generator=g, device="cuda")).bfloat16() for _ in range(2)]
        self.cos, self.sin = turns(longest, dim)

    def run(self, packed, context, new, parents=None):
        """The new tokens' rows [tokens, heads + 2 * kv_heads, dim], new[b] of them behind context[b] cached ones; of trees with parents."""
        self.pages.context = ints(context)
        t = self.pages.step(ints(new), len(packed), max(new), parents)
        q, k, v = packed.split([self.heads, self.kv_heads, self.kv_heads], 1)
        q = ops.qkv_to_cache(self.cache, q, k, v, t.slots, *self.weights, self.cos, self.sin, t.positions)
        return ops.tree_attention(q, self.cache, self.pages.table, self.pages.context, t.q_start, max_new=max(new), max_context=max(context), mask=t.mask)


def tree(tokens, g):
    """Parents of a random tree of drafted tokens: a token sees its ancestors and itself."""
    return [-1] + [int(torch.randint(max(0, t - 4), t, (1,), generator=g)) for t in range(1, tokens)]


def main(prompts=(700, 33, 250), drafts=(13, 30, 1), chunk=256, heads=32, kv_heads=8, dim=128, codes=torch.int8):
    """Largest difference between verified drafts and the same tokens one by one, and the largest value there is."""
    g = torch.Generator().manual_seed(1)
    layer = Layer(len(prompts), max(prompts) + max(drafts), heads, kv_heads, dim, codes)
    rows = lambda n: torch.randn((n, heads + 2 * kv_heads, dim), generator=g).bfloat16().cuda()      # noqa: E731
    have = [0] * len(prompts)
    while any(h < p for h, p in zip(have, prompts)):
        new = [min(chunk, p - h) for h, p in zip(have, prompts)]
        layer.run(rows(sum(new)), have, new)
        have = [h + n for h, n in zip(have, new)]
    trees = [tree(n, g) for n in drafts]
    drafted = rows(sum(drafts))
    verified = layer.run(drafted, have, list(drafts), ints(sum(trees, [])))
    # the path to each tree's last token, one token of every sequence that still has one at a time
    paths, starts = [], [sum(drafts[:b]) for b in range(len(drafts))]
    for parents, n in zip(trees, drafts):
        path = [n - 1]
        while parents[path[-1]] >= 0:
            path.append(parents[path[-1]])
        paths.append(path[::-1])
    worst = 0.0
    for step in range(max(map(len, paths))):
        new = [1 if step < len(p) else 0 for p in paths]
        which = torch.tensor([s + p[step] for s, p in zip(starts, paths) if step < len(p)], device="cuda")
        out = layer.run(drafted[which], have, new)
        worst = max(worst, float((out.float() - verified[which].float()).abs().max()))
        have = [h + n for h, n in zip(have, new)]
    return worst, float(drafted[:, heads + kv_heads:].abs().max())


class Model:
    """A few layers with random weights: from tokens to the probabilities of what follows them."""

    def __init__(self, layers, vocabulary, heads, kv_heads, dim, cap, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        width = heads * dim
        some = lambda *shape: (torch.randn(shape, generator=g, device="cuda") * shape[-1] ** -0.5).bfloat16()      # noqa: E731
        self.heads, self.kv_heads, self.dim, self.cap = heads, kv_heads, dim, cap
        self.embedding = torch.randn((vocabulary, width), generator=g, device="cuda").bfloat16()
        self.layers = [(some((heads + 2 * kv_heads) * dim, width), some(width, width), *(torch.ones(dim, device="cuda").bfloat16() for _ in range(2))) for _ in range(layers)]

    def probabilities(self, x):
        return torch.softmax(x.float() @ self.embedding.float().t() * (4.0 / x.shape[-1]), -1)

    def run(self, tokens, caches, pages, t, cos, sin, max_new, max_context):
        x = self.embedding[tokens.long()]
        for (to_heads, back, q_weight, k_weight), cache in zip(self.layers, caches):
            q, k, v = (x @ to_heads.t()).view(len(x), -1, self.dim).split([self.heads, self.kv_heads, self.kv_heads], 1)
            q = ops.qkv_to_cache(cache, q, k, v, t.slots, q_weight, k_weight, cos, sin, t.positions)
            y = ops.tree_attention(q, cache, pages.table, pages.context, t.q_start, max_new=max_new, max_context=max_context, mask=t.mask, cap=self.cap)
            x = x + y.flatten(1) @ back.t()
        return self.probabilities(x)


def generate(prompts=(70, 5, 131), steps=8, drafts=4, layers=2, vocabulary=500, heads=8, kv_heads=2, dim=64, cap=30.0, codes=torch.int8, page=32, seed=0):
    """What each prompt is continued with: in each step the model's layers see the last token and `drafts` drafted ones, and decide up to
    drafts + 1. The loop never waits for the GPU; drafts come from the last token's embedding alone, one behind the other."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    model = Model(layers, vocabulary, heads, kv_heads, dim, cap, seed)
    batch, new = len(prompts), drafts + 1
    longest = max(prompts) + (steps + 1) * new
    entries = -(-longest // page)
    pages = Pages(batch, batch * entries, entries, page, g)
    caches = [ops.KvCache.allocate(batch * entries, kv_heads, page, dim, codes=codes) for _ in range(layers)]
    cos, sin = turns(longest, dim)
    tokens = torch.randint(0, vocabulary, (sum(prompts),), generator=g, device="cuda", dtype=torch.int32)
    t = pages.step(ints(prompts), len(tokens), max(prompts))
    seen = model.run(tokens, caches, pages, t, cos, sin, max(prompts), 0)
    # the first token of each is drawn from the last row: nothing is drafted
    alone = torch.arange(batch + 1, dtype=torch.int32, device="cuda")
    last = ops.verify_drafts(seen[t.q_start[1:].long() - 1], alone[1:], alone, torch.rand(batch, generator=g, device="cuda"), max_new=1).out[:, 0]
    pages.context = ints(prompts)
    decided, q_start = [last[:, None]], new * alone
    for _ in range(steps):
        row, guessed = [last], []
        for _ in range(drafts):
            guessed.append(model.probabilities(model.embedding[row[-1].long()]))
            row.append(torch.multinomial(guessed[-1], 1, generator=g)[:, 0].to(torch.int32))
        tokens = torch.stack(row, 1).flatten()
        draft = torch.stack([torch.zeros_like(guessed[0]), *guessed], 1).flatten(0, 1)
        t = pages.step(torch.full_like(alone[1:], new), len(tokens), new)
        target = model.run(tokens, caches, pages, t, cos, sin, new, longest)
        v = ops.verify_drafts(target, tokens, q_start, torch.rand(len(tokens), generator=g, device="cuda"), max_new=new, draft=draft)
        ops.kv_keep(caches, pages.table, pages.context, v.path, v.count)
        pages.context = pages.context + v.count
        last = v.out.gather(1, (v.count - 1).long()[:, None])[:, 0]
        decided.append(v.out)
    return [[x for x in row if x >= 0] for row in torch.cat(decided, 1).tolist()]


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--dim", type=int, default=128)
    parser.add_argument("--heads", type=int, default=32)
    parser.add_argument("--kv-heads", type=int, default=8)
    parser.add_argument("--codes", choices=["int8", "e4m3"], default="int8")
    args = parser.parse_args()
    difference, largest = main(heads=args.heads, kv_heads=args.kv_heads, dim=args.dim, codes=torch.int8 if args.codes == "int8" else torch.float8_e4m3fn)
    written = generate(heads=args.heads, kv_heads=args.kv_heads, dim=args.dim, codes=torch.int8 if args.codes == "int8" else torch.float8_e4m3fn)
    print(f"verified as trees and one by one: at most {difference:.3g} apart, values up to {largest:.3g}")
    print("tokens decided in 8 steps of 4 drafted ones:", ", ".join(str(len(w)) for w in written))
