"""A server's attention layer, from a prompt to drafted tokens that are verified as a tree, on the operators of
fusedkernellibrary_amd.attention:

    python examples/verify_drafts.py [--dim 128] [--heads 32] [--kv-heads 8] [--codes int8|e4m3]

Some sequences' prompts go through the layer in chunks. Then each sequence has a tree of drafted tokens, all of which one
call verifies; the tokens of one path through each tree are fed one by one as well, and both ways have to agree.
Weights, prompts and drafts are random.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from fusedkernellibrary_amd import attention as ops  # noqa: E402


class Layer:
    """Norm, rotation, cache and attention of one layer; what a model projects its tokens to comes in as packed rows."""

    def __init__(self, batch, longest, heads, kv_heads, dim, codes, page=32, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.page = heads, kv_heads, dim, page
        pages = -(-longest // page)
        self.cache = ops.KvCache.allocate(batch * pages, kv_heads, page, dim, codes=codes)
        self.page_table = torch.randperm(batch * pages, generator=g, device="cuda").to(torch.int32).view(batch, pages)
        self.weights = [(1 + 0.1 * torch.randn(dim, generator=g, device="cuda")).bfloat16() for _ in range(2)]
        turns = torch.arange(longest, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, dim, 2, device="cuda") / dim)
        self.cos, self.sin = turns.cos(), turns.sin()

    def run(self, packed, context, new, positions=None, mask=None):
        """The new tokens' rows [tokens, heads + 2 * kv_heads, dim], new[b] of them behind context[b] cached ones."""
        starts = [sum(new[:b]) for b in range(len(new) + 1)]
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")      # noqa: E731
        of = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda()
        j = ints(context)[of] + torch.arange(starts[-1], device="cuda") - ints(starts)[of]
        slots = (self.page_table[of, j // self.page] * self.page + j % self.page).to(torch.int32)
        q, k, v = packed.split([self.heads, self.kv_heads, self.kv_heads], 1)
        q = ops.qkv_to_cache(self.cache, q, k, v, slots, *self.weights, self.cos, self.sin, (j if positions is None else positions).to(torch.int32))
        return ops.tree_attention(q, self.cache, self.page_table, ints(context), ints(starts), max_new=max(new), max_context=max(context), mask=mask)


def tree(tokens, g):
    """(parents, depths, mask) of a random tree of drafted tokens: a token sees its ancestors and itself."""
    parents = [-1] + [int(torch.randint(max(0, t - 4), t, (1,), generator=g)) for t in range(1, tokens)]
    depths, bits = [], []
    for t, p in enumerate(parents):
        depths.append(0 if p < 0 else depths[p] + 1)
        bits.append((0 if p < 0 else bits[p]) | 1 << t)
    return parents, depths, [b - (1 << 64) if b >> 63 else b for b in bits]


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
    positions = torch.tensor([h + d for h, t in zip(have, trees) for d in t[1]], device="cuda")
    mask = torch.tensor([b for t in trees for b in t[2]], dtype=torch.int64, device="cuda")[:, None]
    verified = layer.run(drafted, have, list(drafts), positions, mask)
    # the path to each tree's last token, one token of every sequence that still has one at a time
    paths, starts = [], [sum(drafts[:b]) for b in range(len(drafts))]
    for (parents, _, _), n in zip(trees, drafts):
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


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--dim", type=int, default=128)
    parser.add_argument("--heads", type=int, default=32)
    parser.add_argument("--kv-heads", type=int, default=8)
    parser.add_argument("--codes", choices=["int8", "e4m3"], default="int8")
    args = parser.parse_args()
    difference, largest = main(heads=args.heads, kv_heads=args.kv_heads, dim=args.dim, codes=torch.int8 if args.codes == "int8" else torch.float8_e4m3fn)
    print(f"verified as trees and one by one: at most {difference:.3g} apart, values up to {largest:.3g}")
