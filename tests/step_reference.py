"""What a server's step does around attention, from the definitions in include/fklhip.h, one request after the other on the CPU."""
import math

import torch


def step_tables(table, held, context, new, free, available, page, tokens, max_new, parents=None):
    """(page_table, q_start, slots, positions, held, left, mask) as lists; `table` and the others are lists too."""
    width = len(table[0]) if table else 0
    table, words = [list(r) for r in table], max(1, -(-max_new // 64))
    avail = min(max(available, 0), len(free))
    start, slots, positions, masks, held_out, taken = [], [], [], [], [], 0
    for b in range(len(table)):
        n, c, h = min(max(new[b], 0), max_new), min(max(context[b], 0), 1 << 30), min(max(held[b], 0), width)
        lo = len(slots)
        start.append(lo)
        need = max(0, min(-(-(c + n) // page), width) - h) if n else 0
        for i in range(need):
            if taken < avail:
                table[b][h] = free[avail - 1 - taken]
                h += 1
            taken += 1
        held_out.append(h)
        depth, seen = [], []
        for t in range(min(n, tokens - lo)):
            j = c + t
            entry = table[b][j // page] if j // page < h else -1
            slots.append(entry * page + j % page if 0 <= entry <= (2 ** 31 - 1) // page else -1)
            p = parents[lo + t] if parents is not None else t - 1
            p = p if 0 <= p < t else -1
            depth.append(depth[p] + 1 if p >= 0 else 0)
            seen.append((seen[p] if p >= 0 else 0) | 1 << t)
            positions.append(c + depth[t])
            masks.append([signed(seen[t] >> 64 * w & (1 << 64) - 1) for w in range(words)])
    start.append(len(slots))
    behind = tokens - len(slots)
    return table, start, slots + [-1] * behind, positions + [0] * behind, held_out, avail - taken, masks + [[0] * words] * behind


def signed(word):
    return word - (1 << 64) if word >> 63 else word


def probability(x):
    return x if 0 < x < math.inf else 0.0


def uniform(u):
    return min(u, 1 - 2.0 ** -24) if u > 0 else 0.0


def verify(target, ids, q_start, uniforms, max_new, draft=None, parents=None):
    """(path, count, out, margin) as lists: margin is how near, relative to the whole sum, a drawn token's border is to another's
    (from sums without rounding). target and draft are lists of rows, of exact values."""
    tokens, paths, counts, outs, margin = len(target), [], [], [], 1.0
    for b in range(len(q_start) - 1):
        lo = min(max(q_start[b], 0), tokens)
        n = min(max(q_start[b + 1] - lo, 0), max_new, tokens - lo)
        if n == 0:
            paths.append([-1] * max_new), counts.append(0), outs.append([-1] * max_new)
            continue
        p = [[probability(x) for x in row] for row in target[lo:lo + n]]
        q = None if draft is None else [[probability(x) for x in row] for row in draft[lo:lo + n]]
        u = [uniform(x) for x in uniforms[lo:lo + n]]
        at = lambda row, x: row[x] if 0 <= x < len(row) else 0.0      # noqa: E731
        path = [0]
        while True:
            here, rest, refused, go = path[-1], 1.0, [], None
            for t in range(1, n):
                parent = t - 1 if parents is None else parents[lo + t]
                if parent != here or parent >= t:
                    continue
                x = ids[lo + t]
                px = 0.0 if x in [ids[lo + r] for r in refused] else at(p[here], x)
                if px > u[t] * (rest if q is None else at(q[t], x)):
                    go = t
                    break
                refused.append(t)
                rest -= px
            if go is None:
                break
            path.append(go)
        weight = list(p[here])
        if q is not None and refused:
            weight = [max(x - y, 0.0) for x, y in zip(weight, q[refused[-1]])]
        elif q is None:
            for r in refused:
                if 0 <= ids[lo + r] < len(weight):
                    weight[ids[lo + r]] = 0.0
        if not sum(weight) > 0:
            weight = p[here]
        total = math.fsum(weight)
        token, border, have = -1, u[0] * total, 0.0
        some = [i for i, w in enumerate(weight) if w > 0]
        if some:
            ends = torch.tensor([weight[i] for i in some], dtype=torch.float64).cumsum(0)
            over = (ends > border).nonzero()
            token = some[int(over[0]) if len(over) else -1]
            margin = min(margin, float((ends - border).abs().min()) / total)
        paths.append(path + [-1] * (max_new - len(path)))
        counts.append(len(path))
        outs.append([ids[lo + t] for t in path[1:]] + [token] + [-1] * (max_new - len(path)))
    return paths, counts, outs, margin
