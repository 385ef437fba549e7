"""Attention with scores of another shape (include/fklhip.h, fklhip_scores) in 64 bits on the CPU, and how far a result may be off."""
import math

import torch

import attention_reference as ref


def seen_keys(context, new, mask=None, first=None, prefix=None):
    """[new, context + new]: what each new token of a sequence sees. mask: its rows' words; first: its rows'; prefix: its own."""
    j, i = torch.arange(context + new), context + torch.arange(new)
    if mask is None:
        seen = j[None] <= i[:, None]
        if prefix is not None:
            seen = seen | (j < prefix)[None]
    else:
        tree = torch.stack([(mask[:, u // 64] >> (u % 64)) & 1 == 1 for u in range(new)], 1)
        seen = torch.cat([torch.ones((new, context), dtype=torch.bool), tree], 1)
    if first is not None and new:
        seen = seen & (j[None] >= torch.maximum(first, first[0])[:, None])
    return seen


def attention(q, slots, page, page_table, context, q_start, scale, dtype, mask=None, cap=None, slopes=None, positions=None, first=None, prefix=None):
    """(out, its error bound, lse, its error bound)."""
    tokens, hq, dim = q.shape
    out, bound = torch.zeros((2, tokens, hq, dim), dtype=torch.float64)
    lse = torch.full((tokens, hq), -math.inf, dtype=torch.float64)
    lse_bound = torch.zeros((tokens, hq), dtype=torch.float64)
    for b in range(len(context)):
        lo, hi, have = int(q_start[b]), int(q_start[b + 1]), int(context[b])
        n = have + hi - lo
        if hi == lo or n == 0:
            continue
        seen = seen_keys(have, hi - lo, None if mask is None else mask[lo:hi], None if first is None else first[lo:hi].long(), None if prefix is None else int(prefix[b]))
        keys = seen.any(0).nonzero()[:, 0]                                  # (a key that nobody sees may hold anything)
        if not len(keys):
            continue
        k, v = (f(page_table[b].long()[keys // page] * page + keys % page) for f in (slots.keys, slots.values))
        seen = seen[:, keys]
        at = torch.arange(n)
        if positions is not None:
            at = torch.cat([at[:have], positions[lo:hi].long()])
        group = hq // k.shape[1]
        for h in range(hq):
            kh, vh, qh = k[:, h // group], v[:, h // group], q[lo:hi, h].double()
            s = qh @ kh.t() * scale
            size = qh.abs() @ kh.abs().t() * abs(scale)
            if cap is not None:
                s = cap * torch.tanh(s / cap)
            far = (at[have:, None] - at[keys][None]).double() * (0.0 if slopes is None else float(slopes[h]))
            s = torch.where(seen, s - far, -math.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.where(seen, (s - torch.where(top > -math.inf, top, 0.0)).exp(), 0.0)
            total = p.sum(-1, keepdim=True)
            w = p / torch.where(total == 0, 1.0, total)
            out[lo:hi, h] = w @ vh
            mean = w @ vh.abs()
            # As tests/attention_reference.py has it: weights rounded to half precision, sums in 32 bits, queries held to 2^-16 of their
            # largest element. A score's own error: of the tanh's 1 / (1 + e), whose exponential and reciprocal are off by 2^-22 of
            # themselves each, twice the cap; of the distance's part and of what it is added to, three roundings of 2^-24.
            fixed = 2.0 ** -17 * qh.abs().amax(-1, keepdim=True) * kh.abs().sum(-1).max() * abs(scale)
            off = torch.where(seen, 2 * (dim + 8) * 2.0 ** -24 * size + 2.0 ** -22 * (far.abs() + s.abs()), 0.0) + 2 * fixed + (0.0 if cap is None else cap * 2.0 ** -20)
            off = torch.where(seen, off, 0.0)
            bound[lo:hi, h] = out[lo:hi, h].abs() * ref.ROUND[dtype] + (2.0 ** -11 + 2.0 ** -18) * mean + (w * off) @ vh.abs() + (w * off).sum(-1, keepdim=True) * mean \
                + 2.0 ** -31 * n * vh.abs().max() + ref.LEAST[dtype]
            lse[lo:hi, h] = torch.where(total[:, 0] == 0, -math.inf, top[:, 0] + total[:, 0].log())
            lse_bound[lo:hi, h] = 2.0 ** -12 + 2.0 ** -20 * lse[lo:hi, h].abs().nan_to_num(0.0, 0.0, 0.0) + (w * off).sum(-1)
    return out, bound, lse, lse_bound
