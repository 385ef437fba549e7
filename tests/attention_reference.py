"""The operators of fusedkernellibrary_amd.attention from their formulas, in 64 bits on the CPU, and how far a result may be off.

A cache here is a list of codes and scales by slot (`Slots`), whatever the pages' layout is; `cache_tensors` lays it out."""
import math

import torch

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # half a unit in the last place, relative
LEAST = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}    # (the smallest subnormal)


def norm_rotate(x, weight, cos, sin, positions, eps, pairs):
    """([tokens, heads, dim] in 64 bits, its error bound in 32-bit arithmetic before the last rounding)."""
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    size = x.abs()
    if cos is not None:
        c, s = cos.double()[positions.long()].unsqueeze(1), sin.double()[positions.long()].unsqueeze(1)
        half = c.shape[-1]
        i = torch.arange(half)
        first, second = (2 * i, 2 * i + 1) if pairs else (i, i + half)
        y, size = x.clone(), size.clone()
        y[..., first] = x[..., first] * c - x[..., second] * s
        y[..., second] = x[..., second] * c + x[..., first] * s
        size[..., first] = size[..., second] = x[..., first].abs() + x[..., second].abs()
        x = y
    # the sum of squares, a root, a reciprocal and four products and sums: well under 2^4 roundings of 2^-24
    return x, size * 2.0 ** -20


def quantise(x, codes):
    """(codes as int8 bytes, scale) of float32 rows, bit by bit as the definition in include/fklhip.h says."""
    x = x.float()
    top = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    scale = torch.where(bad, torch.nan, top / TOP[codes])
    y = torch.where((scale > 0).unsqueeze(-1), x / scale.unsqueeze(-1), torch.zeros(()))
    y = y.clamp(-TOP[codes], TOP[codes])
    return (y.round() if codes == torch.int8 else y).to(codes).view(torch.int8), scale


def values_of(codes, kind, scale):
    return codes.view(kind).float().double() * scale.double().unsqueeze(-1)


class Slots:
    """Codes (bytes) [slots, heads, dim] and scales [slots, heads] of keys and values."""

    def __init__(self, slots, heads, dim, kind, generator=None, fill=None):
        self.kind, self.page = kind, None
        x = torch.randn((2, slots, heads, dim), generator=generator)
        (self.k, self.ks), (self.v, self.vs) = (quantise(t, kind) for t in x)
        if fill is not None:
            self.k.fill_(fill[0]), self.v.fill_(fill[0]), self.ks.fill_(fill[1]), self.vs.fill_(fill[1])

    def tensors(self, page, device):
        """k, v, k_scale, v_scale in the layout of include/fklhip.h."""
        slots, heads, dim = self.k.shape
        pages = slots // page
        k = self.k.view(pages, page, heads, dim).transpose(1, 2).contiguous()
        v = self.v.view(pages, page // 4, 4, heads, dim).permute(0, 3, 1, 4, 2).contiguous()
        ks, vs = (s.view(pages, page, heads).transpose(1, 2).contiguous() for s in (self.ks, self.vs))
        return [t.to(device) for t in (k.view(self.kind), v.view(self.kind), ks, vs)]

    @classmethod
    def of(cls, cache):
        """What a cache of the framework's holds."""
        self = cls.__new__(cls)
        self.kind = cache.k.dtype
        k, v = cache.k.cpu().view(torch.int8), cache.v.cpu().view(torch.int8)
        pages, heads, page, dim = k.shape
        self.k = k.transpose(1, 2).reshape(pages * page, heads, dim)
        self.v = v.permute(0, 2, 4, 1, 3).reshape(pages * page, heads, dim)
        self.ks, self.vs = (s.cpu().transpose(1, 2).reshape(pages * page, heads) for s in (cache.k_scale, cache.v_scale))
        return self

    def keys(self, at):
        return values_of(self.k[at], self.kind, self.ks[at])

    def values(self, at):
        return values_of(self.v[at], self.kind, self.vs[at])


def attention(q, slots, page, page_table, context, q_start, mask, scale, dtype):
    """(out, its error bound, lse) in 64 bits."""
    tokens, hq, dim = q.shape
    out, bound = torch.zeros((2, tokens, hq, dim), dtype=torch.float64)
    lse = torch.full((tokens, hq), -math.inf, dtype=torch.float64)
    for b in range(len(context)):
        lo, hi, have = int(q_start[b]), int(q_start[b + 1]), int(context[b])
        n = have + hi - lo
        if hi == lo or n == 0:
            continue
        j = torch.arange(n)
        at = page_table[b].long()[j // page] * page + j % page
        k, v = slots.keys(at), slots.values(at)                             # [n, heads, dim]
        u = torch.arange(hi - lo)
        if mask is None:
            new = u[None] <= u[:, None]
        else:
            new = torch.stack([(mask[lo:hi, i // 64] >> (i % 64)) & 1 == 1 for i in range(hi - lo)], 1)
        seen = torch.cat([torch.ones((hi - lo, have), dtype=torch.bool), new], 1)
        group = hq // k.shape[1]
        for h in range(hq):
            kh, vh = k[:, h // group], v[:, h // group]
            s = q[lo:hi, h].double() @ kh.t() * scale
            size = (q[lo:hi, h].double().abs() @ kh.abs().t() * abs(scale)).nan_to_num(0.0, 0.0)
            s = torch.where(seen, s, -math.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.where(seen, (s - torch.where(top > -math.inf, top, 0.0)).exp(), 0.0)
            total = p.sum(-1, keepdim=True)
            w = p / torch.where(total == 0, 1.0, total)
            rows = seen.any(0)                                              # (a key that nobody sees may hold anything)
            out[lo:hi, h] = w[:, rows] @ vh[rows]
            if not rows.all():
                # a row's own unseen keys take no part either
                for r in range(hi - lo):
                    out[lo + r, h] = w[r, seen[r]] @ vh[seen[r]]
            else:
                for r in (~seen).any(1).nonzero()[:, 0].tolist():
                    out[lo + r, h] = w[r, seen[r]] @ vh[seen[r]]
            mean = torch.where(seen, w, 0.0) @ vh.abs().nan_to_num(0.0)
            # Weights rounded to half precision (2^-11 each), the scores' sums in 32 bits (dim products and the rounding of
            # their scaling, on the sum of magnitudes), exponentials and sums in 32 bits, weights below half precision's
            # normal numbers (2^-25 of a scale, against a sum of at least 2^6), the result's own rounding. Query elements are
            # held to 2^-16 of their row's largest (half of that, rounded) where products are taken on codes.
            fixed = 2.0 ** -17 * q[lo:hi, h].double().abs().amax(-1, keepdim=True) * kh.abs().sum(-1).nan_to_num(0.0).max() * abs(scale)
            slack = 2.0 ** -11 + 2.0 ** -18 + 2 * (dim + 8) * 2.0 ** -24 * size.amax(-1, keepdim=True) + 2 * fixed
            bound[lo:hi, h] = out[lo:hi, h].abs() * ROUND[dtype] + slack * mean + 2.0 ** -31 * n * vh.abs().nan_to_num(0.0).max() + LEAST[dtype]
            lse[lo:hi, h] = torch.where(total[:, 0] == 0, -math.inf, top[:, 0] + total[:, 0].log())
    return out, bound, lse


def check(got, want, bound, what=""):
    got = got.double().cpu()
    assert got.shape == want.shape
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan), f"{what}: NaN at other places"
    off = ((got - want).abs() - bound)[~nan]
    assert off.numel() == 0 or off.max() <= 0, f"{what}: {int((off > 0).sum())} of {off.numel()} outside of the bound, the worst by {off.max():.3g}"
