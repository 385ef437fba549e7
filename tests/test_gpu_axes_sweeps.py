"""Norm and rotation by positions of several axes where a group of lanes goes over several chunks of a token's heads: against the formula in
64 bits, into new tensors and in place, alone and on the way into a cache."""
import pytest
import torch

import attention_reference as ref
import fusedkernellibrary_amd as fkl
from test_gpu_attention import gen, tables
from test_gpu_axes import BF16, E4M3, F16, INT8, layout, ops, turns  # noqa: F401

pytestmark = pytest.mark.gpu

# Heads are taken two at a time. Sweeps of two chunks to four, of whole ones or with a shorter last one, and with queries' last chunk and
# keys' first in one sweep or not; odd numbers of heads leave half of a chunk.
SIZES = [(2500, 28, 4, 128, 128, False), (2500, 27, 5, 128, 64, True), (4100, 32, 8, 128, 128, False), (4099, 27, 5, 128, 128, False), (6100, 13, 7, 64, 64, True), (6101, 16, 8, 64, 64, False),
         (2501, 9, 5, 256, 256, False), (2500, 12, 4, 192, 96, True), (3300, 11, 3, 96, 96, False), (8191, 21, 1, 72, 40, True)]


def halves(n):
    return (n + 1) // 2


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("tokens,hq,hkv,dim,rot,pairs", SIZES)
def test_alone(ops, device, tokens, hq, hkv, dim, rot, pairs, in_place):  # noqa: F811
    g = gen(tokens + dim)
    dtype = F16 if hq % 2 else BF16
    packed = (3 * torch.randn((tokens, hq + hkv + 1, dim), generator=g)).to(dtype)
    wq, wk = ((1 + 0.3 * torch.randn(dim, generator=g)).to(dtype) for _ in range(2))
    cos, sin = tables(50, rot)
    axes = layout("any" if pairs else "cycle", rot // 2, g)
    positions = torch.randint(0, 50, (max(axes) + 1, tokens), generator=g, dtype=torch.int32)
    on = packed.to(device)
    q, k = on[:, :hq], on[:, hq:hq + hkv]
    got = ops.qk_norm_rope(q, k, wq.to(device), wk.to(device), cos.to(device), sin.to(device), positions.to(device), eps=1e-5, pairs=pairs, axes=axes,
                           **(dict(q_out=q, k_out=k) if in_place else {}))
    many = fkl.last_launch()["grid"][0]
    assert (many < halves(hq) + halves(hkv)) == (tokens * hkv > 6144)
    for x, y, w in ((packed[:, :hq], got[0], wq), (packed[:, hq:hq + hkv], got[1], wk)):
        want, slack = ref.norm_rotate(x, w, *turns(cos, sin, positions, axes), 1e-5, pairs)
        ref.check(y, want, slack * 1.01 + want.abs() * ref.ROUND[dtype] + ref.LEAST[dtype])
    assert torch.equal(on[:, hq + hkv:].cpu(), packed[:, hq + hkv:]) and (in_place or torch.equal(on.cpu(), packed))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("tokens,hq,hkv,dim,rot,pairs", SIZES[:8:2] + SIZES[3:8:2])
def test_into_a_cache(ops, device, kind, tokens, hq, hkv, dim, rot, pairs, in_place):  # noqa: F811
    """Some tokens have no slot: what belongs to nobody stays."""
    g = gen(tokens + dim + 1)
    dtype, page = F16 if hq % 2 else BF16, 64
    pages = tokens // page + 2
    slots = torch.randperm(pages * page, generator=g)[:tokens].to(torch.int32)
    slots[5::50] = torch.tensor([-1, pages * page, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32)[torch.arange(len(slots[5::50])) % 4]
    stored = (slots >= 0) & (slots < pages * page)
    cache = ops.KvCache.allocate(pages, hkv, page, dim, codes=kind, device=device)
    for t in (cache.k, cache.v):
        t.view(torch.int8).fill_(9)
    for t in (cache.k_scale, cache.v_scale):
        t.fill_(0.25)
    packed = torch.randn((tokens, hq + 2 * hkv, dim), generator=g).to(dtype)
    wq, wk = ((1 + 0.3 * torch.randn(dim, generator=g)).to(dtype) for _ in range(2))
    cos, sin = tables(70, rot)
    axes = layout("any" if pairs else "sections", rot // 2, g)
    positions = torch.randint(0, 70, (max(axes) + 1, tokens), generator=g, dtype=torch.int32)
    on = packed.to(device)
    q, k, v = on.split([hq, hkv, hkv], 1)
    got = ops.qkv_to_cache(cache, q, k, v, slots.to(device), wq.to(device), wk.to(device), cos.to(device), sin.to(device), positions.to(device), pairs=pairs, axes=axes, q_out=q if in_place else None)
    assert fkl.last_launch()["grid"][0] - -(-hkv // 4) < halves(hq) + halves(hkv)
    turned = turns(cos, sin, positions, axes)
    want, slack = ref.norm_rotate(packed[:, :hq], wq, *turned, 1e-6, pairs)
    ref.check(got, want, slack * 1.01 + want.abs() * ref.ROUND[dtype] + ref.LEAST[dtype])
    have, at = ref.Slots.of(cache), slots[stored].long()
    want, slack = (x[stored] for x in ref.norm_rotate(packed[:, hq:hq + hkv], wk, *turned, 1e-6, pairs))
    # as in test_gpu_axes.py: half a step of the codes, of a value and a scale that have been rounded in 32 bits
    step = (want.abs().amax(-1) / ref.TOP[kind]).unsqueeze(-1)
    half = 0.5 * step if kind == INT8 else torch.maximum(want.abs() * 2.0 ** -4, step * 2.0 ** -10)
    ref.check(have.keys(at), want, half * 1.001 + slack.amax(-1, keepdim=True) * 1.1)
    codes, scale = ref.quantise(packed[:, hq + hkv:][stored], kind)
    assert torch.equal(have.vs[at], scale) and torch.equal(have.values(at), ref.values_of(codes, kind, scale))
    others = torch.ones(pages * page, dtype=torch.bool)
    others[at] = False
    assert all((x[others] == y).all() for x, y in ((have.k.view(torch.int8), 9), (have.v.view(torch.int8), 9), (have.ks, 0.25), (have.vs, 0.25)))
    assert torch.equal(on[:, hq:].cpu(), packed[:, hq:]) and (in_place or torch.equal(on.cpu(), packed))
