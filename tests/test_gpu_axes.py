"""Norm and rotation by positions of several axes against their formula in 64 bits, alone and on the way into a cache."""
import pytest
import torch

import attention_reference as ref
from test_gpu_attention import gen, tables

pytestmark = pytest.mark.gpu

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    from fusedkernellibrary_amd import attention
    return attention


def turns(cos, sin, positions, axes):
    """A row of the tables for each token: pair i's entry by the position of its axis. (Rows outside of the table: NaN.)"""
    at = positions.long()[torch.tensor(axes)].t()
    there = (at >= 0) & (at < len(cos))
    pick = lambda t: torch.where(there, t[at.clamp(0, len(cos) - 1), torch.arange(len(axes))], torch.nan)      # noqa: E731
    return pick(cos), pick(sin), torch.arange(positions.shape[1])


def layout(name, pairs, g):
    if name == "sections":
        return [0 if 4 * i < pairs else 1 if 8 * i < 5 * pairs else 2 for i in range(pairs)]
    if name == "cycle":
        return [i % 3 for i in range(pairs)]
    if name == "one":
        return [0] * pairs
    return [int(x) for x in torch.randint(0, 4, (pairs,), generator=g)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("name", ["sections", "cycle", "one", "any"])
@pytest.mark.parametrize("tokens,hq,hkv,dim,rot,pairs", [
    (1, 8, 1, 64, 64, False), (3, 7, 1, 128, 64, True), (17, 5, 5, 96, 96, False), (64, 6, 3, 8, 8, True), (65, 4, 2, 256, 256, False), (257, 9, 3, 128, 128, False), (300, 6, 2, 72, 40, True),
    (259, 5, 1, 192, 192, True), (1000, 3, 1, 64, 16, False), (2100, 5, 3, 64, 64, True), (1237, 6, 6, 128, 128, False), (1300, 5, 5, 256, 256, False)])
def test_norm_and_rotation(ops, device, dtype, name, tokens, hq, hkv, dim, rot, pairs):
    g = gen(tokens * dim)
    packed = (3 * torch.randn((tokens, hq + hkv + 2, dim), generator=g)).to(dtype)
    wq, wk = ((1 + 0.3 * torch.randn(dim, generator=g)).to(dtype) for _ in range(2))
    cos, sin = tables(50, rot)
    axes = layout(name, rot // 2, g)
    positions = torch.randint(0, 50, (max(axes) + 1, tokens), generator=g, dtype=torch.int32)
    on = packed.to(device)
    got = ops.qk_norm_rope(on[:, :hq], on[:, hq:hq + hkv], wq.to(device), wk.to(device), cos.to(device), sin.to(device), positions.to(device), eps=1e-5, pairs=pairs, axes=axes)
    for x, y, w in ((packed[:, :hq], got[0], wq), (packed[:, hq:hq + hkv], got[1], wk)):
        want, slack = ref.norm_rotate(x, w, *turns(cos, sin, positions, axes), 1e-5, pairs)
        ref.check(y, want, slack * 1.01 + want.abs() * ref.ROUND[dtype] + ref.LEAST[dtype])
    assert torch.equal(on.cpu(), packed)


@pytest.mark.parametrize("tokens", [9, 700])
def test_axes_that_agree_are_one(ops, device, tokens):
    """The same position on all axes gives the bits of the form with one."""
    g = gen(3)
    q, k = (torch.randn((tokens, n, 128), generator=g).to(BF16).to(device) for n in (4, 2))
    cos, sin = (t.to(device) for t in tables(900, 128))
    at = torch.arange(tokens, dtype=torch.int32, device=device)
    one = ops.qk_norm_rope(q, k, None, None, cos, sin, at)
    for axes in (tuple(i % 4 for i in range(64)), torch.tensor([i // 16 for i in range(64)]).tolist()):
        several = ops.qk_norm_rope(q, k, None, None, cos, sin, at.expand(4, tokens).contiguous(), axes=axes)
        assert all(torch.equal(a, b) for a, b in zip(one, several))


def test_positions_outside_of_the_table(ops, device):
    """The pairs of the axis are NaN, the others are not."""
    q = torch.ones((2, 2, 64), dtype=BF16, device=device)
    cos, sin = (t.to(device) for t in tables(8, 32))
    for axes in ([0] * 8 + [1] * 8, [0, 1] * 8):
        got, _ = ops.qk_norm_rope(q, q[:, :1], None, None, cos, sin, torch.tensor([[7, 8], [0, -1]], dtype=torch.int32, device=device)[:, :2].contiguous(), axes=axes)
        assert not got[0].isnan().any() and got[1, :, :32].isnan().all() and (got[1, :, 32:] == 1).all()
        got, _ = ops.qk_norm_rope(q, q[:, :1], None, None, cos, sin, torch.tensor([[3, 3], [0, 2 ** 31 - 1]], dtype=torch.int32, device=device), axes=axes)
        hit = torch.tensor(axes * 2 + [0] * 32, device=device) == 1
        assert got[1, 0].isnan().equal(hit)


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("dtype,name,tokens,heads,dim,pairs", [(BF16, "sections", 5, 3, 128, False), (F16, "cycle", 301, 2, 96, True), (BF16, "any", 2101, 3, 64, False), (F16, "cycle", 1300, 5, 256, False)])
def test_into_a_cache(ops, device, kind, dtype, name, tokens, heads, dim, pairs):
    g = gen(tokens)
    page = 32
    pages = tokens // page + 2
    slots = torch.randperm(pages * page, generator=g)[:tokens].to(torch.int32)
    cache = ops.KvCache.allocate(pages, heads, page, dim, codes=kind, device=device)
    for t in (cache.k, cache.v):
        t.view(torch.int8).zero_()
    for t in (cache.k_scale, cache.v_scale):
        t.zero_()
    packed = torch.randn((tokens, 4 * heads, dim), generator=g).to(dtype)
    q, k, v = packed[:, :2 * heads], packed[:, 2 * heads:3 * heads], packed[:, 3 * heads:]
    w = (1 + 0.3 * torch.randn(dim, generator=g)).to(dtype)
    cos, sin = tables(70, dim)
    axes = layout(name, dim // 2, g)
    positions = torch.randint(0, 70, (max(axes) + 1, tokens), generator=g, dtype=torch.int32)
    on = [t.to(device) for t in (w, cos, sin, positions)]
    got = ops.qkv_to_cache(cache, q.to(device), k.to(device), v.to(device), slots.to(device), on[0], on[0], *on[1:], pairs=pairs, axes=axes)
    turned = turns(cos, sin, positions, axes)
    want, slack = ref.norm_rotate(q, w, *turned, 1e-6, pairs)
    ref.check(got, want, slack * 1.01 + want.abs() * ref.ROUND[dtype] + ref.LEAST[dtype])
    have, at = ref.Slots.of(cache), slots.long()
    want, slack = ref.norm_rotate(k, w, *turned, 1e-6, pairs)
    top = want.abs().amax(-1)
    # A stored value is off by half a step of its type (int8: of the scale; e4m3: 2^-4 of itself, or of the smallest normal number's
    # neighbours, 2^-10 of the scale), where the scale itself and the value have been rounded in 32 bits.
    step = (top / ref.TOP[kind]).unsqueeze(-1)
    half = 0.5 * step if kind == INT8 else torch.maximum(want.abs() * 2.0 ** -4, step * 2.0 ** -10)
    ref.check(have.keys(at), want, half * 1.001 + slack.amax(-1, keepdim=True) * 1.1)
    stored, scale = ref.quantise(v, kind)
    assert torch.equal(have.vs[at], scale) and torch.equal(have.values(at), ref.values_of(stored, kind, scale))


def test_axes_that_do_not_fit(ops, device):
    q = torch.ones((2, 2, 64), dtype=BF16, device=device)
    cos, sin = (t.to(device) for t in tables(8, 32))
    at = torch.zeros((2, 2), dtype=torch.int32, device=device)
    call = lambda positions=at, cos=cos, sin=sin, axes=[0, 1] * 8: ops.qk_norm_rope(q, q, None, None, cos, sin, positions, axes=axes)      # noqa: E731
    call()
    for change, word in ((dict(axes=[0, 1]), "16 pairs"), (dict(axes=[0, 2] * 8), "none of them"), (dict(axes=[0, 4] * 8), "0 to 3"), (dict(axes=[-1, 0] * 8), "0 to 3"),
                         (dict(positions=at[0]), "positions"), (dict(positions=at.long()), "positions"), (dict(positions=at.expand(2, 2).t()[:, :1]), "positions"),
                         (dict(cos=None, sin=None), "without cos"), (dict(positions=torch.zeros((5, 2), dtype=torch.int32, device=device)), "1 to 4")):
        with pytest.raises(ValueError, match=word):
            call(**change)
    with pytest.raises(TypeError):
        call(axes=3)


def test_a_captured_call(ops, device):
    g = gen(8)
    q, k = (torch.randn((20, n, 128), generator=g).to(BF16).to(device) for n in (4, 2))
    cos, sin = (t.to(device) for t in tables(90, 128))
    axes = [i % 3 for i in range(64)]
    at = torch.zeros((3, 20), dtype=torch.int32, device=device)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ops.qk_norm_rope(q, k, None, None, cos, sin, at, axes=axes)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = ops.qk_norm_rope(q, k, None, None, cos, sin, at, axes=axes)
    for _ in range(3):
        at.copy_(torch.randint(0, 90, (3, 20), generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, ops.qk_norm_rope(q, k, None, None, cos, sin, at, axes=axes)))
