"""Calls of the attention operators at the edges of what they accept, on the GPU."""
import math

import pytest
import torch

import attention_reference as ref
from test_gpu_attention import run_attention, tree_mask

pytestmark = pytest.mark.gpu

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    from fusedkernellibrary_amd import attention
    return attention


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ints(device, *values):
    return torch.tensor(values, dtype=torch.int32, device=device)


# every form without shares: one tile with eight waves and with four, two tiles, four
@pytest.mark.parametrize("batch,new,hq,hkv,dim", [(1, 1, 8, 2, 64), (3, 5, 6, 2, 96), (150, 2, 4, 2, 128), (130, 9, 6, 2, 128), (65, 64, 8, 8, 64), (150, 20, 2, 2, 192), (2, 3, 4, 1, 256)])
@pytest.mark.parametrize("kind,dtype", [(INT8, BF16), (E4M3, F16)])
def test_page_tables_without_columns(ops, device, batch, new, hq, hkv, dim, kind, dtype):
    """No token of a sequence has a page, so nobody sees anything, whatever the contexts are said to be: zeros and -inf."""
    cache = ops.KvCache.allocate(1, hkv, 16, dim, codes=kind, device=device)
    tokens = batch * new
    q = torch.randn((tokens, hq, dim), generator=gen(batch)).to(dtype).to(device)
    start = ints(device, *range(0, tokens + 1, new))
    for context in (0, 700):
        for mask in (None, torch.full((tokens, 1), -1, dtype=torch.int64, device=device)):
            lse = torch.full((tokens, hq), 5.0, device=device)
            out = ops.tree_attention(q, cache, torch.zeros((batch, 0), dtype=torch.int32, device=device), ints(device, *[context] * batch), start, max_new=new, max_context=context, mask=mask,
                                     out=torch.full_like(q, 3.0), lse=lse)
            assert (out == 0).all() and (lse == -math.inf).all()


def test_a_cache_is_of_its_tensors_as_they_are(ops, device):
    """Other memory for a cache's tensors is what the next call reads and writes; other shapes, or too little of it, are refused."""
    g = gen(3)
    x = torch.randn((2, 40, 2, 64), generator=g).to(BF16).to(device)
    slots = torch.arange(40, dtype=torch.int32, device=device)
    one, two = (ops.KvCache.allocate(4, 2, 16, 64, device=device) for _ in range(2))
    ops.kv_write(one, x[0], x[0], slots)
    ops.kv_write(two, x[1], x[1], slots)
    first, second = (ops.kv_read(c, slots) for c in (one, two))
    assert not torch.equal(first[0], second[0])
    q, table, ends = x[0, :1, :1].repeat(1, 4, 1), torch.arange(4, dtype=torch.int32, device=device)[None], (ints(device, 39), ints(device, 0, 1))
    attend = lambda c: ops.tree_attention(q, c, table, *ends, max_new=1, max_context=39)      # noqa: E731
    want = attend(two)
    for to, of in zip(one._tensors, two._tensors):
        to.data = of.clone()
    assert all(torch.equal(a, b) for a, b in zip(ops.kv_read(one, slots), second)) and torch.equal(attend(one), want)
    kept = [t.clone() for t in two._tensors]
    ops.kv_write(one, x[0], x[0], slots)
    assert all(torch.equal(a, b) for a, b in zip(ops.kv_read(one, slots), first))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(two._tensors, kept))
    calls = (lambda: ops.kv_write(one, x[0], x[0], slots), lambda: ops.kv_read(one, slots), lambda: attend(one),
             lambda: ops.qkv_to_cache(one, x[0], x[0], x[0], slots, None, None, None, None, None))
    good = one.k.data
    for bad in (good[:, :, :, :32].contiguous(), good[:3].contiguous(), good.view(torch.uint8), good.cpu()):
        one.k.data = bad
        for call in calls:
            with pytest.raises(ValueError):
                call()
    one.k.data = good
    one.v_scale.untyped_storage().resize_(16)
    for call in calls:
        with pytest.raises(ValueError, match="storage"):
            call()


def test_gradients_and_tangents_are_refused_wherever_they_are_asked_for(ops, device):
    """Norm weights are parameters that ask for gradients in most models: under grad mode they are refused like rows, not detached."""
    q, weight, table = torch.ones((3, 2, 64), dtype=BF16, device=device), torch.ones(64, dtype=BF16, device=device), torch.ones((4, 32), device=device)
    positions = ints(device, 0, 1, 2)
    cache = ops.KvCache.allocate(1, 2, 16, 64, device=device)
    norm = lambda **c: ops.qk_norm_rope(**{**dict(q=q, k=q, q_weight=weight, k_weight=weight, cos=table, sin=table, positions=positions), **c})      # noqa: E731
    store = lambda **c: ops.qkv_to_cache(**{**dict(cache=cache, q=q, k=q, v=q, slots=positions, q_weight=weight, k_weight=weight, cos=table, sin=table, positions=positions), **c})      # noqa: E731
    for call, names in ((norm, ("q", "k", "q_weight", "k_weight", "cos", "sin", "q_out", "k_out")), (store, ("q", "k", "v", "q_weight", "k_weight", "cos", "sin", "q_out"))):
        call()
        for name in names:
            given = {"q_weight": weight, "k_weight": weight, "cos": table, "sin": table}.get(name, q).clone()
            with pytest.raises(ValueError, match=f"{name} asks for a gradient"):
                call(**{name: torch.nn.Parameter(given)})
            with torch.no_grad():
                call(**{name: torch.nn.Parameter(given)})
            with torch.autograd.forward_ad.dual_level():
                with pytest.raises(ValueError, match=f"{name} carries a forward-mode tangent"):
                    call(**{name: torch.autograd.forward_ad.make_dual(given, torch.ones_like(given))})
    lse = torch.zeros((3, 2), device=device, requires_grad=True)
    with pytest.raises(ValueError, match="lse asks for a gradient"):
        ops.tree_attention(q, cache, ints(device, 0)[None], ints(device, 0), ints(device, 0, 3), max_new=3, max_context=0, lse=lse)
    scales = torch.zeros((1, 2, 16), device=device, requires_grad=True)
    with pytest.raises(ValueError, match="k_scale asks for a gradient"):
        ops.KvCache(cache.k, cache.v, scales, cache.v_scale)


def test_what_a_call_writes_to_is_known_to_autograd(ops, device):
    """Outputs that the caller gives, and a cache's tensors, count as changed: a backward pass that had saved one refuses to run."""
    q, positions = torch.ones((3, 2, 64), dtype=BF16, device=device), ints(device, 0, 1, 2)
    cache = ops.KvCache.allocate(1, 2, 16, 64, device=device)
    args = (ints(device, 0)[None], ints(device, 0), ints(device, 0, 3))
    lse = torch.zeros((3, 2), device=device)
    outs = [torch.zeros_like(q) for _ in range(7)]
    before = [t._version for t in (*outs, *cache._tensors, lse, q)]
    ops.qk_norm_rope(q, q, None, None, None, None, None, q_out=outs[0], k_out=outs[1])
    ops.qkv_to_cache(cache, q, q, q, positions, None, None, None, None, None, q_out=outs[2])
    ops.kv_read(cache, positions, k_out=outs[3], v_out=outs[4])
    ops.tree_attention(q, cache, *args, max_new=3, max_context=0, out=outs[5], lse=lse)
    ops.kv_write(cache, q, q, positions)
    after = [t._version for t in (*outs, *cache._tensors, lse, q)]
    assert [a - b for a, b in zip(after, before)] == [1] * 6 + [0] + [2] * 4 + [1, 0]
    saved, weight = torch.ones_like(q), torch.ones(64, dtype=BF16, device=device, requires_grad=True)
    loss = (saved * weight).sum()
    ops.qk_norm_rope(q, q, None, None, None, None, None, q_out=saved)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    with torch.inference_mode():
        made_there = torch.zeros_like(q)
        ops.qk_norm_rope(q, q, None, None, None, None, None, q_out=made_there)
    ops.qk_norm_rope(q, q, None, None, None, None, None, q_out=made_there)
    assert torch.equal(made_there, q)


def test_tracers_are_refused(ops, device):
    """A tracer would record what a call happened to write, or an empty tensor, in place of the call."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode
    q = torch.ones((3, 2, 64), dtype=BF16, device=device)
    call = lambda x: ops.qk_norm_rope(x, x, None, None, None, None, None)[0] + 1      # noqa: E731
    with pytest.raises(ValueError, match="tracer"):
        torch.jit.trace(call, (q,))
    with pytest.raises(ValueError, match="tracer"):
        make_fx(call)(q)
    with FlopCounterMode(display=False):
        assert torch.equal(call(q), q + 1)
    assert torch.equal(torch.compile(call, backend="eager")(q), q + 1)


# keys' codes as they are, with two and three parts of a query, and keys as halves; one tile, two and four; whole blocks and shares
every_product = pytest.mark.parametrize("kind,dtype,dim", [(INT8, BF16, 128), (INT8, F16, 64), (E4M3, BF16, 128), (E4M3, F16, 128), (E4M3, BF16, 64), (INT8, F16, 96), (INT8, BF16, 256)])
every_form = pytest.mark.parametrize("new,said", [(4, 0), (9, 20000), (40, 20000)])


def queries_that_are_not_finite(ops, device, kind, dtype, dim, new, said, what):
    """(out, lse, rows that see nothing, rows whose query holds `what` somewhere) of drafted tokens without a context."""
    g, page, hkv, batch = gen(new + dim), 16, 2, 20
    columns = max(new, said + new) // page + 1
    cache = ops.KvCache.allocate(batch * (new // page + 1), hkv, page, dim, codes=kind, device=device)
    table = torch.full((batch, columns), -1, dtype=torch.int32)
    table[:, :new // page + 1] = torch.arange(table[:, :new // page + 1].numel()).view(batch, -1)
    slots = (table[:, :new // page + 1, None] * page + torch.arange(page)).view(-1).to(torch.int32).to(device)
    x = torch.randn((2, len(slots), hkv, dim), generator=g).to(dtype).to(device)
    ops.kv_write(cache, x[0], x[1], slots)
    q = torch.randn((batch * new, 4, dim), generator=g).to(dtype)
    mask = torch.randint(0, 1 << new, (batch * new, 1), generator=g)
    mask[torch.rand(batch * new, generator=g) < 0.4] = 0
    bad = torch.rand((batch * new, 4), generator=g) < 0.5
    q[bad, torch.randint(0, dim, (int(bad.sum()),), generator=g)] = what
    lse = torch.zeros((batch * new, 4), device=device)
    out = ops.tree_attention(q.to(device), cache, table.to(device), ints(device, *[0] * batch), ints(device, *range(0, batch * new + 1, new)), max_new=new, max_context=said, mask=mask.to(device),
                             lse=lse)
    blind = (mask == 0).expand(-1, 4)
    assert (blind & bad).any() and (~blind & bad).any() and (~blind & ~bad).any()
    return out.cpu(), lse.cpu(), blind, bad


@every_product
@every_form
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_queries_that_are_not_finite_make_their_rows_nan(ops, device, kind, dtype, dim, new, said, what):
    """A row that sees a key is NaN with such a query, whatever the signs of its scores, and others are not."""
    out, lse, blind, bad = queries_that_are_not_finite(ops, device, kind, dtype, dim, new, said, what)
    assert out[~blind & bad].isnan().all() and lse[~blind & bad].isnan().all()
    assert out[~blind & ~bad].isfinite().all() and lse[~blind & ~bad].isfinite().all()


@every_product
@every_form
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_rows_that_see_nothing_are_zero_whatever_their_queries_hold(ops, device, kind, dtype, dim, new, said, what):
    out, lse, blind, _ = queries_that_are_not_finite(ops, device, kind, dtype, dim, new, said, what)
    assert (out[blind] == 0).all() and (lse[blind] == -math.inf).all()


@pytest.mark.parametrize("kind,dtype", [(INT8, BF16), (E4M3, F16)])
# whole blocks: one tile of eight waves and of four, two, four; shares whose parts groups of lanes join, and workgroups
@pytest.mark.parametrize("dim,hq,hkv,copies,max_new,said", [(64, 4, 2, 1, 3, 0), (96, 6, 2, 1, 3, 0), (128, 4, 2, 40, 3, 0), (192, 40, 2, 40, 3, 0), (64, 32, 2, 40, 6, 0), (64, 4, 2, 1, 3, 60000),
                                                            (96, 6, 2, 30, 3, 30000), (256, 10, 1, 1, 6, 60000), (128, 12, 1, 20, 6, 20000)])
def test_rows_of_no_sequence_are_zero(ops, device, kind, dtype, dim, hq, hkv, copies, max_new, said):
    """A padded batch: rows in front of the first sequence, behind the last, and above max_new, of sequences with and without others."""
    new, cut = [2, 0, 9, 1, 4] * copies, lambda n: min(n, max_new)      # noqa: E731
    g, page, front, behind = gen(dim), 16, 3, 21
    starts = [front + sum(new[:b]) for b in range(len(new) + 1)]
    tokens = starts[-1] + behind
    context = torch.tensor([(b * 7) % 40 for b in range(len(new))], dtype=torch.int32)
    if said == 0:
        context.zero_()
    cache = ops.KvCache.allocate(8, hkv, page, dim, codes=kind, device=device)
    x = torch.randn((2, 8 * page, hkv, dim), generator=g).to(dtype).to(device)
    ops.kv_write(cache, x[0], x[1], torch.arange(8 * page, dtype=torch.int32, device=device))
    table = torch.randint(0, 8, (len(new), (said + max_new) // page + 1), generator=g, dtype=torch.int32).to(device)
    q = torch.randn((tokens, hq, dim), generator=g).to(dtype).to(device)
    wide = torch.full((tokens, hq + 1, dim + 8), math.nan, dtype=dtype, device=device)
    lse = torch.full((tokens, hq), math.nan, device=device)
    args = dict(page_table=table, context=context.to(device), max_new=max_new, max_context=said)
    out = ops.tree_attention(q, cache, q_start=ints(device, *starts), out=wide[:, :hq, :dim], lse=lse, **args)
    mine = torch.zeros(tokens, dtype=torch.bool)
    for b, n in enumerate(new):
        mine[starts[b]:starts[b] + cut(n)] = True
    assert (~mine).sum() >= front + behind + copies * (9 - max_new)
    assert (out[~mine] == 0).all() and (lse[~mine] == -math.inf).all() and out[mine].isfinite().all() and (out[mine] != 0).any(-1).all() and lse[mine].isfinite().all()
    assert wide[:, hq:].isnan().all() and wide[:, :, dim:].isnan().all()
    # the same rows by themselves
    alone = ops.tree_attention(q[mine.to(device)], cache, q_start=ints(device, *[sum(map(cut, new[:b])) for b in range(len(new) + 1)]), **args)
    assert torch.equal(out[mine.to(device)], alone)


def test_calls_without_sequences_or_new_tokens_give_zeros(ops, device):
    cache = ops.KvCache.allocate(1, 1, 16, 64, device=device)
    q = torch.ones((5, 2, 64), dtype=BF16, device=device)
    for batch, max_new in ((0, 3), (2, 0)):
        lse = torch.zeros((5, 2), device=device)
        out = ops.tree_attention(q, cache, torch.zeros((batch, 1), dtype=torch.int32, device=device), ints(device, *[1] * batch), ints(device, *range(batch + 1)), max_new=max_new, max_context=4,
                                 out=torch.full_like(q, math.nan), lse=lse)
        assert (out == 0).all() and (lse == -math.inf).all()


def test_outputs_that_overlap_themselves_are_refused(ops, device):
    cache = ops.KvCache.allocate(1, 2, 16, 64, device=device)
    q, slots = torch.ones((3, 2, 64), dtype=BF16, device=device), ints(device, 0, 1, 2)
    one = torch.zeros((1, 2, 64), dtype=BF16, device=device).expand(3, 2, 64)
    ops.kv_write(cache, q, q, slots)
    for call in (lambda: ops.qk_norm_rope(q, q, None, None, None, None, None, q_out=one), lambda: ops.qk_norm_rope(q, q, None, None, None, None, None, k_out=one),
                 lambda: ops.kv_read(cache, slots, v_out=one), lambda: ops.qkv_to_cache(cache, q, q, q, slots, None, None, None, None, None, q_out=one),
                 lambda: ops.tree_attention(q, cache, ints(device, 0)[None], ints(device, 0), ints(device, 0, 3), max_new=3, max_context=0, out=one)):
        with pytest.raises(ValueError, match="overlap"):
            call()
    # inputs may overlap: one row for all tokens
    assert torch.equal(ops.qk_norm_rope(one + 1, one, None, None, None, None, None)[1], one)


@pytest.mark.parametrize("scale", [-0.1, -0.0, 0.0, 0.5])
@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim,new,said", [(64, 3, None), (96, 12, None), (128, 1, 9000), (128, 40, 9000), (256, 9, None)])
def test_scales_of_all_signs(ops, device, scale, kind, dtype, dim, new, said):
    """Below 0 the queries turn round, of 0 every key weighs the same."""
    out = run_attention(ops, device, context=[40, 0, 77], new=[new] * 3, hq=4, hkv=2, dim=dim, page=16, kind=kind, dtype=dtype, seed=dim, said=said, scale=scale,
                        mask=tree_mask([new] * 3, 1, gen(dim)) if new > 1 else None)
    assert out.isfinite().all()


@pytest.mark.parametrize("kind,dtype", [(INT8, BF16), (E4M3, F16)])
@pytest.mark.parametrize("new,dim,hq,words", [([65, 100, 3], 128, 2, 2), ([130, 64, 128], 64, 4, 3), ([200, 1, 70], 256, 1, 5)])
def test_masks_of_several_words_over_shares(ops, device, kind, dtype, new, dim, hq, words):
    """Words of masks are read again for each share of a row's keys; more words than the longest tree needs may be there."""
    import fusedkernellibrary_amd as fkl
    run_attention(ops, device, context=[300, 0, 61], new=new, hq=hq, hkv=1, dim=dim, page=32, kind=kind, dtype=dtype, seed=dim, said=20000, mask=tree_mask(new, words, gen(dim)))
    assert fkl.last_launch()["grid"][1:] == [1, 1] and fkl.last_launch()["grid"][0] >= 64


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("large", [1.0, 40.0])
@pytest.mark.parametrize("new", [1, 20])
def test_scores_next_to_one_large_product(ops, device, kind, dtype, dim, large, new):
    """One channel of queries and keys is larger than the rest, as in many models: the other channels' part of a score has to stay.
    A row that sees one key has that key's score for its lse."""
    g, batch, heads = gen(dim), 40, 16
    x = torch.randn((batch * 32, 1, dim), generator=g)
    x[..., 5] *= large
    q = torch.randn((batch * new, heads, dim), generator=g)
    q[..., 5] *= large
    q, x = q.to(dtype), x.to(dtype)
    cache = ops.KvCache.allocate(batch * 2, 1, 16, dim, codes=kind, device=device)
    ops.kv_write(cache, x.to(device), x.to(device), torch.arange(batch * 32, dtype=torch.int32, device=device))
    mask = torch.randint(0, new, (batch * new,), generator=g)
    lse = torch.zeros((batch * new, heads), device=device)
    ops.tree_attention(q.to(device), cache, torch.arange(batch * 2, dtype=torch.int32, device=device).view(batch, 2), ints(device, *[0] * batch), ints(device, *range(0, batch * new + 1, new)),
                       max_new=new, max_context=0, mask=(1 << mask)[:, None].to(device), lse=lse, scale=0.25)
    k = ref.Slots.of(cache).keys(torch.arange(batch * 32))[torch.arange(batch).repeat_interleave(new) * 32 + mask]                # [rows, 1, dim]
    q = q.double()
    want, size = (q * k).sum(-1) * 0.25, (q * k).abs().sum(-1) * 0.25
    # what of a query's elements may be cut off, in parts of its row's largest (fixed point of 14 or 21 bits for int8, subnormal halves
    # else); products and sums in 32 bits; the scaling by three factors and the two logarithms
    cut = {(INT8, BF16): 2.0 ** -15, (INT8, F16): 2.0 ** -22}.get((kind, dtype), 2.0 ** -24) if kind == E4M3 or dim % 64 == 0 else 2.0 ** -24
    bound = cut * q.abs().amax(-1) * k.abs().sum(-1) * 0.25 + (dim + 8) * 2.0 ** -24 * size + 2.0 ** -21 * want.abs() + 2.0 ** -20
    ref.check(lse, want, bound)
