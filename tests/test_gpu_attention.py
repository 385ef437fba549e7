"""Attention over a quantised, paged cache on the GPU against its formulas in 64 bits: norm and rotation, the quantising write
and the read, attention of drafted and single tokens, and the step that chains them."""
import math

import pytest
import torch

import attention_reference as ref

pytestmark = pytest.mark.gpu

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    from fusedkernellibrary_amd import attention
    return attention


def gen(seed):
    return torch.Generator().manual_seed(seed)


def tables(rows, rot):
    angle = torch.arange(rows).double()[:, None] * 10000.0 ** (-torch.arange(0, rot, 2).double() / max(rot, 1))
    return angle.cos().float(), angle.sin().float()


# ---- norm and rotation ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens,hq,hkv,dim,rot,pairs", [
    (1, 8, 1, 64, 64, False), (3, 7, 1, 128, 64, True), (17, 5, 5, 96, 96, False), (64, 6, 3, 8, 8, True), (65, 4, 2, 256, 128, False),
    (257, 9, 3, 128, 128, False), (300, 6, 2, 72, 40, True), (259, 5, 1, 192, 192, True), (1000, 3, 1, 64, 16, False),
    # rows enough for several heads of a token to a group of lanes
    (2100, 5, 3, 64, 64, True), (1237, 6, 6, 128, 64, False), (1300, 5, 5, 256, 256, False), (6200, 2, 1, 96, 48, False)])
def test_norm_and_rotation(ops, device, dtype, tokens, hq, hkv, dim, rot, pairs):
    g = gen(tokens * dim)
    packed = (3 * torch.randn((tokens, hq + hkv + 2, dim), generator=g)).to(dtype)
    wq, wk = ((1 + 0.3 * torch.randn(dim, generator=g)).to(dtype) for _ in range(2))
    cos, sin = tables(50, rot)
    positions = torch.randint(0, 50, (tokens,), generator=g, dtype=torch.int32)
    on = packed.to(device)
    q, k = on[:, :hq], on[:, hq:hq + hkv]                                          # rows with other things behind them
    got = ops.qk_norm_rope(q, k, wq.to(device), wk.to(device), cos.to(device), sin.to(device), positions.to(device), eps=1e-5, pairs=pairs)
    for x, y, w in ((packed[:, :hq], got[0], wq), (packed[:, hq:hq + hkv], got[1], wk)):
        want, slack = ref.norm_rotate(x, w, cos, sin, positions, 1e-5, pairs)
        ref.check(y, want, slack * 1.01 + want.abs() * ref.ROUND[dtype] + ref.LEAST[dtype])
    assert torch.equal(on.cpu(), packed)


def test_norm_alone_rotation_alone_and_in_place(ops, device):
    g = gen(5)
    q, k = torch.randn((40, 4, 128), generator=g).to(BF16), torch.randn((40, 2, 128), generator=g).to(BF16)
    w = torch.ones(128, dtype=BF16)
    cos, sin = tables(64, 128)
    positions = torch.arange(40, dtype=torch.int32)
    alone = ops.qk_norm_rope(q.to(device), k.to(device), w.to(device), w.to(device), None, None, None)
    turned = ops.qk_norm_rope(q.to(device), k.to(device), None, None, cos.to(device), sin.to(device), positions.to(device))
    for i, x in enumerate((q, k)):
        want, slack = ref.norm_rotate(x, w, None, None, None, 1e-6, False)
        ref.check(alone[i], want, slack + want.abs() * ref.ROUND[BF16])
        want, slack = ref.norm_rotate(x, None, cos, sin, positions, 1e-6, False)
        ref.check(turned[i], want, slack + want.abs() * ref.ROUND[BF16])
    both = ops.qk_norm_rope(q.to(device), k.to(device), w.to(device), w.to(device), cos.to(device), sin.to(device), positions.to(device))
    qd, kd = q.to(device), k.to(device)
    here = ops.qk_norm_rope(qd, kd, w.to(device), w.to(device), cos.to(device), sin.to(device), positions.to(device), q_out=qd, k_out=kd)
    assert here[0] is qd and torch.equal(qd, both[0]) and torch.equal(kd, both[1])


def test_positions_outside_of_the_table_and_empty_calls(ops, device):
    q = torch.ones((3, 2, 64), dtype=BF16, device=device)
    cos, sin = (t.to(device) for t in tables(8, 32))
    got, _ = ops.qk_norm_rope(q, q[:, :1], None, None, cos, sin, torch.tensor([7, 8, -1], dtype=torch.int32, device=device))
    assert not got[0].isnan().any() and got[1:, :, :32].isnan().all() and (got[1:, :, 32:] == 1).all()
    none = q[:0]
    got = ops.qk_norm_rope(none, none[:, :1], None, None, cos, sin, torch.zeros(0, dtype=torch.int32, device=device))
    assert got[0].shape == (0, 2, 64) and got[1].shape == (0, 1, 64)


# ---- cache ------------------------------------------------------------------------------------------------------------

def some_slots(g, tokens, slots, order):
    if order == "run":
        return torch.arange(tokens, dtype=torch.int32) + 4
    if order == "odd run":
        return torch.arange(tokens, dtype=torch.int32) + 7
    return torch.randperm(slots, generator=g)[:tokens].to(torch.int32)


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens,heads,dim,page,order", [
    (1, 1, 64, 16, "run"), (5, 3, 128, 16, "odd run"), (32, 8, 128, 64, "any"), (301, 2, 96, 32, "run"), (303, 5, 256, 128, "odd run"),
    (290, 4, 64, 256, "any"), (270, 1, 72, 32, "odd run"), (9, 2, 8, 16, "any"),
    # rows enough for several heads of a token, and four tokens' values, to a group of lanes
    (2101, 3, 64, 64, "odd run"), (1237, 6, 128, 16, "any"), (1300, 5, 256, 128, "run"), (6203, 1, 96, 32, "odd run")])
def test_cache_write_and_read(ops, device, kind, dtype, tokens, heads, dim, page, order):
    g = gen(tokens + dim)
    pages = -(-(tokens + 16) // page) + 1
    slots = some_slots(g, tokens, pages * page, order)
    cache = ops.KvCache.allocate(pages, heads, page, dim, codes=kind, device=device)
    for t in (cache.k, cache.v):
        t.view(torch.int8).fill_(0x55)
    for t in (cache.k_scale, cache.v_scale):
        t.fill_(-7.0)
    packed = torch.randn((tokens, 2 * heads + 1, dim), generator=g).to(dtype)
    packed[0, :, :] *= 1e-3
    packed[tokens // 2, 0] = 0.0                                                    # a row of zeros
    on = packed.to(device)
    ops.kv_write(cache, on[:, :heads], on[:, heads:2 * heads], slots.to(device))
    have = ref.Slots.of(cache)
    untouched = torch.ones(pages * page, dtype=torch.bool)
    untouched[slots.long()] = False
    for codes, scale, x in ((have.k, have.ks, packed[:, :heads]), (have.v, have.vs, packed[:, heads:2 * heads])):
        want, want_scale = ref.quantise(x, kind)
        assert torch.equal(scale[slots.long()], want_scale)
        # (an e4m3 zero may have either sign)
        a, b = codes[slots.long()], want
        assert torch.equal(torch.where(a == -128, 0, a) if kind == E4M3 else a, torch.where(b == -128, 0, b) if kind == E4M3 else b)
        assert (codes[untouched] == 0x55).all() and (scale[untouched] == -7.0).all()
    k, v = ops.kv_read(cache, slots.to(device), dtype=dtype)
    for got, want in ((k, have.keys(slots.long())), (v, have.values(slots.long()))):
        assert torch.equal(got.cpu(), want.float().to(dtype))                          # one rounding of a float32 product


@pytest.mark.parametrize("kind,dim,pages", [(INT8, 64, 40), (E4M3, 128, 180), (INT8, 192, 160)])
def test_writes_of_runs_that_begin_anywhere(ops, device, kind, dim, pages):
    """Stretches of all lengths that begin at any place of four, in any order, some slots outside, over the edges of workgroups."""
    g = gen(dim)
    page, heads = 16, 3
    left, slots = list(range(pages * page)), []
    while len(left) > 60:
        n, at = int(torch.randint(1, 24, (1,), generator=g)), int(torch.randint(0, len(left), (1,), generator=g))
        slots += left[at:at + n]                                                    # (with gaps where something has been taken out)
        del left[at:at + n]
        if n % 5 == 0:
            slots += [-1, pages * page + n, -4, -3, -2, -1][:n % 7]
    slots = torch.tensor(slots, dtype=torch.int32)
    tokens, there = len(slots), (slots >= 0) & (slots < pages * page)
    cache = ops.KvCache.allocate(pages, heads, page, dim, codes=kind, device=device)
    for t in (cache.k, cache.v):
        t.view(torch.int8).fill_(0x55)
    for t in (cache.k_scale, cache.v_scale):
        t.fill_(-7.0)
    x = torch.randn((2, tokens, heads, dim), generator=g).to(BF16)
    ops.kv_write(cache, x[0].to(device), x[1].to(device), slots.to(device))
    have = ref.Slots.of(cache)
    untouched = torch.ones(pages * page, dtype=torch.bool)
    untouched[slots[there].long()] = False
    for codes, scale, rows in ((have.k, have.ks, x[0]), (have.v, have.vs, x[1])):
        want, want_scale = ref.quantise(rows[there], kind)
        assert torch.equal(scale[slots[there].long()], want_scale)
        assert torch.equal(ref.values_of(codes[slots[there].long()], kind, want_scale), ref.values_of(want, kind, want_scale))
        assert (codes[untouched] == 0x55).all() and (scale[untouched] == -7.0).all()
    k, v = ops.kv_read(cache, slots.to(device))
    for got, want in ((k, have.keys), (v, have.values)):
        assert torch.equal(got.cpu()[there], want(slots[there].long()).float().to(BF16)) and (got.cpu()[~there] == 0).all()


@pytest.mark.parametrize("kind", [INT8, E4M3])
def test_rows_with_infinities_slots_outside_and_strides(ops, device, kind):
    g = gen(1)
    cache = ops.KvCache.allocate(2, 2, 16, 64, codes=kind, device=device)
    for t in (cache.k, cache.v):
        t.view(torch.int8).zero_()
    for t in (cache.k_scale, cache.v_scale):
        t.fill_(1.0)
    k, v = torch.randn((2, 6, 2, 64), generator=g).to(BF16)
    k[0, 0, 3], k[1, 1, 5], v[2, 0, 0] = math.inf, math.nan, -math.inf
    slots = torch.tensor([3, 30, 7, -1, 32, 2 ** 31 - 1], dtype=torch.int32)
    ops.kv_write(cache, k.to(device), v.to(device), slots.to(device))
    have = ref.Slots.of(cache)
    for codes, scale, x in ((have.k, have.ks, k), (have.v, have.vs, v)):
        want, want_scale = ref.quantise(x[:3], kind)
        assert torch.equal(scale[slots[:3].long()].nan_to_num(99.0), want_scale.nan_to_num(99.0))
        assert torch.equal(codes[slots[:3].long()], torch.where(want_scale.isnan().unsqueeze(-1), 0, want).to(torch.int8))
        rest = torch.ones(32, dtype=torch.bool)
        rest[slots[:3].long()] = False
        assert (codes[rest] == 0).all() and (scale[rest] == 1.0).all()
    out = torch.full((6, 5, 64), 9.0, dtype=F16, device=device)
    ops.kv_read(cache, slots.to(device), dtype=F16, k_out=out[:, :2], v_out=out[:, 3:])
    assert out[0, 0].isnan().all() and out[1, 1].isnan().all() and out[2, 3].isnan().all() and not out[0, 1].isnan().any()
    assert (out[3:, :2] == 0).all() and (out[3:, 3:] == 0).all() and (out[:, 2] == 9.0).all()


# ---- attention --------------------------------------------------------------------------------------------------------

def paged(lengths, page, g, spare=2):
    """A page table of pages in random order for sequences of these lengths, and the number of pages."""
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lengths), max(max(need), 1)), 1 << 29, dtype=torch.int32)    # entries behind a sequence's are never used
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


def tree_mask(new, words, g):
    """Ancestors (and the token itself) of random trees, one after another."""
    rows = []
    for n in new:
        seen = []
        for t in range(n):
            bits = seen[int(torch.randint(0, t, (1,), generator=g))] if t else 0
            seen.append(bits | 1 << t)
        rows += [[((s >> 64 * w) & (2 ** 64 - 1)) - (2 ** 64 if (s >> 64 * w) >> 63 & 1 else 0) for w in range(words)] for s in seen]
    return torch.tensor(rows, dtype=torch.int64).view(-1, words)


def run_attention(ops, device, *, context, new, hq, hkv, dim, page, kind, dtype, mask=None, scale=None, q=None, slots=None, seed=0, poison=True, table=None, said=None, **more):
    g = gen(seed)
    lengths = [c + n for c, n in zip(context, new)]
    if table is None:
        table, pages = paged(lengths, page, g)
        if slots is None:
            slots = ref.Slots(pages * page, hkv, dim, kind, g)
            if poison:
                # what no token was written to holds NaN
                used = torch.zeros(pages * page, dtype=torch.bool)
                for b, n in enumerate(lengths):
                    j = torch.arange(n)
                    used[table[b].long()[j // page] * page + j % page] = True
                for codes, s in ((slots.k, slots.ks), (slots.v, slots.vs)):
                    codes[~used], s[~used] = 0x7f, math.nan
    q_start = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32)
    if q is None:
        q = (1.5 * torch.randn((sum(new), hq, dim), generator=g)).to(dtype)
    cache = ops.KvCache(*slots.tensors(page, device))
    lse = torch.full((sum(new), hq), 5.0, dtype=torch.float32, device=device)
    context = torch.tensor(context, dtype=torch.int32)
    if said is not None:                                                           # the longest context there might be
        table = torch.nn.functional.pad(table, (0, -(-(said + max(new)) // page) - table.shape[1]), value=-1)
    out = ops.tree_attention(q.to(device), cache, table.to(device), context.to(device), q_start.to(device), max_new=max(new), max_context=int(context.max()) if said is None else said,
                             mask=None if mask is None else mask.to(device), scale=scale, lse=lse, **more)
    want, bound, want_lse = ref.attention(q, slots, page, table, context, q_start, mask, dim ** -0.5 if scale is None else scale, dtype)
    ref.check(out, want, bound, "out")
    finite = want_lse.isfinite()
    assert torch.equal(lse.cpu().isfinite(), finite) and torch.equal(lse.cpu().double()[~finite].nan_to_num(1.0), want_lse[~finite].nan_to_num(1.0))
    assert ((lse.cpu().double() - want_lse).abs()[finite] <= 2.0 ** -12 + 2.0 ** -20 * want_lse.abs()[finite]).all()
    return out


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
def test_single_tokens(ops, device, kind, dim):
    """Contexts around every edge of a tile and a page, one new token each."""
    context = [0, 1, 15, 16, 17, 30, 31, 32, 33, 63, 64, 95, 127, 128, 129, 255, 300]
    run_attention(ops, device, context=context, new=[1] * len(context), hq=8, hkv=2, dim=dim, page=16, kind=kind, dtype=BF16, seed=dim)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (14, 2), (16, 2), (20, 20), (64, 1), (33, 11)])
@pytest.mark.parametrize("page,kind,dtype", [(16, INT8, F16), (64, E4M3, BF16), (256, INT8, BF16)])
def test_shared_heads_and_pages(ops, device, hq, hkv, page, kind, dtype):
    run_attention(ops, device, context=[5, 130, 77], new=[3, 1, 9], hq=hq, hkv=hkv, dim=64, page=page, kind=kind, dtype=dtype, seed=hq)


@pytest.mark.parametrize("kind,dtype", [(INT8, BF16), (E4M3, F16)])
@pytest.mark.parametrize("new", [[1, 2, 5, 16], [17, 31, 3], [64, 63, 33, 1], [70, 128, 100]])
def test_trees(ops, device, kind, dtype, new):
    g = gen(len(new))
    words = -(-max(new) // 64)
    mask = tree_mask(new, words, g)
    run_attention(ops, device, context=[(b * 37) % 101 for b in range(len(new))], new=new, hq=8, hkv=2, dim=128, page=32, kind=kind, dtype=dtype, mask=mask, seed=7)


@pytest.mark.parametrize("new", [[33, 0, 150], [200]])
def test_without_a_mask_new_tokens_see_those_before_them(ops, device, new):
    run_attention(ops, device, context=[40, 3, 0][:len(new)], new=new, hq=4, hkv=2, dim=128, page=16, kind=INT8, dtype=BF16, seed=3)


def test_sequences_without_new_tokens_and_rows_that_see_nothing(ops, device):
    """Masks without a bit over an empty context give zeros and -inf; sequences without new tokens or context take no part."""
    mask = torch.zeros((6, 1), dtype=torch.int64)
    mask[3, 0], mask[5, 0] = 0b010, 0b101
    out = run_attention(ops, device, context=[0, 9, 0, 40], new=[2, 1, 3, 0], hq=4, hkv=1, dim=64, page=16, kind=E4M3, dtype=BF16, mask=mask, seed=2)
    assert (out[:2] == 0).all() and (out[4] == 0).all() and (out[2] != 0).any() and (out[3] != 0).any()


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("hidden", [math.nan, math.inf])
def test_what_a_mask_hides_may_hold_anything(ops, device, kind, hidden):
    """A drafted token with a key and value that are NaN or infinite (stored as NaN): rows that see it are NaN, others are not."""
    g = gen(4)
    table, pages = paged([50 + 6], 16, g)
    slots = ref.Slots(pages * 16, 2, 64, kind, g)
    j = torch.tensor([52])
    at = int(table[0].long()[j // 16] * 16 + j % 16)
    slots.ks[at], slots.vs[at], slots.k[at], slots.v[at] = math.nan, math.nan, 0, 0
    mask = torch.tensor([[0b1], [0b11], [0b101], [0b1001], [0b10101], [0b100001]])
    q = torch.randn((6, 4, 64), generator=g).to(BF16)
    q_start = torch.tensor([0, 6], dtype=torch.int32)
    cache = ops.KvCache(*slots.tensors(16, device))
    out = ops.tree_attention(q.to(device), cache, table.to(device), torch.tensor([50], dtype=torch.int32, device=device), q_start.to(device), max_new=6, max_context=50, mask=mask.to(device))
    sees = torch.tensor([False, False, True, False, True, False])
    assert torch.equal(out.isnan().all(-1).all(-1).cpu(), sees) and torch.equal(out.isnan().any(-1).any(-1).cpu(), sees)
    want, bound, _ = ref.attention(q, slots, 16, table, torch.tensor([50]), q_start, mask, 64 ** -0.5, BF16)
    ref.check(out[~sees], want[~sees], bound[~sees])


@pytest.mark.parametrize("kind", [INT8, E4M3])
def test_scores_that_rise_and_scales_of_all_sizes(ops, device, kind):
    """The running maximum has to move: keys that grow along the sequence, and value scales over many orders of magnitude."""
    g = gen(9)
    n = 700
    table, pages = paged([n], 32, g)
    slots = ref.Slots(pages * 32, 2, 128, kind, g)
    j = torch.arange(n)
    at = table[0].long()[j // 32] * 32 + j % 32
    slots.ks[at] *= (0.2 + j / 100.0).unsqueeze(1)
    slots.vs[at] *= (10.0 ** ((j * 7 % 13) - 9.0)).unsqueeze(1)
    slots.vs[at[::11]] = 0.0
    run_attention(ops, device, context=[n - 2], new=[2], hq=6, hkv=2, dim=128, page=32, kind=kind, dtype=BF16, slots=slots, table=table, seed=9)


def test_queries_of_all_sizes_and_of_zeros(ops, device):
    g = gen(11)
    q = torch.randn((5, 4, 64), generator=g)
    q[0] *= 1e-30
    q[1] *= 1e30
    q[2] = 0.0
    q[3, 0] = 0.0
    q = q.to(BF16)
    # 1e30 makes the softmax pick one key: the bound's score term covers the sums' rounding, the pick itself has to agree
    out = run_attention(ops, device, context=[0], new=[5], hq=4, hkv=2, dim=64, page=16, kind=INT8, dtype=BF16, q=q[[0, 2, 3, 4, 0]].contiguous(), seed=11)
    assert out.isfinite().all()
    g = gen(12)
    slots = ref.Slots(64, 2, 64, INT8, g)
    cache = ops.KvCache(*slots.tensors(16, device))
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)      # noqa: E731
    out = ops.tree_attention(q[1:2].to(device), cache, ints(0, 1, 2, 3).view(1, 4), ints(40), ints(0, 1), max_new=1, max_context=40)
    assert out.isfinite().all()


@pytest.mark.parametrize("kind,dim,new", [(INT8, 128, 1), (E4M3, 64, 5), (INT8, 256, 3), (E4M3, 96, 2)])
def test_long_contexts_are_shared_out(ops, device, kind, dim, new):
    """One long and some short sequences: the long one's keys go to many workgroups, whose parts are joined."""
    out = run_attention(ops, device, context=[5003, 0, 40, 1999], new=[new, 1, new, 1], hq=6, hkv=2, dim=dim, page=64, kind=kind, dtype=F16, seed=dim + new)
    assert out.isfinite().all()


def ragged(n, top, g):
    return [int(x) for x in torch.randint(0, top, (n,), generator=g)]


@pytest.mark.parametrize("kind,dtype", [(INT8, BF16), (E4M3, BF16), (INT8, F16), (E4M3, F16)])
@pytest.mark.parametrize("form,dim,batch,new,hq,hkv,said,shared", [
    ("1x8", 128, 7, 3, 4, 2, None, False), ("1x4", 64, 150, 2, 4, 2, None, False), ("2x4", 128, 130, 9, 6, 2, None, False), ("4x4", 64, 65, 64, 8, 8, None, False),
    ("4x4", 128, 33, 64, 16, 16, None, False), ("1x4", 128, 40, 5, 2, 1, 20000, True), ("1x4", 256, 30, 4, 6, 2, 30000, True), ("2x4", 64, 19, 9, 6, 2, 9000, True),
    ("2x4", 256, 9, 8, 8, 2, 70000, True), ("2x4", 192, 150, 20, 2, 2, None, False), ("4x4", 128, 11, 33, 6, 3, 20000, True), ("4x4", 96, 9, 50, 4, 2, 70000, True),
    ("4x4", 64, 70, 40, 8, 4, 4000, True)])
def test_every_form(ops, device, kind, dtype, form, dim, batch, new, hq, hkv, said, shared):
    """The tiles and waves of a workgroup, and shares or none, that sizes lead to: with sequences of all lengths, some without new tokens."""
    import fusedkernellibrary_amd as fkl
    g = gen(batch)
    some = ragged(batch, new + 1, g)
    some[batch // 2] = new
    context = ragged(batch, 200, g)
    run_attention(ops, device, context=context, new=some, hq=hq, hkv=hkv, dim=dim, page=16, kind=kind, dtype=dtype, seed=batch, said=said,
                  mask=tree_mask(some, 1, g) if new > 1 else None)
    last = fkl.last_launch()
    assert last["form"] == "tree_attention_" + form
    assert (last["grid"][1:] == [1, 1] and last["grid"][0] >= 64) if shared else last["grid"][2] == batch


@pytest.mark.parametrize("kind,dtype", [(INT8, BF16), (E4M3, F16)])
def test_one_sequence_of_many_rows(ops, device, kind, dtype):
    """So many row blocks that none is shared, over a context that may be long and is not; every row sees every new token but one."""
    import fusedkernellibrary_amd as fkl
    mask = torch.full((256, 4), -1, dtype=torch.int64)
    mask[100, 1] = ~(1 << 36)
    run_attention(ops, device, context=[37], new=[256], hq=256, hkv=16, dim=64, page=32, kind=kind, dtype=dtype, seed=77, said=3000, mask=mask)
    last = fkl.last_launch()
    assert last["form"] == "tree_attention_4x4" and last["grid"] == [16, 64, 1]


def test_results_do_not_change_from_call_to_call(ops, device):
    g = gen(21)
    table, pages = paged([4000, 3000], 16, g)
    cache = ops.KvCache(*ref.Slots(pages * 16, 2, 128, INT8, g).tensors(16, device))
    q = torch.randn((6, 8, 128), generator=g).to(BF16).to(device)
    args = dict(max_new=4, max_context=3998)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)      # noqa: E731
    first = ops.tree_attention(q, cache, table.to(device), ints(3996, 2998), ints(0, 4, 6), **args)
    for _ in range(3):
        assert torch.equal(ops.tree_attention(q, cache, table.to(device), ints(3996, 2998), ints(0, 4, 6), **args), first)


def test_strided_queries_and_outputs(ops, device):
    g = gen(31)
    table, pages = paged([90], 16, g)
    slots = ref.Slots(pages * 16, 2, 64, INT8, g)
    cache = ops.KvCache(*slots.tensors(16, device))
    wide = torch.randn((3, 7, 96), generator=g).to(F16).to(device)
    out = torch.full((3, 9, 72), 3.0, dtype=F16, device=device)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)      # noqa: E731
    q = wide[:, 1:5, 8:72]
    ops.tree_attention(q, cache, table.to(device), ints(87), ints(0, 3), max_new=3, max_context=87, out=out[:, 4:8, :64])
    want, bound, _ = ref.attention(q.cpu(), slots, 16, table, torch.tensor([87]), torch.tensor([0, 3]), None, 0.125, F16)
    ref.check(out[:, 4:8, :64], want, bound)
    rest = torch.ones_like(out, dtype=torch.bool)
    rest[:, 4:8, :64] = False
    assert (out[rest] == 3.0).all()


def test_lengths_and_pages_beyond_what_was_said_are_cut_off(ops, device):
    """Values only the device sees: lengths above max_context and max_new, tokens behind the page table, pages outside of the
    cache. The kernels stay inside what they were given (here everything is inside of larger tensors as well)."""
    g = gen(41)
    slots = ref.Slots(8 * 16, 1, 64, INT8, g)
    cache = ops.KvCache(*slots.tensors(16, device))
    q = torch.randn((4, 2, 64), generator=g).to(BF16)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)      # noqa: E731
    table = torch.tensor([[3, 5, 1]], dtype=torch.int32)
    call = lambda table, context, start, **kw: ops.tree_attention(q.to(device), cache, table.to(device), context, start, out=torch.zeros_like(q, device=device), **kw)   # noqa: E731
    want, bound, _ = ref.attention(q, slots, 16, table, torch.tensor([20]), torch.tensor([0, 4]), None, 0.125, BF16)
    ref.check(call(table, ints(1 << 30), ints(0, 4), max_new=4, max_context=20), want, bound)               # a longer context than said
    assert torch.equal(call(table, ints(-5), ints(0, 4), max_new=4, max_context=20), call(table, ints(0), ints(0, 4), max_new=4, max_context=20))
    got = call(table, ints(20), ints(0, 4), max_new=2, max_context=20)                                      # more new tokens than said
    assert torch.equal(got[2:].cpu(), torch.zeros_like(q[2:])) and not got[:2].eq(0).all()
    assert torch.equal(call(table, ints(20), ints(0, 99), max_new=64, max_context=20), call(table, ints(20), ints(0, 4), max_new=64, max_context=20))
    far = torch.tensor([[3, 1 << 30, -7]], dtype=torch.int32)                                              # read as the last page
    last = torch.tensor([[3, 7, 7]], dtype=torch.int32)
    assert torch.equal(call(far, ints(40), ints(0, 4), max_new=4, max_context=40), call(last, ints(40), ints(0, 4), max_new=4, max_context=40))
    # 48 slots in the table's row: 46 tokens of context leave room for two new ones
    short = call(table, ints(46), ints(0, 4), max_new=4, max_context=46)
    assert short.isfinite().all()


# ---- the step ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind,dtype,dim,rot,pairs,page", [(INT8, BF16, 128, 128, False, 64), (E4M3, F16, 64, 32, True, 16), (INT8, F16, 256, 256, False, 32), (E4M3, BF16, 96, 96, True, 16)])
@pytest.mark.parametrize("tokens,heads", [(1237, 6), (6203, 1)])
def test_many_tokens_to_the_cache(ops, device, kind, dtype, dim, rot, pairs, page, tokens, heads):
    """One launch or two: the keys are quantised from 32 bits in one, so they are the norm's and rotation's, and the values as written."""
    g = gen(tokens + dim)
    pages = tokens // page + 3
    packed = torch.randn((tokens, 4 * heads, dim), generator=g).to(dtype).to(device)
    wq, wk = ((1 + 0.2 * torch.randn(dim, generator=g)).to(dtype).to(device) for _ in range(2))
    cos, sin = (t.to(device) for t in tables(tokens, rot))
    positions = torch.arange(tokens, dtype=torch.int32, device=device)
    slots = (torch.arange(tokens) + 5).to(torch.int32).to(device)
    one, two = (ops.KvCache.allocate(pages, heads, page, dim, codes=kind, device=device) for _ in range(2))
    q = ops.qkv_to_cache(one, packed[:, :2 * heads], packed[:, 2 * heads:3 * heads], packed[:, 3 * heads:], slots, wq, wk, cos, sin, positions, pairs=pairs)
    q_alone, k_alone = ops.qk_norm_rope(packed[:, :2 * heads], packed[:, 2 * heads:3 * heads], wq, wk, cos, sin, positions, pairs=pairs)
    ops.kv_write(two, k_alone, packed[:, 3 * heads:], slots)
    assert torch.equal(q, q_alone)
    (k1, v1), (k2, v2) = ops.kv_read(one, slots, dtype=dtype), ops.kv_read(two, slots, dtype=dtype)
    assert torch.equal(v1, v2)
    # the rounding of k_alone to 16 bits, a step of the codes (either way), and the last rounding of both
    top = k_alone.double().abs().amax(-1, keepdim=True)
    step = top / 127 if kind == INT8 else k_alone.double().abs() / 8 + top / 448 / 512
    assert ((k1.double() - k2.double()).abs() <= 1.01 * step + 4 * ref.ROUND[dtype] * top).all()


@pytest.mark.parametrize("kind,dtype,dim,rot,pairs,page", [(INT8, BF16, 128, 128, False, 64), (E4M3, F16, 64, 32, True, 16), (INT8, F16, 256, 256, False, 32), (E4M3, BF16, 96, 96, True, 16)])
def test_a_whole_step(ops, device, kind, dtype, dim, rot, pairs, page):
    """Norm, rotation and write in one launch, then attention: the stored keys are the rotated ones, quantised from 32 bits."""
    g = gen(dim + page)
    context, new, hq, hkv = [37, 0, 300], [5, 3, 8], 6, 2
    table, pages = paged([c + n for c, n in zip(context, new)], page, g)
    slots = ref.Slots(pages * page, hkv, dim, kind, g)
    tokens = sum(new)
    packed = torch.randn((tokens, hq + 2 * hkv, dim), generator=g).to(dtype)
    wq, wk = ((1 + 0.2 * torch.randn(dim, generator=g)).to(dtype) for _ in range(2))
    cos, sin = tables(400, rot)
    mask = tree_mask(new, 1, g)
    of = torch.repeat_interleave(torch.arange(3), torch.tensor(new))
    start = torch.tensor([0, 5, 8, 16], dtype=torch.int32)
    j = torch.tensor(context)[of] + torch.arange(tokens) - start[of]
    positions = j.to(torch.int32)
    where = (table[of, j // page] * page + j % page).to(torch.int32)
    cache = ops.KvCache(*slots.tensors(page, device))
    on = packed.to(device)
    q = ops.qkv_to_cache(cache, on[:, :hq], on[:, hq:hq + hkv], on[:, hq + hkv:], where.to(device), wq.to(device), wk.to(device), cos.to(device), sin.to(device),
                         positions.to(device), pairs=pairs)
    out = ops.tree_attention(q, cache, table.to(device), torch.tensor(context, dtype=torch.int32, device=device), start.to(device), max_new=8, max_context=300, mask=mask.to(device))
    want, slack = ref.norm_rotate(packed[:, :hq], wq, cos, sin, positions, 1e-6, pairs)
    ref.check(q, want, slack * 1.01 + want.abs() * ref.ROUND[dtype] + ref.LEAST[dtype], "q")
    have = ref.Slots.of(cache)
    want, slack = ref.norm_rotate(packed[:, hq:hq + hkv], wk, cos, sin, positions, 1e-6, pairs)
    # half a step of the codes: of the scale for int8, of the value (three bits behind its first) or of the smallest step for e4m3
    scale = (want.abs().amax(-1, keepdim=True) / ref.TOP[kind])
    step = 0.5 * scale if kind == INT8 else torch.maximum(want.abs() * 2.0 ** -4, scale * 2.0 ** -10)
    ref.check(have.keys(where.long()), want, step * 1.001 + 2 * slack.amax(-1, keepdim=True))
    codes, vs = ref.quantise(packed[:, hq + hkv:], kind)
    assert torch.equal(have.vs[where.long()], vs) and torch.equal(ref.values_of(have.v[where.long()], kind, vs), ref.values_of(codes, kind, vs))
    want, bound, _ = ref.attention(q.cpu(), have, page, table, torch.tensor(context), start, mask, dim ** -0.5, dtype)
    ref.check(out, want, bound, "out")


def test_on_another_stream_and_in_a_graph(ops, device):
    """The step on a stream of its own, then captured: every replay, with eager work between them, gives the eager result."""
    g = gen(51)
    table, pages = paged([3001, 33], 16, g)
    cache = ops.KvCache(*ref.Slots(pages * 16, 2, 64, INT8, g).tensors(16, device))
    packed = torch.randn((4, 12, 64), generator=g).to(BF16).to(device)
    cos, sin = (t.to(device) for t in tables(4000, 64))
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)      # noqa: E731
    context, start, positions = ints(2998, 32), ints(0, 3, 4), ints(2998, 2999, 3000, 32)
    j = positions.long()
    where = (table.to(device)[ints(0, 0, 0, 1).long(), j // 16] * 16 + j % 16).to(torch.int32)
    w = torch.ones(64, dtype=BF16, device=device)
    tab = table.to(device)

    def step():
        q = ops.qkv_to_cache(cache, packed[:, :8], packed[:, 8:10], packed[:, 10:], where, w, w, cos, sin, positions)
        return ops.tree_attention(q, cache, tab, context, start, max_new=3, max_context=2998), *ops.kv_read(cache, where)

    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for replay in range(4):
        for t in held:
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), replay
        step()
        torch.cuda.synchronize()


def test_last_launch_names_the_kernels(ops, device):
    import fusedkernellibrary_amd as fkl
    cache = ops.KvCache.allocate(2, 1, 16, 64, device=device)
    x = torch.zeros((1, 1, 64), dtype=BF16, device=device)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)      # noqa: E731
    ops.kv_write(cache, x, x, ints(0))
    assert fkl.last_launch()["form"] == "heads"
    ops.kv_read(cache, ints(0))
    assert fkl.last_launch()["form"] == "kv_read"
    ops.tree_attention(x, cache, ints(0, 1).view(1, 2), ints(0), ints(0, 1), max_new=1, max_context=0)
    assert fkl.last_launch()["form"] == "tree_attention_1x8"


@pytest.mark.parametrize("kind,new,said", [(INT8, 1, None), (E4M3, 40, None), (INT8, 5, 60000)])
def test_caches_beyond_4_gib(ops, device, kind, new, said):
    """Pages whose keys and values lie beyond 2^32 bytes, and whose slots' elements are beyond 2^32: the same bits as in a small cache."""
    g = gen(new)
    heads, page, dim, tokens = 8, 128, 128, 700
    pages = 2 ** 32 // (heads * page * dim) + 16
    large, small = (ops.KvCache.allocate(n, heads, page, dim, codes=kind, device=device) for n in (pages, 16))
    order = torch.randperm(8, generator=g)[:6]
    k, v = torch.randn((2, tokens, heads, dim), generator=g).to(BF16).to(device)
    q = torch.randn((new, 16, dim), generator=g).to(BF16).to(device)
    j, got = torch.arange(tokens), []
    for cache, first in ((large, pages - 8), (small, 4)):
        table = (order + first).to(torch.int32)
        slots = (table[j // page] * page + j % page).to(torch.int32).to(device)
        if said is not None:
            table = torch.nn.functional.pad(table, (0, said // page + 1 - len(table)), value=1 << 30)
        ops.kv_write(cache, k, v, slots)
        context, start = (torch.tensor(x, dtype=torch.int32, device=device) for x in ([tokens - new], [0, new]))
        out = ops.tree_attention(q, cache, table[None].to(device), context, start, max_new=new, max_context=tokens - new if said is None else said)
        got.append((out, *ops.kv_read(cache, slots)))
    assert (pages - 8) * heads * page * dim > 2 ** 32
    for a, b in zip(*got):
        assert a.abs().max() > 0 and torch.equal(a, b)


# ---- the step from C++, the example, refusals -------------------------------------------------------------------------

def test_a_step_through_the_host_api(ops, device):
    """The same kernels on the same inputs from the C++ host API: the same bits. Long contexts make its workspace grow."""
    import ctypes as C
    import os
    import fusedkernellibrary_amd as fkl
    fkl.lib()
    step = C.CDLL(os.path.join(os.path.dirname(os.path.abspath(__file__)), "cases", "libattention_step.so"))
    step.attention_step_error.restype = C.c_char_p
    p, i64, i32 = C.c_void_p, C.c_int64, C.c_int32
    step.attention_step_open.argtypes = [i64, i32, i32, i32, i32, C.POINTER(p)]
    step.attention_step_close.argtypes = [p]
    step.attention_step_run.argtypes = [p] * 9 + [i64] + [p] * 3 + [i64, p, p, i32, i64] + [i32] * 4 + [p]
    server = p()
    assert step.attention_step_open(0, 2, 16, 64, 0, C.byref(server)) == 2                      # no pages
    hq, hkv, dim, page, entries = 8, 2, 64, 16, 400
    assert step.attention_step_open(2 * entries, hkv, page, dim, 0, C.byref(server)) == 0, step.attention_step_error()
    try:
        g = gen(8)
        cache = ops.KvCache.allocate(2 * entries, hkv, page, dim, device=device)
        table = torch.randperm(2 * entries, generator=g).to(torch.int32).view(2, entries)
        wq, wk = ((1 + 0.2 * torch.randn(dim, generator=g)).to(BF16).to(device) for _ in range(2))
        cos, sin = (t.to(device) for t in tables(entries * page, dim))
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)      # noqa: E731
        on = table.to(device)
        for context, new in (([0, 0], [5000, 70]), ([5000, 70], [1, 3])):
            tokens = sum(new)
            packed = torch.randn((tokens, hq + 2 * hkv, dim), generator=g).to(BF16).to(device)
            of = torch.repeat_interleave(torch.arange(2), torch.tensor(new)).to(device)
            start, have = ints([0, new[0], tokens]), ints(context)
            j = have[of] + torch.arange(tokens, device=device) - start[of]
            slots = (on[of, j.long() // page] * page + j % page).to(torch.int32)
            positions = j.to(torch.int32)
            again = packed.clone()
            out, k_out, v_out = torch.empty_like(packed[:, :hq]).contiguous(), *(torch.empty((tokens, hkv, dim), dtype=BF16, device=device) for _ in range(2))
            q = ops.qkv_to_cache(cache, packed[:, :hq], packed[:, hq:hq + hkv], packed[:, hq + hkv:], slots, wq, wk, cos, sin, positions)
            want = ops.tree_attention(q, cache, on, have, start, max_new=max(new), max_context=max(context))
            want_k, want_v = ops.kv_read(cache, slots)
            rc = step.attention_step_run(server, again.data_ptr(), out.data_ptr(), k_out.data_ptr(), v_out.data_ptr(), wq.data_ptr(), wk.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                                         entries * page, positions.data_ptr(), slots.data_ptr(), on.data_ptr(), entries, have.data_ptr(), start.data_ptr(), 2, tokens, hq, max(new),
                                         max(context), 0, torch.cuda.current_stream().cuda_stream)
            assert rc == 0, step.attention_step_error()
            torch.cuda.synchronize()
            for got, expected in ((again[:, :hq], q), (out, want), (k_out, want_k), (v_out, want_v)):
                assert torch.equal(got, expected)
    finally:
        torch.cuda.synchronize()
        step.attention_step_close(server)


@pytest.mark.parametrize("heads,kv_heads,dim,codes", [(32, 8, 128, INT8), (6, 2, 64, E4M3)])
def test_drafts_verified_as_trees_and_one_by_one(ops, device, heads, kv_heads, dim, codes):
    """The example: both ways round a result (2^-8 of it) and their weights (2^-11 of the values) by themselves."""
    import importlib.util
    import os
    spec = importlib.util.spec_from_file_location("verify_drafts", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "verify_drafts.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    difference, largest = example.main(heads=heads, kv_heads=kv_heads, dim=dim, codes=codes)
    assert 0 < largest and difference <= 2 * (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -12) * largest


def test_bindings_refuse_what_does_not_fit(ops, device):
    cache = ops.KvCache.allocate(4, 2, 16, 64, device=device)
    rows = lambda heads=4, tokens=3, dim=64, dtype=BF16, where=device: torch.zeros((tokens, heads, dim), dtype=dtype, device=where)      # noqa: E731
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)      # noqa: E731
    table, lengths, start = ints(0, 1).view(1, 2), ints(4), ints(0, 3)
    call = lambda **c: ops.tree_attention(**{**dict(q=rows(), cache=cache, page_table=table, context=lengths, q_start=start, max_new=3, max_context=4), **c})      # noqa: E731
    call()
    for change, word in ((dict(q=rows(dim=128)), "different sizes"), (dict(q=rows(dtype=torch.float32)), "bfloat16"), (dict(q=rows(where="cpu")), "device"), (dict(q=rows(heads=3)), "multiple of kv_heads"),
                         (dict(page_table=table.long()), "page_table"), (dict(page_table=table[0]), "page_table"), (dict(context=ints(4, 4)), "context"), (dict(q_start=ints(0)), "q_start"),
                         (dict(mask=torch.zeros((2, 1), dtype=torch.int64, device=device)), "mask"), (dict(mask=torch.zeros((3, 1), dtype=torch.int32, device=device)), "mask"),
                         (dict(mask=torch.zeros((3, 0), dtype=torch.int64, device=device)), "word"), (dict(out=rows(heads=5)), "out"), (dict(lse=torch.zeros((3, 4), device=device).half()), "lse"),
                         (dict(max_new=1 << 40), "max_new"), (dict(max_new=-1), "max_new"), (dict(q=rows().transpose(1, 2).contiguous().transpose(1, 2)), "tight"),
                         (dict(q=rows().requires_grad_()), "gradient"), (dict(scale=float("inf")), "finite")):
        with pytest.raises(ValueError, match=word):
            call(**change)
    with torch.no_grad():
        call(q=rows().requires_grad_())
    x, slots = rows(heads=2), ints(0, 1, 2)
    for f, word in ((lambda: ops.kv_write(cache, x, x, slots[:2]), "slots"), (lambda: ops.kv_write(cache, x, rows(heads=3), slots), "v has to be"), (lambda: ops.kv_write(cache, x, x.half(), slots), "v has to be"),
                    (lambda: ops.kv_read(cache, slots, dtype=torch.float32), "dtype"), (lambda: ops.kv_read(cache, slots.view(1, 3)), "one dimension"), (lambda: ops.kv_read(cache, slots, k_out=x.half()), "type"),
                    (lambda: ops.qk_norm_rope(rows(), x, None, None, torch.zeros((9, 32), device=device), None, slots), "neither"),
                    (lambda: ops.qk_norm_rope(rows(), x, torch.ones(64, device=device), torch.ones(64, device=device), None, None, None), "q_weight"),
                    (lambda: ops.qkv_to_cache(cache, rows(heads=3), rows(heads=3), rows(heads=3), slots, None, None, None, None, None), "other heads"),
                    (lambda: ops.KvCache(cache.k, cache.k, cache.k_scale, cache.v_scale), "v has to be"), (lambda: ops.KvCache(cache.k, cache.v, cache.k_scale.half(), cache.v_scale), "k_scale")):
        with pytest.raises(ValueError, match=word):
            f()
    with pytest.raises(ValueError, match="page_tokens"):
        ops.KvCache.allocate(4, 2, 24, 64, device=device)
    with pytest.raises(AttributeError):
        cache.k = cache.k                                                          # a cache is of its tensors for good
    with pytest.raises(ValueError, match="16 bytes"):
        call(q=torch.zeros(3 * 4 * 64 + 1, dtype=BF16, device=device)[1:].view(3, 4, 64))
